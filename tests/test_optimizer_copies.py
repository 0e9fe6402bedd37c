"""What a copy of the AdamW optimizer keeps (no GPU)."""
import copy
import pickle

import torch

from mluop_hip.optim import AdamW


def test_copies_have_all_that_a_step_needs():
    opt = AdamW([torch.nn.Parameter(torch.ones(4))], lr=0.5)
    own = set(vars(opt)) - set(vars(torch.optim.SGD([torch.nn.Parameter(torch.ones(4))], lr=0.5)))   # (and not torch's)
    assert own
    for twin in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt)), copy.copy(opt)):
        assert own <= set(vars(twin))
        assert twin.param_groups[0]["lr"] == 0.5
        twin.step()   # (no gradient: nothing to do)
