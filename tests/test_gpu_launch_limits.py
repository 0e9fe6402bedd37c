"""Sizes whose workgroups do not fit into one launch: a grid has fewer than 2^32 work-items along x, 2^24 workgroups of 256
threads, and 65 536 workgroups along y."""
import pytest

pytestmark = pytest.mark.gpu


def room_for(gib):
    import torch
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib * 2 ** 30:
        pytest.skip("needs %d GiB of free device memory" % gib)


def all_are(tensor, value):
    """(a plain truth value: pytest would spell out a comparison of such tensors element by element)"""
    return all(bool((part == value).all()) for part in tensor.split(1 << 30))


@pytest.fixture
def handle(gpu_handle):
    """without guard bands, whose checks would read all of these tensors once more"""
    import torch
    import mluop_hip
    kept, mluop_hip.GUARD_BYTES = mluop_hip.GUARD_BYTES, 0
    try:
        yield gpu_handle
    finally:
        mluop_hip.GUARD_BYTES = kept
        torch.cuda.empty_cache()


def test_adamw_of_a_tensor_longer_than_a_launch(handle):
    """2^24 workgroups of 2048 elements, behind a small tensor; the gradient is the parameter itself, which is read first"""
    import torch
    import mluop_hip
    room_for(140)
    n = (1 << 35) + 5000
    params = [torch.ones(k, dtype=torch.bfloat16, device="cuda") for k in (3000, n)]
    codes = [[torch.zeros(p.numel(), dtype=torch.uint8, device="cuda") for p in params] for _ in range(2)]
    scales = [[torch.zeros(-(-p.numel() // 256), device="cuda") for p in params] for _ in range(2)]
    plan = mluop_hip.AdamWTensors(params, *codes, None, *scales)
    plan.step(handle, params, 1, lr=0.5, betas=(0.5, 0.75), eps=0.0, weight_decay=0.0)
    # m = 1/2 and the root of v = 1/2, corrected both are 1: a step of 0.5, and every code the largest
    for p, m, r, ms, rs in zip(params, *codes, *scales):
        assert all_are(p, 0.5)
        assert all_are(m, 0x7e) and all_are(r, 0x7e)
        want = float(torch.tensor(0.5) * torch.tensor(1.0 / 448.0))
        assert all_are(ms, want) and all_are(rs, want)
