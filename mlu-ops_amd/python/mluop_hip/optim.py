"""AdamW over the library's step for many tensors (mluOpExtAdamWStep): a torch optimizer whose step is one launch for every 65 to
106 parameters, by their kind of state, with states in 32 bits or in 8."""
import torch

from . import AdamWTensors
from .nn import _handle

BLOCK = 256  # elements that share a scale of 8-bit states (MLUOP_EXT_ADAMW_BLOCK)


def _lies_as(state, p):
    return state.device == p.device and state.shape == p.shape and state.stride() == p.stride()


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay, as torch.optim.AdamW computes it, in fp32 whatever the parameters' type.

    `state_bits` 32: exp_avg and exp_avg_sq are fp32.  8: float8_e4m3fn codes of exp_avg and of the root of exp_avg_sq
    ("exp_avg_sq" in the state) with one fp32 scale for each 256 elements, for parameters of at least `min_8bit_size`
    elements; smaller ones, whose states weigh nothing, keep 32 bits.  `master_weights`: 16-bit parameters have an fp32 copy
    in the state ("master"), from which every step starts; without it, updates smaller than half a unit in the last
    place of a 16-bit parameter are lost.  All state tensors are ordinary entries of `state`, so state_dict() saves them.
    `step(grad_scale=...)` multiplies the gradients, e.g. by the reciprocal of a loss scale.  Hyperparameters are read on
    the host at every step: a step captured into a graph keeps those of its capture, its step count too."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32,
                 master_weights=False, min_8bit_size=4096):
        if state_bits not in (8, 32):
            raise ValueError("state_bits is 8 or 32")
        if lr < 0 or eps < 0 or weight_decay < 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError("lr, eps and weight_decay are not negative, betas lie in [0, 1)")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, master_weights=bool(master_weights),
                                      min_8bit_size=int(min_8bit_size)))
        self._plans = {}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plans = {}   # (of what a copy was made from; torch copies groups and states only)

    def _state_of(self, p, group):
        state = self.state[p]
        if not state:
            state["step"] = 0
            if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]:
                blocks = -(-p.numel() // BLOCK)
                for name in ("exp_avg", "exp_avg_sq"):
                    state[name] = torch.zeros_like(p, dtype=torch.uint8).view(torch.float8_e4m3fn)
                    state[name + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
            else:
                for name in ("exp_avg", "exp_avg_sq"):
                    state[name] = torch.zeros_like(p, dtype=torch.float32)
            if group["master_weights"] and p.dtype != torch.float32:
                state["master"] = p.detach().to(torch.float32, copy=True)
        return state

    def load_state_dict(self, state_dict):
        """(torch casts a state's floating tensors to their parameter's type: these keep the type they were saved with.)"""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        numbers = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(numbers, (p for g in self.param_groups for p in g["params"])):
            for name, value in saved.get(i, {}).items():
                if isinstance(value, torch.Tensor):
                    self.state[p][name] = value.to(p.device, copy=True)
        self._plans = {}

    @torch.no_grad()
    def step(self, closure=None, grad_scale=1.0):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for number, group in enumerate(self.param_groups):
            for p in group["params"]:
                if p.grad is not None:
                    if p.grad.is_sparse:
                        raise RuntimeError("sparse gradients are not supported")
                    self._state_of(p, group)
            # what a single call can take, but for the step count: one type, one kind of state
            kinds = {}
            for p in group["params"]:
                state = self.state.get(p)
                if state and (p.grad is not None or _lies_as(state["exp_avg"], p)):
                    kinds.setdefault((p.dtype, p.device, "exp_avg_scale" in state, "master" in state), []).append(p)
            for (dtype, device, eight, masters), params in kinds.items():
                # (parameters that have missed gradients are behind; None leaves a parameter alone)
                counts = {}
                for place, p in enumerate(params):
                    if p.grad is not None:
                        counts.setdefault(self.state[p]["step"] + 1, []).append(place)
                if not counts:
                    continue
                with torch.cuda.device(device):
                    plan = self._plan(number, params, eight, masters)
                    for step, places in counts.items():
                        grads = [None] * len(params)
                        for place in places:
                            grads[place] = params[place].grad
                        plan.step(_handle(), grads, step, group["lr"], group["betas"], group["eps"], group["weight_decay"],
                                  grad_scale)
                        for place in places:   # (a step that was refused does not count)
                            self.state[params[place]]["step"] = step
        return loss

    def _plan(self, number, params, eight, masters):
        """The checked tensors of a call, kept while parameters and states stay where they were and as they lay there."""
        states = [self.state[p] for p in params]
        names = ["exp_avg", "exp_avg_sq"] + ["master"] * masters + ["exp_avg_scale", "exp_avg_sq_scale"] * eight
        # (a state follows its parameter's layout; looking at its own too took 270 us of the host in place of 165 for 200
        # parameters with 8-bit states)
        where = ([(p.data_ptr(), p.shape, p.stride()) for p in params] +
                 [s[n].data_ptr() for s in states for n in names])
        key = (number, params[0].dtype, params[0].device, eight, masters)
        kept = self._plans.get(key)
        if kept is None or kept[0] != where:
            def all_of(name):
                return [s[name] for s in states]
            plan = AdamWTensors([p.detach() for p in params], all_of("exp_avg"), all_of("exp_avg_sq"),
                                all_of("master") if masters else None, all_of("exp_avg_scale") if eight else None,
                                all_of("exp_avg_sq_scale") if eight else None)
            kept = self._plans[key] = (where, plan)
        return kept[1]
