"""More operators of a training step over ragged rows: layer norm, a gated linear recurrence along every sample's rows, rows put
into expert order and back with weights, and dropout onto a residual from a counter-based generator.

`run` computes them with elementary torch operations in 32 bits, or, where `own` is set, through this repository's
package.  Sizes are those of the repository's benchmark clouds (3001, 120 000 and 248 636 rows of 64 and 128 channels) and
generic widths of the same kind."""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-5
STEPS = 1 << 16      # a probability of dropping is a multiple of 1 / STEPS
LOW = 0xFFFFFFFF
MULTIPLIERS, WEYL, ROUNDS = (0xD2511F53, 0xCD9E8D57), (0x9E3779B9, 0xBB67AE85), 10   # Philox4x32 (Salmon et al., 2011)


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------

def listed():
    return [
        # The norm of a few rows while a model answers: latency of one small call.
        dict(name="norm_few", op="norm", direction="forward", dtype="bfloat16", params="bfloat16", rows=16, channels=1024),
        # The norm in front of a layer over the voxels of a dense cloud, fp32 parameters.
        dict(name="norm_scene", op="norm", direction="forward", dtype="float16", params="float32", rows=248_636,
             channels=128),
        # Its backward pass, with the gradients of weight and bias, on a batch of wide rows.
        dict(name="norm_grad_wide", op="norm", direction="backward", dtype="bfloat16", params="float32", rows=32_768,
             channels=2048),
        # One step of 64 sequences while a model answers: states in, states out.
        dict(name="scan_step", op="scan", direction="forward", dtype="bfloat16", kind="sigmoid", reverse=False, rows=64,
             samples=64, channels=1024, states=True, padding=0),
        # The recurrence along the voxels of four clouds of different sizes, put into one order.
        dict(name="scan_scene", op="scan", direction="forward", dtype="float16", kind="sigmoid", reverse=False,
             rows=248_636, samples=4, channels=128, states=False, padding=0),
        # A training step through three long wide sequences, from the last row to the first.
        dict(name="scan_train_wide", op="scan", direction="training", dtype="bfloat16", kind="exp", reverse=True, rows=65_536,
             samples=3, channels=1024, states=True, padding=0),
        # A dozen rows sent to two of 32 experts each, one step of a model that answers.
        dict(name="route_few", op="route", direction="forward", dtype="bfloat16", rows=12, choices=2, experts=32,
             channels=1024, skew=0.5, dropped=0.0),
        # A training batch to two of eight wide experts and back.
        dict(name="route_wide", op="route", direction="forward", dtype="bfloat16", rows=32_768, choices=2, experts=8,
             channels=2048, skew=0.3, dropped=0.0),
        # The gradients of rows sent to four of 64 uneven experts, a few of the choices turned away by full ones.
        dict(name="route_grad", op="route", direction="backward", dtype="float16", rows=16_384, choices=4, experts=64,
             channels=1024, skew=0.7, dropped=0.03),
        # The residual behind a layer of a small cloud.
        dict(name="drop_small", op="dropout", direction="forward", dtype="float16", rows=3001, channels=64, p=0.1,
             residual=True),
        # The residual behind a layer over a large batch of wide rows.
        dict(name="drop_wide", op="dropout", direction="forward", dtype="bfloat16", rows=65_536, channels=2048, p=0.1,
             residual=True),
        # Forward and backward over a whole cloud in fp32.
        dict(name="drop_train", op="dropout", direction="training", dtype="float32", rows=248_636, channels=128, p=0.25,
             residual=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "scan", "route", "dropout"])
    dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
    channels = rng.choice([16, 33, 64, 96, 128, 250, 512, 1000, 1024, 2048])
    if op == "norm":
        channels = rng.choice([channels, channels, 4096, 8192])
        return dict(op=op, direction=rng.choice(["forward", "backward"]), dtype=dtype, params=rng.choice(["float32", dtype]),
                    rows=min(_log(rng, 1, 400_000), 60_000_000 // channels), channels=channels)
    if op == "scan":
        rows = min(_log(rng, 1, 300_000), 30_000_000 // channels)
        return dict(op=op, direction=rng.choice(["forward", "training"]), dtype=dtype, kind=rng.choice(["sigmoid", "exp"]),
                    reverse=rng.random() < 0.4, rows=rows, samples=min(rows, rng.choice([1, 1, 2, 5, 16, 64])),
                    channels=channels, states=rng.random() < 0.6, padding=rng.choice([0, 0, 17]))
    if op == "route":
        experts = rng.choice([4, 8, 16, 27, 64, 128, 512])
        choices = rng.choice([1, 2, 2, 3, 4])
        return dict(op=op, direction=rng.choice(["forward", "backward"]), dtype=dtype,
                    rows=min(_log(rng, 1, 60_000), 60_000_000 // (channels * choices)), choices=choices, experts=experts,
                    channels=channels, skew=rng.choice([0.0, 0.5, 1.5]), dropped=rng.choice([0.0, 0.03, 0.3]))
    return dict(op=op, direction=rng.choice(["forward", "training"]), dtype=dtype,
                rows=min(_log(rng, 1, 400_000), 60_000_000 // channels), channels=channels,
                p=rng.choice([0.02, 0.1, 0.25, 0.5]), residual=rng.random() < 0.7)


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(DTYPES[dtype])


def _split(total, parts, skew, rng):
    """`parts` sizes of at least one that add up to `total`, uneven by `skew`."""
    weights = [math.exp(rng.gauss(0.0, skew)) for _ in range(parts)]
    scale = (total - parts) / sum(weights)
    sizes = [1 + int(w * scale) for w in weights]
    for i in range(total - sum(sizes)):
        sizes[i % parts] += 1
    return sizes


def _starts(sizes):
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    return starts


def _package():
    path = os.path.join("mlu-ops_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mluop_hip
    return mluop_hip


def prepare(case, seed):
    g, rng = _generator(seed), random.Random(seed)
    rows, channels, dtype = case["rows"], case["channels"], case["dtype"]
    s = {"case": case}
    if case["op"] == "norm":
        # (rows lie off zero by different amounts, as they do behind residuals)
        s["features"] = (torch.randn((rows, channels), generator=g, device="cuda") +
                         2.0 * torch.randn((rows, 1), generator=g, device="cuda")).to(DTYPES[dtype])
        s["weight"] = (1.0 + 0.2 * torch.randn(channels, generator=g, device="cuda")).to(DTYPES[case["params"]])
        s["bias"] = (0.2 * torch.randn(channels, generator=g, device="cuda")).to(DTYPES[case["params"]])
        if case["direction"] == "backward":
            s["output_grad"] = _randn(g, (rows, channels), dtype)
            s["mean"], s["rstd"] = _moments(s["features"].float())
    elif case["op"] == "scan":
        samples = case["samples"]
        s["host_starts"] = _starts(_split(rows, samples, 0.4, rng))
        s["row_starts"] = torch.tensor(s["host_starts"], dtype=torch.int32, device="cuda")
        # (rows behind the last sequence, as a batch of a fixed size has them)
        shape = (rows + case["padding"], channels)
        s["features"] = _randn(g, shape, dtype)
        gates = torch.randn(shape, generator=g, device="cuda")
        # (memories of one to some hundred rows)
        gates = 1.5 + 1.5 * gates if case["kind"] == "sigmoid" else -torch.exp(1.2 * gates - 2.0)
        s["gates"] = gates.to(DTYPES[dtype])
        s["initial"] = torch.randn((samples, channels), generator=g, device="cuda") if case["states"] else None
        if case["direction"] == "training":
            s["output_grad"] = _randn(g, shape, dtype)
            s["final_grad"] = torch.randn((samples, channels), generator=g, device="cuda") if case["states"] else None
    elif case["op"] == "route":
        experts, choices = case["experts"], case["choices"]
        popular = case["skew"] * torch.randn(experts, generator=g, device="cuda")
        scores, chosen = torch.topk(popular + torch.randn((rows, experts), generator=g, device="cuda"), choices, dim=1)
        gone = torch.rand((rows, choices), generator=g, device="cuda") < case["dropped"]
        s["chosen"] = torch.where(gone, torch.full_like(chosen, -1), chosen).to(torch.int32)
        s["weights"] = torch.softmax(scores, dim=1)
        if case["direction"] == "forward":
            s["features"] = _randn(g, (rows, channels), dtype)
            s["results"] = _randn(g, (rows * choices, channels), dtype)
        else:
            _, s["group_starts"], s["places"] = _order(s["chosen"], experts)
            s["ordered_grad"] = _randn(g, (rows * choices, channels), dtype)
            s["results"] = _randn(g, (rows * choices, channels), dtype)
            s["output_grad"] = _randn(g, (rows, channels), dtype)
    else:
        s["features"] = _randn(g, (rows, channels), dtype)
        s["residual"] = _randn(g, (rows, channels), dtype, 2.0) if case["residual"] else None
        s["output_grad"] = _randn(g, (rows, channels), dtype) if case["direction"] == "training" else None
        # seed of the generator and number of the call
        s["state"] = torch.tensor([rng.randrange(1 << 62), rng.randrange(1 << 40)], dtype=torch.int64, device="cuda")
    if own:
        s["handle"] = _package().make_handle_on_current_stream()
    return s


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return (_RUN_OWN if own else _RUN_PLAIN)[case["op"]](state, case)


def _moments(x):
    mean = x.mean(dim=1)
    off = x - mean.unsqueeze(1)
    return mean, torch.rsqrt((off * off).mean(dim=1) + EPS)


def _norm_plain(s, case):
    x, w, b = s["features"].float(), s["weight"].float(), s["bias"].float()
    mean, rstd = _moments(x) if case["direction"] == "forward" else (s["mean"], s["rstd"])
    xhat = (x - mean.unsqueeze(1)) * rstd.unsqueeze(1)
    if case["direction"] == "forward":
        return (xhat * w + b).to(s["features"].dtype), mean, rstd
    dy = s["output_grad"].float()
    dw, db = (dy * xhat).sum(dim=0), dy.sum(dim=0)
    d = dy * w
    dx = rstd.unsqueeze(1) * (d - d.mean(dim=1, keepdim=True) - xhat * (d * xhat).mean(dim=1, keepdim=True))
    return dx.to(s["features"].dtype), dw.to(s["weight"].dtype), db.to(s["bias"].dtype)


def _norm_own(s, case):
    package = _package()
    if case["direction"] == "forward":
        return package.layer_norm_forward(s["handle"], s["features"], s["weight"], s["bias"], EPS)
    return package.layer_norm_backward(s["handle"], s["output_grad"], s["features"], s["weight"], s["bias"], s["mean"],
                                       s["rstd"])


def _scan(a, b):
    """h_t = a_t h_(t-1) + b_t down the rows, from zero: every step doubles how far a row has looked back."""
    d = 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], torch.addcmul(b[d:], a[d:], b[:-d])])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _scan_plain(s, case):
    x, gates, starts = s["features"].float(), s["gates"].float(), s["row_starts"].long()
    rows = x.shape[0]
    if case["reverse"]:
        x, gates, starts = x.flip(0), gates.flip(0), rows - starts.flip(0)
    initial = s["initial"]
    if initial is None:
        initial = torch.zeros((case["samples"], case["channels"]), device="cuda")
    elif case["reverse"]:
        initial = initial.flip(0)
    a = torch.sigmoid(gates) if case["kind"] == "sigmoid" else torch.exp(gates)
    u = torch.sigmoid(-gates) if case["kind"] == "sigmoid" else torch.ones_like(a)
    # every sample has a row: its first does not look back but at the initial state
    first, last = starts[:-1], starts[1:] - 1
    begins = torch.zeros((rows, 1), device="cuda")
    begins[first] = 1.0
    before = torch.zeros_like(a)
    before[first] = initial
    row = torch.arange(rows, device="cuda").unsqueeze(1)
    inside = ((row >= starts[0]) & (row < starts[-1])).float()
    h = _scan(a * (1.0 - begins), (u * x + a * before) * inside) * inside
    final = h[last]
    outputs = {"out": _back(h, s, case), "final": final.flip(0) if case["reverse"] else final}
    if case["direction"] == "forward":
        return outputs
    dh = (s["output_grad"].flip(0) if case["reverse"] else s["output_grad"]).float() * inside
    if s["final_grad"] is not None:
        dh[last] += s["final_grad"].flip(0) if case["reverse"] else s["final_grad"]
    # l_t = dh_t + a_(t+1) l_(t+1), not across a sample's end
    after = torch.cat([(a * (1.0 - begins))[1:], torch.zeros_like(a[:1])])
    after[last] = 0.0
    l = _scan(after.flip(0), dh.flip(0)).flip(0) * inside
    previous = torch.cat([torch.zeros_like(h[:1]), h[:-1]]) * (1.0 - begins) + before
    if case["kind"] == "sigmoid":
        dx, dg = u * l, l * (previous - x) * a * u
    else:
        dx, dg = l, l * previous * a
    outputs["features_grad"], outputs["gates_grad"] = _back(dx, s, case), _back(dg, s, case)
    if s["initial"] is not None:
        di = (a * l)[first]
        outputs["initial_grad"] = di.flip(0) if case["reverse"] else di
    return outputs


def _back(rows, s, case):
    return (rows.flip(0) if case["reverse"] else rows).to(s["features"].dtype)


def _scan_own(s, case):
    package = _package()
    out, final, carries = package.gated_scan_forward(s["handle"], s["features"], s["gates"], s["row_starts"], s["initial"],
                                                     case["kind"], case["reverse"])
    outputs = {"out": out, "final": final}
    if case["direction"] == "training":
        dx, dg, di = package.gated_scan_backward(s["handle"], s["output_grad"], s["final_grad"], s["features"], s["gates"],
                                                 carries, s["row_starts"], case["kind"], case["reverse"])
        outputs["features_grad"], outputs["gates_grad"] = dx, dg
        if s["initial"] is not None:
            outputs["initial_grad"] = di
    return outputs


def _order(chosen, experts):
    """The row at every place when all choices are ordered by expert (-1 behind the last expert's), where each expert's begin,
    and the place of every choice (-1 of one without an expert)."""
    flat = chosen.reshape(-1).long()
    flat = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    ordered, order = torch.sort(flat, stable=True)
    starts = torch.searchsorted(ordered, torch.arange(experts + 1, device="cuda"), out_int32=True)
    places = torch.empty_like(order)
    places[order] = torch.arange(order.shape[0], device="cuda")
    rows = torch.where(ordered < experts, order // chosen.shape[1], -1).to(torch.int32)
    return rows, starts, torch.where(flat < experts, places, -1).to(torch.int32).view(chosen.shape)


def _of_places(rows, places):
    """Rows in 32 bits at [row, choice], zeros where a choice has no place."""
    found = rows[places.long().clamp(min=0)].float()
    return torch.where((places >= 0).unsqueeze(2), found, torch.zeros((), device="cuda"))


def _to_places(values, places):
    """[row, choice, channels] brought to the places, zeros behind them."""
    n = places.numel()
    out = torch.zeros((n + 1, values.shape[2]), dtype=values.dtype, device="cuda")
    out[torch.where(places >= 0, places.long(), n).view(-1)] = values.reshape(n, -1)
    return out[:n]


def _route_plain(s, case):
    w, results = s["weights"].unsqueeze(2), s["results"]
    if case["direction"] == "forward":
        rows, starts, places = _order(s["chosen"], case["experts"])
        x = s["features"]
        ordered = _to_places(x.unsqueeze(1).expand(-1, case["choices"], -1), places)
        out = (_of_places(results, places) * w).sum(dim=1).to(results.dtype)
        return {"rows": rows, "starts": starts, "places": places, "ordered": ordered, "out": out}
    places, dy = s["places"], s["output_grad"].float().unsqueeze(1)
    return {"features_grad": _of_places(s["ordered_grad"], places).sum(dim=1).to(results.dtype),
            "results_grad": _to_places((dy * w).to(results.dtype), places),
            "weights_grad": (dy * _of_places(results, places)).sum(dim=2)}


def _route_own(s, case):
    package, handle = _package(), s["handle"]
    if case["direction"] == "forward":
        rows, starts, places = package.expert_order(handle, s["chosen"], case["experts"])
        ordered = package.expert_dispatch(handle, s["features"], places, starts)
        out = package.expert_combine(handle, s["results"], places, s["weights"])
        return {"rows": rows, "starts": starts, "places": places, "ordered": ordered, "out": out}
    dx = package.expert_combine(handle, s["ordered_grad"], s["places"])
    dr, dw = package.expert_combine_backward(handle, s["output_grad"], s["results"], s["places"], s["weights"],
                                             s["group_starts"])
    return {"features_grad": dx, "results_grad": dr, "weights_grad": dw}


def _random_words(state, count):
    """Four words for each of `count` counters: Philox4x32 with the counter (element group, call) and the seed as key."""
    group = torch.arange(count, device="cuda")
    key = [state[0] & LOW, (state[0] >> 32) & LOW]
    c = [group & LOW, group >> 32, (state[1] & LOW).expand(count), ((state[1] >> 32) & LOW).expand(count)]
    for _ in range(ROUNDS):
        # (products of two 32-bit words: 64 bits, whose sign does not matter)
        p, q = c[0] * MULTIPLIERS[0], c[2] * MULTIPLIERS[1]
        c = [((q >> 32) & LOW) ^ c[1] ^ key[0], q & LOW, ((p >> 32) & LOW) ^ c[3] ^ key[1], p & LOW]
        key = [(k + w) & LOW for k, w in zip(key, WEYL)]
    return c


def _threshold(p):
    return int(math.floor(p * STEPS + 0.5))


def _kept(state, n, p):
    """Which of n elements are kept: eight of them share a counter, two each of its words, the lower half first."""
    words = torch.stack(_random_words(state, -(-n // 8)), dim=1)
    halves = torch.stack([words & 0xFFFF, words >> 16], dim=2)
    return halves.view(-1)[:n] >= _threshold(p)


def _dropout_plain(s, case):
    x, p = s["features"], case["p"]
    kept, scale = _kept(s["state"], x.numel(), p).view(x.shape), STEPS / (STEPS - _threshold(p))
    zero = torch.zeros((), device="cuda")
    out = torch.where(kept, x.float() * scale, zero)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    if case["direction"] == "forward":
        return out.to(x.dtype)
    return out.to(x.dtype), torch.where(kept, s["output_grad"].float() * scale, zero).to(x.dtype)


def _dropout_own(s, case):
    package = _package()
    out = package.dropout_add_forward(s["handle"], s["features"], s["residual"], case["p"], s["state"])
    if case["direction"] == "forward":
        return out
    return out, package.dropout_add_backward(s["handle"], s["output_grad"], case["p"], s["state"])


_RUN_PLAIN = {"norm": _norm_plain, "scan": _scan_plain, "route": _route_plain, "dropout": _dropout_plain}
_RUN_OWN = {"norm": _norm_own, "scan": _scan_own, "route": _route_own, "dropout": _dropout_own}


# ---------------------------------------------------------------------------------------------
# Least work, and the definitions in 64 bits
# ---------------------------------------------------------------------------------------------

def work(case):
    op, forward = case["op"], case["direction"] == "forward"
    size = 4 if case["dtype"] == "float32" else 2
    values = case["rows"] * case["channels"]
    if op == "norm":
        # x in, y out; x and dy in, dx out
        return {"bytes": values * size * (2 if forward else 3), "flops": values * (8 if forward else 16)}
    if op == "scan":
        # x and gates in, h out; the outputs' gradients in, two gradients out
        states = 4 * case["samples"] * case["channels"] * (2 if case["states"] else 1)
        return {"bytes": values * size * (3 if forward else 6) + states, "flops": values * (8 if forward else 24)}
    if op == "route":
        # features to their places and results back; both of their gradients
        k, n = case["choices"], case["rows"] * case["choices"]
        return {"bytes": values * size * (2 * k + 2 if forward else 3 * k + 2) + 16 * n,
                "flops": values * k * (2 if forward else 4)}
    tensors = 2 + (1 if case["residual"] else 0) + (0 if forward else 2)
    return {"bytes": values * size * tensors, "flops": values * 16 * (1 if forward else 2)}


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return _EXACT[case["op"]](s, case)


def _norm_exact(s, case):
    x, w, b = s["features"].double(), s["weight"].double(), s["bias"].double()
    if case["direction"] == "forward":
        var, mean = torch.var_mean(x, dim=1, unbiased=False)
        rstd = (var + EPS) ** -0.5
        return torch.addcmul(b, (x - mean[:, None]) / torch.sqrt(var + EPS)[:, None], w), mean, rstd
    mean, rstd, dy = s["mean"].double(), s["rstd"].double(), s["output_grad"].double()
    n = (x - mean[:, None]) * rstd[:, None]
    c = x.shape[1]
    d = dy * w
    along = (d * n).sum(1) / c
    dx = (d - (d.sum(1) / c)[:, None] - n * along[:, None]) * rstd[:, None]
    return dx, (dy * n).sum(0), dy.sum(0)


def _scan_exact(s, case):
    """One row after the other."""
    x, g = s["features"].double(), s["gates"].double()
    mixed = case["kind"] == "sigmoid"
    a = 1.0 / (1.0 + torch.exp(-g)) if mixed else torch.exp(g)
    u = 1.0 / (1.0 + torch.exp(g)) if mixed else torch.ones_like(g)
    b = u * x
    training = case["direction"] == "training"
    h, l, previous = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    shape = (case["samples"], case["channels"])
    final, di = (torch.zeros(shape, dtype=torch.float64, device="cuda") for _ in range(2))
    dy = s["output_grad"].double() if training else None
    for k, (lo, hi) in enumerate(zip(s["host_starts"], s["host_starts"][1:])):
        way = list(range(lo, hi))
        if case["reverse"]:
            way.reverse()
        at = torch.zeros_like(x[0]) if s["initial"] is None else s["initial"][k].double()
        for t in way:
            if training:
                previous[t] = at
            at = torch.addcmul(b[t], a[t], at, out=h[t])
        final[k] = at
        if training:
            at = torch.zeros_like(x[0]) if s["final_grad"] is None else s["final_grad"][k].double()
            for t in reversed(way):
                torch.add(dy[t], at, out=l[t])
                at = a[t] * l[t]
            di[k] = at
    outputs = {"out": h, "final": final}
    if training:
        outputs["features_grad"] = u * l
        outputs["gates_grad"] = l * (previous - x) * a * u if mixed else l * previous * a
        if s["initial"] is not None:
            outputs["initial_grad"] = di
    return outputs


def _route_exact(s, case):
    choices, r = case["choices"], s["results"].double()
    if case["direction"] == "forward":
        # the places anew, on the host
        chosen = s["chosen"].cpu().numpy().reshape(-1).astype(np.int64)
        order = np.argsort(np.where(chosen < 0, case["experts"], chosen), kind="stable")
        places = np.empty_like(order)
        places[order] = np.arange(order.size)
        places = torch.from_numpy(places).cuda().view(-1, choices)
        there = (s["chosen"] >= 0).double()
        x = s["features"].double()
        ordered = x[torch.from_numpy(order // choices).cuda()]
        ordered[int((chosen >= 0).sum()):] = 0.0
        out = 0.0
        for k in range(choices):
            out = out + r[places[:, k]] * (s["weights"][:, k].double() * there[:, k])[:, None]
        return {"rows": None, "starts": None, "places": None, "ordered": ordered, "out": out}
    dx, dw, dr = 0.0, [], torch.zeros_like(r)
    dy = s["output_grad"].double()
    for k in range(choices):
        there = torch.nonzero(s["places"][:, k] >= 0)[:, 0]
        at = s["places"][there, k].long()
        part = torch.zeros_like(dy)
        part[there] = s["ordered_grad"][at].double()
        dx = dx + part
        dr[at] = dy[there] * s["weights"][there, k].double()[:, None]
        along = torch.zeros(dy.shape[0], dtype=torch.float64, device="cuda")
        along[there] = torch.linalg.vecdot(dy[there], r[at])
        dw.append(along)
    return {"features_grad": dx, "results_grad": dr, "weights_grad": torch.stack(dw, dim=1)}


def _dropout_exact(s, case):
    """The generator anew with unsigned words of 64 bits on the host, some counters at a time."""
    n, (seed, call) = s["features"].numel(), (int(v) for v in s["state"].cpu())
    kept = np.empty(-(-n // 8) * 8, dtype=bool)
    low, shift = np.uint64(LOW), np.uint64(32)
    for at in range(0, kept.size // 8, 1 << 18):
        c0 = np.arange(at, min(at + (1 << 18), kept.size // 8), dtype=np.uint64)
        c1, c0 = c0 >> shift, c0 & low
        c2, c3 = np.full_like(c0, call & LOW), np.full_like(c0, call >> 32)
        for r in range(ROUNDS):
            k0, k1 = np.uint64(((seed & LOW) + r * WEYL[0]) & LOW), np.uint64(((seed >> 32) + r * WEYL[1]) & LOW)
            p, q = c0 * np.uint64(MULTIPLIERS[0]), c2 * np.uint64(MULTIPLIERS[1])
            c0, c1, c2, c3 = (q >> shift) ^ c1 ^ k0, q & low, (p >> shift) ^ c3 ^ k1, p & low
        words = np.stack([c0, c1, c2, c3], axis=1).astype("<u4").view("<u2")
        kept[8 * at:8 * at + words.size] = words.reshape(-1) >= _threshold(case["p"])
    kept = torch.from_numpy(kept[:n]).cuda().view(s["features"].shape)
    scale = 1.0 / (1.0 - _threshold(case["p"]) / STEPS)
    out = s["features"].double().mul_(scale).mul_(kept)
    if s["residual"] is not None:
        out += s["residual"].double()
    if case["direction"] == "forward":
        return out
    return out, s["output_grad"].double() * scale * kept


_EXACT = {"norm": _norm_exact, "scan": _scan_exact, "route": _route_exact, "dropout": _dropout_exact}
