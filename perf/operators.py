"""Operators around the sparse convolutions in a training step: embedding lookup with the gradient of its table, group norm
with an activation over ragged samples, products grouped by expert and the AdamW step over many tensors.

`run` computes them with elementary torch operations in 32 bits, or, where `own` is set, through this repository's
package.  Sizes are those of the repository's benchmark clouds (3001, 120 000, 248 636 and 400 000 rows of 64 and 128
channels) and generic widths of the same kind."""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BLOCK = 256          # elements that share a scale of the 8-bit optimizer states
E4M3_MAX = 448.0
E4M3_LEAST = 2.0 ** -9
EPS = 1e-5
ADAMW = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.01)


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------

def listed():
    return [
        # The categories of a few rows looked up while a model answers: latency of one small call.
        dict(name="embed_few", op="embedding", direction="forward", dtype="bfloat16", tokens=64, rows=32_768,
             channels=1024, skew=1.0, outside=0.0),
        # Gradient of a small fp32 table of categories over a cloud's voxels: every row is named hundreds of times.
        dict(name="embed_grad_categories", op="embedding", direction="backward", dtype="float32", tokens=120_000,
             rows=517, channels=64, skew=1.0, outside=0.01),
        # Gradient of a large table in a training step: most rows unnamed, the commonest named thousands of times.
        dict(name="embed_grad_large", op="embedding", direction="backward", dtype="bfloat16", tokens=65_536,
             rows=131_072, channels=2048, skew=1.0, outside=0.02),
        # The norm behind a layer of a small cloud, as a program that answers runs it.
        dict(name="norm_small", op="norm", direction="forward", dtype="float16", params="float32", rows=3001, samples=1,
             channels=64, groups=16, activation="relu"),
        # The norm behind the widest layer of an encoder, four clouds of different sizes.
        dict(name="norm_scene", op="norm", direction="forward", dtype="float16", params="float32", rows=248_636,
             samples=4, channels=128, groups=32, activation="silu"),
        # Its backward pass on a large batch.
        dict(name="norm_grad_large", op="norm", direction="backward", dtype="bfloat16", params="float32", rows=400_000,
             samples=2, channels=128, groups=32, activation="silu"),
        # A dozen rows sent to ten of 32 experts, one step of a model that answers: the filters are what is read.
        dict(name="experts_few", op="experts", direction="forward", dtype="bfloat16", rows=12, groups=32, active=10,
             ci=1024, co=2048, skew=0.5),
        # A long prompt or a training batch through eight wide experts.
        dict(name="experts_wide", op="experts", direction="forward", dtype="bfloat16", rows=32_768, groups=8, active=8,
             ci=2048, co=8192, skew=0.3),
        # Both gradients of a layer with many experts of uneven loads, some without a row.
        dict(name="experts_grad", op="experts", direction="backward", dtype="float16", rows=16_384, groups=24, active=21,
             ci=1024, co=4096, skew=0.7),
        # The step of a small sparse encoder: a few dozen small fp32 tensors.
        dict(name="adamw_encoder", op="adamw", dtype="float32", master=False, bits=32, tensors=33, total=1_900_000, step=7),
        # 16-bit parameters with fp32 copies and 32-bit states.
        dict(name="adamw_master", op="adamw", dtype="bfloat16", master=True, bits=32, tensors=150, total=130_000_000,
             step=300),
        # 16-bit parameters with 8-bit states and no copies: the step of a large model on one card.
        dict(name="adamw_8bit", op="adamw", dtype="bfloat16", master=False, bits=8, tensors=200, total=250_000_000, step=20),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["embedding", "norm", "experts", "adamw"])
    dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
    if op == "embedding":
        channels = rng.choice([16, 33, 64, 96, 250, 512, 1000, 1024, 2048])
        rows = min(_log(rng, 17, 131_072), 250_000_000 // channels)
        return dict(op=op, direction=rng.choice(["forward", "backward", "backward"]), dtype=dtype,
                    tokens=min(_log(rng, 1, 300_000), 130_000_000 // channels), rows=rows, channels=channels,
                    skew=rng.choice([0.0, 0.7, 1.0, 1.3]), outside=rng.choice([0.0, 0.05, 0.3]))
    if op == "norm":
        groups = rng.choice([1, 4, 8, 16, 32])
        channels = groups * rng.choice([1, 2, 3, 4, 8, 16])
        samples = rng.choice([1, 1, 2, 4, 7, 16])
        return dict(op=op, direction=rng.choice(["forward", "backward"]), dtype=dtype,
                    params=rng.choice(["float32", dtype]), rows=min(_log(rng, 16, 400_000), 50_000_000 // channels),
                    samples=samples, channels=channels, groups=groups,
                    activation=rng.choice(["none", "relu", "silu"]))
    if op == "experts":
        groups = rng.choice([1, 4, 8, 16, 27, 64, 128])
        rows = _log(rng, 1, 40_000)
        # (an fp32 product takes some eight times as long)
        most = 1.0e12 if dtype != "float32" else 1.2e11
        ci, co = (rng.choice([32, 64, 100, 256, 520, 1024, 2048]) for _ in range(2))
        rows = min(rows, max(1, int(most / (4 * ci * co))))
        return dict(op=op, direction=rng.choice(["forward", "backward"]), dtype=dtype, rows=rows, groups=groups,
                    active=max(1, min(groups, rows) - rng.choice([0, 0, 1, 3])), ci=ci, co=co,
                    skew=rng.choice([0.0, 0.5, 1.5]))
    bits = rng.choice([32, 8])
    tensors = _log(rng, 1, 300)
    return dict(op=op, dtype=dtype, master=dtype != "float32" and rng.random() < 0.5, bits=bits, tensors=tensors,
                total=max(_log(rng, 1000, 100_000_000), 2 * tensors), step=rng.choice([1, 2, 50, 10_000]))


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


def _tokens(case, g):
    """Tokens whose frequencies fall like rank ** -skew, ranks strewn over the table; a share of them names no row."""
    n, rows = case["tokens"], case["rows"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    skew = case["skew"]
    if skew == 1.0:
        rank = torch.exp(u * math.log(rows + 1.0)) - 1.0
    else:
        top = (rows + 1.0) ** (1.0 - skew)
        rank = (1.0 + u * (top - 1.0)) ** (1.0 / (1.0 - skew)) - 1.0
    place = torch.randperm(rows, generator=g, device="cuda")
    tokens = place[rank.long().clamp_(0, rows - 1)]
    gone = torch.rand(n, generator=g, device="cuda") < case["outside"]
    return torch.where(gone, torch.full_like(tokens, -1), tokens).to(torch.int32)


def _adamw_sizes(case):
    """Elements of every tensor: from biases to filters, odd ones among them."""
    rng = random.Random(case["tensors"] * 1_000_003 + case["total"])
    return _split(case["total"], case["tensors"], 1.5, rng)


def _package():
    path = os.path.join("mlu-ops_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mluop_hip
    return mluop_hip


def prepare(case, seed):
    g, rng = _generator(seed), random.Random(seed)
    op, s = case["op"], {"case": case}
    if op == "embedding":
        s["tokens"] = _tokens(case, g)
        s["scale"] = math.sqrt(case["channels"])
        if case["direction"] == "forward":
            s["table"] = _randn(g, (case["rows"], case["channels"]), case["dtype"], 0.02)
        else:
            s["output_grad"] = _randn(g, (case["tokens"], case["channels"]), case["dtype"])
    elif op == "norm":
        rows, channels, samples, groups = case["rows"], case["channels"], case["samples"], case["groups"]
        s["host_starts"] = _starts(_split(rows, samples, 0.4, rng))
        s["row_starts"] = torch.tensor(s["host_starts"], dtype=torch.int32, device="cuda")
        # (channels lie off zero by different amounts, as they do behind a layer)
        s["features"] = (torch.randn((rows, channels), generator=g, device="cuda") +
                         2.0 * torch.randn(channels, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
        s["weight"] = (1.0 + 0.2 * torch.randn(channels, generator=g, device="cuda")).to(DTYPES[case["params"]])
        s["bias"] = (0.2 * torch.randn(channels, generator=g, device="cuda")).to(DTYPES[case["params"]])
        if case["direction"] == "backward":
            s["output_grad"] = _randn(g, (rows, channels), case["dtype"])
            s["mean"], s["rstd"] = _moments(s["features"].float(), _members(s), groups)
    elif op == "experts":
        sizes = [0] * case["groups"]
        for group, n in zip(rng.sample(range(case["groups"]), case["active"]),
                            _split(case["rows"], case["active"], case["skew"], rng)):
            sizes[group] = n
        s["host_starts"] = _starts(sizes)
        s["group_starts"] = torch.tensor(s["host_starts"], dtype=torch.int32, device="cuda")
        s["features"] = _randn(g, (case["rows"], case["ci"]), case["dtype"])
        s["filters"] = _randn(g, (case["groups"], case["ci"], case["co"]), case["dtype"], case["ci"] ** -0.5)
        if case["direction"] == "backward":
            s["output_grad"] = _randn(g, (case["rows"], case["co"]), case["dtype"])
    else:
        _prepare_adamw(s, case, g)
    if own:
        package = _package()
        s["handle"] = package.make_handle_on_current_stream()
        if op == "adamw":
            s["plan"] = package.AdamWTensors(*_adamw_lists(s))
    return s


def _prepare_adamw(s, case, g):
    """Parameters, gradients and states as views of flat buffers, every tensor at a multiple of a state block; what lies
    between two tensors is zero in all of them."""
    sizes = _adamw_sizes(case)
    blocks = [-(-n // BLOCK) for n in sizes]
    places = [b * BLOCK for b in _starts(blocks)]
    total = places[-1]
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    for at, n in zip(places, sizes):
        inside[at:at + n] = True

    def values(scale):
        return torch.randn(total, generator=g, device="cuda").mul_(scale).mul_(inside)

    s["sizes"], s["places"], s["blocks"] = sizes, places, blocks
    master = values(0.05)
    s["param"] = master.to(DTYPES[case["dtype"]])
    s["master"] = master if case["master"] else None
    # (elements of one tensor have gradients of very different sizes)
    size = torch.exp(1.5 * torch.randn(total, generator=g, device="cuda"))
    s["grad"] = values(1e-3).mul_(size).to(DTYPES[case["dtype"]])
    m, r = values(5e-4).mul_(size), values(1e-3).abs_().mul_(size)
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _to_codes(m, False)
        s["v"], s["v_scale"] = _to_codes(r, True)
    else:
        s["m"], s["v"] = m, r.square_()


def _adamw_lists(s):
    """What a program hands over: a list of tensors of each kind."""
    def cut(flat):
        return None if flat is None else [flat[at:at + n] for at, n in zip(s["places"], s["sizes"])]

    def scales(flat):
        return None if flat is None else [flat[at // BLOCK:at // BLOCK + b] for at, b in zip(s["places"], s["blocks"])]

    s["grads"] = cut(s["grad"])
    return (cut(s["param"]), cut(s["m"]), cut(s["v"]), cut(s["master"]), scales(s.get("m_scale")), scales(s.get("v_scale")))


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return (_RUN_OWN if own else _RUN_PLAIN)[case["op"]](state, case)


def _embedding_plain(s, case):
    tokens, scale = s["tokens"].long(), s["scale"]
    if case["direction"] == "forward":
        found = s["table"][tokens.clamp(min=0)].float() * scale
        return torch.where((tokens >= 0).unsqueeze(1), found, torch.zeros((), device="cuda")).to(s["table"].dtype)
    grad = s["output_grad"]
    # (one row more takes what names no row)
    table = torch.zeros((case["rows"] + 1, case["channels"]), device="cuda")
    table.index_add_(0, torch.where(tokens >= 0, tokens, torch.full_like(tokens, case["rows"])), grad.float())
    return (table[:case["rows"]] * scale).to(grad.dtype)


def _embedding_own(s, case):
    package = _package()
    if case["direction"] == "forward":
        return package.embedding_forward(s["handle"], s["table"], s["tokens"], s["scale"])
    return package.embedding_backward(s["handle"], s["output_grad"], s["tokens"], case["rows"], s["scale"])


def _members(s):
    """float [samples, rows]: which rows are a sample's; sums over samples are products with it."""
    starts = s["row_starts"].long()
    row = torch.arange(s["features"].shape[0], device="cuda")
    return ((row >= starts[:-1, None]) & (row < starts[1:, None])).float()


def _moments(x, members, groups):
    rows, channels = x.shape
    count = (members.sum(dim=1, keepdim=True) * (channels // groups))
    x = x.view(rows, groups, channels // groups)
    mean = members @ x.sum(dim=2) / count
    off = x - (members.t() @ mean).unsqueeze(2)
    var = members @ (off * off).sum(dim=2) / count
    return mean, torch.rsqrt(var + EPS)


def _norm_plain(s, case):
    groups, act = case["groups"], case["activation"]
    x, w, b = s["features"].float(), s["weight"].float(), s["bias"].float()
    rows, channels = x.shape
    members = _members(s)
    of_row = members.t()
    mean, rstd = (s["mean"], s["rstd"]) if case["direction"] == "backward" else _moments(x, members, groups)
    r = (of_row @ rstd).unsqueeze(2)
    xhat = ((x.view(rows, groups, -1) - (of_row @ mean).unsqueeze(2)) * r).view(rows, channels)
    z = xhat * w + b
    if case["direction"] == "forward":
        y = torch.relu(z) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z
        return y.to(s["features"].dtype), mean, rstd
    dz = s["output_grad"].float()
    if act == "relu":
        dz = dz * (z > 0)
    elif act == "silu":
        t = torch.sigmoid(z)
        dz = dz * (t * (1.0 + z * (1.0 - t)))
    dw, db = (dz * xhat).sum(dim=0), dz.sum(dim=0)
    d = (dz * w).view(rows, groups, -1)
    xhat = xhat.view(rows, groups, -1)
    count = members.sum(dim=1, keepdim=True) * (channels // groups)
    s1 = (of_row @ (members @ d.sum(dim=2) / count)).unsqueeze(2)
    s2 = (of_row @ (members @ (d * xhat).sum(dim=2) / count)).unsqueeze(2)
    dx = (r * (d - s1 - xhat * s2)).view(rows, channels)
    return dx.to(s["features"].dtype), dw.to(s["weight"].dtype), db.to(s["bias"].dtype)


def _norm_own(s, case):
    package = _package()
    if case["direction"] == "forward":
        return package.group_norm_forward(s["handle"], s["features"], s["weight"], s["bias"], case["groups"],
                                          s["row_starts"], EPS, case["activation"])
    return package.group_norm_backward(s["handle"], s["output_grad"], s["features"], s["weight"], s["bias"], s["mean"],
                                       s["rstd"], case["groups"], s["row_starts"], case["activation"])


def _experts_plain(s, case):
    # One product for each expert that has rows, on sizes that the host knows: the plain form with the least work
    # (all at once would be products of padded sizes).
    starts, x, w = s["host_starts"], s["features"], s["filters"]
    spans = [(k, a, b) for k, (a, b) in enumerate(zip(starts, starts[1:])) if b > a]
    if case["direction"] == "forward":
        return torch.cat([x[a:b].float() @ w[k].float() for k, a, b in spans]).to(x.dtype)
    dy = s["output_grad"]
    dx = torch.cat([dy[a:b].float() @ w[k].float().t() for k, a, b in spans])
    dw = torch.zeros(w.shape, device="cuda")
    for k, a, b in spans:
        torch.mm(x[a:b].float().t(), dy[a:b].float(), out=dw[k])
    return dx.to(x.dtype), dw.to(w.dtype)


def _experts_own(s, case):
    package = _package()
    if case["direction"] == "forward":
        return package.grouped_matmul_forward(s["handle"], s["features"], s["filters"], s["group_starts"])
    return (package.grouped_matmul_backward_data(s["handle"], s["output_grad"], s["filters"], s["group_starts"]),
            package.grouped_matmul_backward_filter(s["handle"], s["features"], s["output_grad"], s["group_starts"]))


def _to_codes(x, keep_from_zero):
    """Blocks of 256 values as e4m3 with one fp32 scale each; a root that is not zero does not become zero."""
    x = x.view(-1, BLOCK)
    most = x.abs().amax(dim=1, keepdim=True)
    q = (x * torch.where(most > 1e-30, E4M3_MAX / most, torch.zeros_like(most))).to(torch.float8_e4m3fn)
    if keep_from_zero:
        f = q.float()
        q = torch.where((f == 0) & (x > 0), torch.full_like(f, E4M3_LEAST), f).to(torch.float8_e4m3fn)
    return q.view(-1), most.view(-1) * (1.0 / E4M3_MAX)


def _from_codes(q, scale):
    return (q.float().view(-1, BLOCK) * scale.unsqueeze(1)).view(-1)


def _adamw_plain(s, case):
    h, step, eight = ADAMW, case["step"], case["bits"] == 8
    g = s["grad"].float()
    m = (_from_codes(s["m"], s["m_scale"]) if eight else s["m"]) * h["beta1"] + g * (1.0 - h["beta1"])
    v = _from_codes(s["v"], s["v_scale"]).square() if eight else s["v"]
    root = torch.sqrt(v * h["beta2"] + g * g * (1.0 - h["beta2"]))
    v = None if eight else v * h["beta2"] + g * g * (1.0 - h["beta2"])
    c1, c2 = 1.0 - h["beta1"] ** step, math.sqrt(1.0 - h["beta2"] ** step)
    p = (s["param"] if s["master"] is None else s["master"]).float()
    p = p * (1.0 - h["lr"] * h["weight_decay"]) - (h["lr"] / c1) * (m / (root * (1.0 / c2) + h["eps"]))
    s["param"].copy_(p)
    if s["master"] is not None:
        s["master"].copy_(p)
    if eight:
        (s["m"], s["m_scale"]), (s["v"], s["v_scale"]) = _to_codes(m, False), _to_codes(root, True)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _adamw_outputs(s)


def _adamw_own(s, case):
    s["plan"].step(s["handle"], s["grads"], case["step"], ADAMW["lr"], (ADAMW["beta1"], ADAMW["beta2"]), ADAMW["eps"],
                   ADAMW["weight_decay"])
    return _adamw_outputs(s)


def _adamw_outputs(s):
    return {k: s[k] for k in ("param", "master", "m", "v", "m_scale", "v_scale") if s.get(k) is not None}


_RUN_PLAIN = {"embedding": _embedding_plain, "norm": _norm_plain, "experts": _experts_plain, "adamw": _adamw_plain}
_RUN_OWN = {"embedding": _embedding_own, "norm": _norm_own, "experts": _experts_own, "adamw": _adamw_own}


# ---------------------------------------------------------------------------------------------
# Least work, and the definitions in 64 bits
# ---------------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "float32" else 2
    if op == "embedding":
        n, rows, channels = case["tokens"], case["rows"], case["channels"]
        # (of the table at most the rows that are named are read; of its gradient every row is written)
        table = min(n, rows) if case["direction"] == "forward" else rows
        return {"bytes": (n + table) * channels * size + 4 * n, "flops": n * channels}
    if op == "norm":
        values = case["rows"] * case["channels"]
        forward = case["direction"] == "forward"
        return {"bytes": values * size * (2 if forward else 3), "flops": values * (10 if forward else 25)}
    if op == "experts":
        rows, ci, co, forward = case["rows"], case["ci"], case["co"], case["direction"] == "forward"
        filters = case["active"] * ci * co
        if forward:
            return {"bytes": size * (rows * (ci + co) + filters), "flops": 2 * rows * ci * co}
        return {"bytes": size * (rows * (2 * ci + co) + filters + case["groups"] * ci * co), "flops": 4 * rows * ci * co}
    states = 4 * (1 + 1.0 / 64) if case["bits"] == 8 else 16
    params = 3 * size - (size if case["master"] else 0) + (8 if case["master"] else 0)
    return {"bytes": case["total"] * (params + states), "flops": 15 * case["total"]}


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return _EXACT[case["op"]](s, case)


def _embedding_exact(s, case):
    tokens = s["tokens"].long()
    named = tokens >= 0
    if case["direction"] == "forward":
        out = torch.zeros((tokens.shape[0], case["channels"]), dtype=torch.float64, device="cuda")
        out[named] = s["table"][tokens[named]].double() * s["scale"]
        return out
    # sums of sorted tokens: differences of running sums at the ends of each token's rows, a few channels at a time
    order = torch.argsort(tokens, stable=True)
    ends = torch.searchsorted(tokens[order], torch.arange(-1, case["rows"], device="cuda"), right=True)
    parts = []
    for c in range(0, case["channels"], 128):
        sums = torch.cumsum(s["output_grad"][order, c:c + 128].double() * s["scale"], dim=0)
        sums = torch.cat([torch.zeros_like(sums[:1]), sums])
        parts.append(sums[ends[1:]] - sums[ends[:-1]])
    return torch.cat(parts, dim=1)


def _norm_exact(s, case):
    groups, act, back = case["groups"], case["activation"], case["direction"] == "backward"
    w, b = s["weight"].double(), s["bias"].double()
    outs, means, rstds, dw, db = [], [], [], 0.0, 0.0
    for k, (lo, hi) in enumerate(zip(s["host_starts"], s["host_starts"][1:])):
        x = s["features"][lo:hi].double().unflatten(1, (groups, -1))
        if back:
            mean, rstd = s["mean"][k].double(), s["rstd"][k].double()
        else:
            mean = x.mean(dim=(0, 2))
            rstd = (x.var(dim=(0, 2), unbiased=False) + EPS) ** -0.5
        n = ((x - mean[None, :, None]) * rstd[None, :, None]).flatten(1)
        z = torch.addcmul(b, n, w)
        if not back:
            outs.append(z.clamp(min=0) if act == "relu" else z / (1.0 + torch.exp(-z)) if act == "silu" else z)
            means.append(mean)
            rstds.append(rstd)
            continue
        slope = torch.ones_like(z)
        if act == "relu":
            slope = torch.where(z > 0, 1.0, 0.0).double()
        elif act == "silu":
            e = torch.exp(-z)
            slope = 1.0 / (1.0 + e) + z * e / (1.0 + e) ** 2
        dz = s["output_grad"][lo:hi].double() * slope
        dw, db = dw + (dz * n).sum(0), db + dz.sum(0)
        d, n = (dz * w).unflatten(1, (groups, -1)), n.unflatten(1, (groups, -1))
        d = d - d.mean(dim=(0, 2), keepdim=True) - n * (d * n).mean(dim=(0, 2), keepdim=True)
        outs.append((d * rstd[None, :, None]).flatten(1))
    if back:
        return torch.cat(outs), dw, db
    return torch.cat(outs), torch.stack(means), torch.stack(rstds)


def _experts_exact(s, case):
    x, w = s["features"], s["filters"]
    first, last = s["host_starts"][:-1], s["host_starts"][1:]
    if case["direction"] == "forward":
        out = torch.empty((x.shape[0], case["co"]), dtype=torch.float64, device="cuda")
        for k, (lo, hi) in enumerate(zip(first, last)):
            out[lo:hi] = x[lo:hi].double() @ w[k].double()
        return out
    dy = s["output_grad"]
    dx = torch.empty((x.shape[0], case["ci"]), dtype=torch.float64, device="cuda")
    dw = torch.empty(w.shape, dtype=torch.float64, device="cuda")
    for k, (lo, hi) in enumerate(zip(first, last)):
        grad = dy[lo:hi].double()
        dx[lo:hi] = (w[k].double() @ grad.t()).t()
        dw[k] = (grad.t() @ x[lo:hi].double()).t()
    return dx, dw


def _adamw_exact(s, case):
    h, t, eight = ADAMW, case["step"], case["bits"] == 8
    g = s["grad"].double()

    def values(codes, scale):
        return codes.double() * scale.double().repeat_interleave(BLOCK)

    m = values(s["m"], s["m_scale"]) if eight else s["m"].double()
    v = values(s["v"], s["v_scale"]) ** 2 if eight else s["v"].double()
    m = m.lerp_(g, 1.0 - h["beta1"])
    v = v.lerp_(g ** 2, 1.0 - h["beta2"])
    del g
    p = (s["param"] if s["master"] is None else s["master"]).double()
    step = (m / (1.0 - h["beta1"] ** t)) / (torch.sqrt(v / (1.0 - h["beta2"] ** t)) + h["eps"])
    p = p - h["lr"] * (step + h["weight_decay"] * p)
    out = {"param": p}
    if s["master"] is not None:
        out["master"] = p
    if not eight:
        return {**out, "m": m, "v": v}
    for name, x in (("m", m), ("v", torch.sqrt(v))):
        # (a code has no 64-bit value: that of the number which it stands for, in units of its block's scale)
        scale = x.abs().view(-1, BLOCK).amax(dim=1) / E4M3_MAX
        unit = scale.repeat_interleave(BLOCK)
        out[name] = torch.where(unit > 0, x / unit, 0.0)
        out[name + "_scale"] = scale
    return out


_EXACT = {"embedding": _embedding_exact, "norm": _norm_exact, "experts": _experts_exact, "adamw": _adamw_exact}
