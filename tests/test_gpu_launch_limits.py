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


@pytest.mark.parametrize("groups,channels,act", [(2, 8, "none"), (1, 3, "silu")])
def test_group_norm_of_very_many_samples(gpu_handle, groups, channels, act):
    """few rows in more samples than a grid has workgroups along y; most samples are empty"""
    import torch
    import mluop_hip
    rows, samples = 1000, 70_001
    g = torch.Generator(device="cuda").manual_seed(channels)
    x = torch.randn(rows, channels, device="cuda", generator=g)
    dy = torch.randn(rows, channels, device="cuda", generator=g)
    w = 1 + 0.3 * torch.randn(channels, device="cuda", generator=g)
    b = 0.3 * torch.randn(channels, device="cuda", generator=g)
    cuts = torch.randint(0, rows // 4, (samples - 1,), device="cuda", generator=g).sort().values * 4
    starts = torch.cat([torch.zeros_like(cuts[:1]), cuts, torch.full_like(cuts[:1], rows)]).to(torch.int32)
    filled = starts[1:] > starts[:-1]
    assert bool((starts[1:] - starts[:-1]).max() >= 4) and int(filled.sum()) > 100
    own = torch.cat([starts[:-1][filled], starts[-1:]])   # the same without samples of no rows
    out, mean, rstd = mluop_hip.group_norm_forward(gpu_handle, x, w, b, groups, starts, 1e-5, act)
    ref, ref_mean, ref_rstd = mluop_hip.group_norm_forward(gpu_handle, x, w, b, groups, own, 1e-5, act)
    # (few rows and samples, and what they are with many, may be added up by different kernels)
    assert torch.allclose(out, ref, atol=1e-4) and torch.allclose(mean[filled], ref_mean, atol=1e-5)
    assert torch.allclose(rstd[filled], ref_rstd, rtol=1e-4) and not bool(mean[~filled].any())
    assert torch.allclose(rstd[~filled], torch.tensor(1e-5 ** -0.5, device="cuda"))
    got = mluop_hip.group_norm_backward(gpu_handle, dy, x, w, b, mean, rstd, groups, starts, act)
    want = mluop_hip.group_norm_backward(gpu_handle, dy, x, w, b, ref_mean, ref_rstd, groups, own, act)
    for a, c in zip(got, want):
        assert torch.allclose(a, c, rtol=1e-3, atol=1e-3 * float(c.abs().max()))


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


def test_lookup_of_more_rows_than_a_launch(handle):
    """four tokens a workgroup: 2^26 of them"""
    import torch
    import mluop_hip
    room_for(24)
    n, channels = (1 << 26) + 1003, 129
    g = torch.Generator(device="cuda").manual_seed(3)
    table = torch.randn(50, channels, device="cuda", generator=g).to(torch.bfloat16)
    tokens = torch.randint(-1, 50, (n,), device="cuda", generator=g, dtype=torch.int32)
    out = mluop_hip.embedding_forward(handle, table, tokens)
    padded = torch.cat([table, torch.zeros_like(table[:1])])   # (-1: the last row)
    same = all(torch.equal(out[at:at + (1 << 22)], padded[tokens[at:at + (1 << 22)].long()]) for at in range(0, n, 1 << 22))
    assert same


@pytest.mark.parametrize("rows,tokens", [((1 << 24) + 77, 24 * ((1 << 24) + 77)),   # a row of the table a workgroup
                                         (30_000_000, (1 << 29) + 1001)])           # 2^24 pieces of 32 words
def test_gradient_of_more_rows_than_a_launch(handle, rows, tokens):
    import torch
    import mluop_hip
    room_for(40)
    g = torch.Generator(device="cuda").manual_seed(rows)
    t = torch.randint(0, rows, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    t[-5000:-1000], t[-1000:] = rows - 1, rows - 2   # rows longer than a piece, in the last pieces
    t[:3000] = 1
    grad = torch.randint(-2, 3, (tokens, 1), device="cuda", generator=g, dtype=torch.int8).to(torch.bfloat16)
    got = mluop_hip.embedding_backward(handle, grad, t, rows)
    want = torch.zeros(rows, device="cuda")
    for at in range(0, tokens, 1 << 27):
        want.index_add_(0, t[at:at + (1 << 27)], grad[at:at + (1 << 27), 0].float())
    same = torch.equal(got[:, 0], want.to(torch.bfloat16))
    assert same


def test_products_of_more_rows_than_a_launch(handle):
    """64 rows a workgroup: 2^30 of them"""
    import torch
    import mluop_hip
    room_for(16)
    rows = (1 << 30) + 5000
    x = torch.ones(rows, 1, dtype=torch.float16, device="cuda")
    x[1::2] = 3.0
    cut = (1 << 30) - 777
    starts = torch.tensor([0, cut, rows - 9], dtype=torch.int32, device="cuda")
    w = torch.tensor([2.0, -5.0], dtype=torch.float16, device="cuda").view(2, 1, 1)
    for call in (mluop_hip.grouped_matmul_forward, mluop_hip.grouped_matmul_backward_data):
        y = call(handle, x, w, starts)
        for lo, hi, by in ((0, cut, 2), (cut, rows - 9, -5), (rows - 9, rows, 0)):
            same = torch.equal(y[lo:hi], by * x[lo:hi])
            assert same, (lo, hi)
