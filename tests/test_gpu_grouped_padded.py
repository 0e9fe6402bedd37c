"""Products by expert whose rows are no whole 16-byte pieces and long enough that padded copies are made of them, and filter
gradients of groups of very different lengths, some of which are cut into slices."""
import pytest

pytestmark = pytest.mark.gpu


def launched(handle, call):
    handle.set_kernel_timing(True)
    try:
        out = call()
        return out, [name for name, _ in handle.kernel_timings()]
    finally:
        handle.set_kernel_timing(False)


def whole_numbers(shape, low, high, dtype, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(low, high + 1, shape, device="cuda", generator=g).to(dtype)


def products(x, w, dy, starts):
    """small whole numbers: every sum is exact in fp32, and one rounding follows"""
    import torch
    y = torch.zeros(x.shape[0], w.shape[2], device="cuda")
    dx = torch.zeros(x.shape[0], w.shape[1], device="cuda")
    dw = torch.zeros(w.shape, device="cuda")
    for g, (a, b) in enumerate(zip(starts, starts[1:])):
        y[a:b] = x[a:b].float() @ w[g].float()
        dx[a:b] = dy[a:b].float() @ w[g].float().t().contiguous()
        dw[g] = x[a:b].float().t().contiguous() @ dy[a:b].float()
    assert max(float(v.abs().max()) for v in (y, dx, dw)) < 2 ** 24
    return y.to(x.dtype), dx.to(x.dtype), dw.to(x.dtype)


PADDED = [  # sizes of the groups, first row, rows behind, ci, co, which of the three products work on copies
    ([300, 0, 1500, 7, 900], 3, 5, 2048, 100, (1, 1, 1)),
    ([2000, 10, 0, 3000], 0, 1, 100, 1024, (1, 1, 1)),
    ([1], 0, 0, 1024, 100, (1, 0, 0)),
    ([0, 2, 0, 0, 1], 1, 0, 100, 2048, (0, 1, 0)),
    ([700, 900], 0, 0, 1001, 333, (1, 1, 0)),
]


@pytest.mark.parametrize("sizes,first,behind,ci,co,copied", PADDED)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_padded(gpu_handle, dtype, sizes, first, behind, ci, co, copied):
    import torch
    import mluop_hip
    print("grouped padded", dtype, sizes, ci, co, flush=True)
    t = getattr(torch, dtype)
    starts = [first]
    for n in sizes:
        starts.append(starts[-1] + n)
    rows = starts[-1] + behind
    x, w, dy = (whole_numbers((rows, ci), -2, 2, t, 1), whole_numbers((len(sizes), ci, co), -1, 1, t, 2),
                whole_numbers((rows, co), -1, 1, t, 3))
    want = products(x, w, dy, starts)
    # nothing of groups without rows and of rows of no group is looked at
    for g, n in enumerate(sizes):
        if n == 0:
            w[g] = float("nan")
    x[:first] = float("inf")
    dy[:first] = float("inf")
    x[starts[-1]:] = float("nan")
    dy[starts[-1]:] = float("nan")
    dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
    # (rows of a wider matrix, at any alignment)
    wide = torch.full((rows, ci + co + 5), 7.0, device="cuda").to(t)
    wide[:, 1:1 + ci], wide[:, ci + 4:ci + 4 + co] = x, dy
    calls = (lambda a, b: mluop_hip.grouped_matmul_forward(gpu_handle, a, w, dev),
             lambda a, b: mluop_hip.grouped_matmul_backward_data(gpu_handle, b, w, dev),
             lambda a, b: mluop_hip.grouped_matmul_backward_filter(gpu_handle, a, b, dev))
    for call, v, copies in zip(calls, want, copied):
        got, names = launched(gpu_handle, lambda: call(x, dy))
        # (fp32 rows of a multiple of four channels are whole)
        if dtype != "float32":
            assert ("groupedPad" in names or "groupedUnpad" in names) == bool(copies), names
        assert torch.equal(got, v)
        assert torch.equal(call(wide[:, 1:1 + ci], wide[:, ci + 4:ci + 4 + co]), v)


UNEVEN = [  # sizes of the groups, ci, co
    ([5000, 10, 0, 300, 64, 1, 900, 0], 256, 256), ([4000, 3, 700, 20], 2048, 264), ([9000, 1, 1, 1], 136, 72),
    ([10] * 60 + [3000] + [0] * 3, 512, 512), ([600] * 8 + [6000], 1024, 520), ([20000], 64, 128),
    ([17 * (k % 5) for k in range(90)] + [4000], 256, 512), ([3000, 0, 5, 2000], 100, 60),
]


@pytest.mark.parametrize("sizes,ci,co", UNEVEN)
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_uneven_groups(gpu_handle, dtype, sizes, ci, co):
    import torch
    import mluop_hip
    print("grouped uneven", dtype, len(sizes), max(sizes), ci, co, flush=True)
    t = getattr(torch, dtype)
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    x, dy = whole_numbers((starts[-1], ci), -2, 2, t, 4), whole_numbers((starts[-1], co), -1, 1, t, 5)
    dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
    got = mluop_hip.grouped_matmul_backward_filter(gpu_handle, x, dy, dev)
    again = mluop_hip.grouped_matmul_backward_filter(gpu_handle, x, dy, dev)
    assert torch.equal(got, again)
    for g, (a, b) in enumerate(zip(starts, starts[1:])):
        assert torch.equal(got[g], (x[a:b].float().t().contiguous() @ dy[a:b].float()).to(t)), g


@pytest.mark.parametrize("rows,ci,co", [(2500, 2048, 100), (6000, 100, 1024), (6000, 256, 512)])
def test_starts_that_make_no_sense(gpu_handle, rows, ci, co):
    """starts that overlap, fall or leave the rows: the calls end, and those after them are right"""
    import torch
    import mluop_hip
    x, w, dy = (whole_numbers((rows, ci), -1, 1, torch.float16, 6), whole_numbers((4, ci, co), -1, 1, torch.float16, 7),
                whole_numbers((rows, co), -1, 1, torch.float16, 8))
    for starts in ([-5, 2 * rows, 50, 10, 1000], [rows, 50, 20, 10, 0], [0, 1 << 30, -(1 << 30), 7, 7], [0, rows, 0, rows, 0]):
        dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
        assert mluop_hip.grouped_matmul_forward(gpu_handle, x, w, dev).shape == (rows, co)
        assert mluop_hip.grouped_matmul_backward_data(gpu_handle, dy, w, dev).shape == (rows, ci)
        assert mluop_hip.grouped_matmul_backward_filter(gpu_handle, x, dy, dev).shape == w.shape
    torch.cuda.synchronize()
    good = torch.tensor([0, 100, 100, 2000, rows], dtype=torch.int32, device="cuda")
    want = products(x, w, dy, good.tolist())
    assert torch.equal(mluop_hip.grouped_matmul_forward(gpu_handle, x, w, good), want[0])
    assert torch.equal(mluop_hip.grouped_matmul_backward_filter(gpu_handle, x, dy, good), want[2])


@pytest.mark.parametrize("sizes,behind", [([8448], 0), ([8192], 0), ([9000, 1], 0), ([4000, 300, 0, 4100], 100), ([8300, 900], 3)])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_a_last_round_that_is_nearly_empty(gpu_handle, dtype, sizes, behind):
    """tiles of 256 x 256 fill 256 CUs once and a little of a second time"""
    import torch
    import mluop_hip
    print("grouped rest", dtype, sizes, flush=True)
    t = getattr(torch, dtype)
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    rows, ci, co = starts[-1] + behind, 1032, 2048
    x, w, dy = (whole_numbers((rows, ci), -2, 2, t, 9), whole_numbers((len(sizes), ci, co), -1, 1, t, 10),
                whole_numbers((rows, co), -1, 1, t, 11))
    dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
    want = products(x, w, dy, starts)
    got, names = launched(gpu_handle, lambda: mluop_hip.grouped_matmul_forward(gpu_handle, x, w, dev))
    if dtype == "float16" and sizes == [8448]:
        assert names == ["groupedTiles256", "groupedRest"]
    assert torch.equal(got, want[0])
    assert torch.equal(mluop_hip.grouped_matmul_backward_data(gpu_handle, dy, w, dev), want[1])
