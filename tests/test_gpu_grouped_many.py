"""Filter gradients by expert of very many groups: more than the workgroups rank by length, in several rounds, and as many as have
no place in LDS (small whole numbers: sums are exact)."""
import pytest

from launches import launched

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups,rows,ci,co,kernel", [
    (255, 9000, 256, 512, "groupedTiles"), (256, 9000, 256, 512, "groupedTiles"), (257, 9000, 256, 512, "groupedTiles"),
    (300, 3000, 264, 520, "groupedTiles"), (1000, 20_000, 128, 256, "groupedTiles"), (2047, 9000, 64, 128, "groupedTiles"),
    (2048, 9000, 64, 128, "groupedAny"), (5000, 9000, 64, 64, "groupedAny")])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_products(gpu_handle, dtype, groups, rows, ci, co, kernel):
    import random
    import torch
    import mluop_hip
    print("grouped many", dtype, groups, rows, ci, co, flush=True)
    g = torch.Generator(device="cuda").manual_seed(groups)
    rng = random.Random(rows)
    dtype = getattr(torch, dtype)
    # a few long groups among many of a few rows or none
    starts = [0] + sorted([rng.randrange(rows + 1) for _ in range(groups // 2)] +
                          [rng.choice((rows // 2, rows // 3, rows - 1)) for _ in range(groups - 1 - groups // 2)]) + [rows]
    x = torch.randint(-2, 3, (rows, ci), device="cuda", generator=g).to(dtype)
    w = torch.randint(-1, 2, (groups, ci, co), device="cuda", generator=g).to(dtype)
    dy = torch.randint(-1, 2, (rows, co), device="cuda", generator=g).to(dtype)
    dev = torch.tensor(starts, dtype=torch.int32, device="cuda")
    y, dx, dw = torch.zeros(rows, co, device="cuda"), torch.zeros(rows, ci, device="cuda"), torch.zeros(w.shape, device="cuda")
    for k, (a, b) in enumerate(zip(starts, starts[1:])):
        if a < b:
            y[a:b] = x[a:b].float() @ w[k].float()
            dx[a:b] = dy[a:b].float() @ w[k].float().t().contiguous()
            dw[k] = x[a:b].float().t().contiguous() @ dy[a:b].float()
    assert torch.equal(mluop_hip.grouped_matmul_forward(gpu_handle, x, w, dev), y.to(dtype))
    assert torch.equal(mluop_hip.grouped_matmul_backward_data(gpu_handle, dy, w, dev), dx.to(dtype))
    got, names = launched(gpu_handle, lambda: mluop_hip.grouped_matmul_backward_filter(gpu_handle, x, dy, dev))
    assert torch.equal(got, dw.to(dtype)) and names[0].startswith(kernel), names
