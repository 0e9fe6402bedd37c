"""The gradient of an embedding's table on both sides of every line between its ways to order the tokens (ranks, a sort of one
pass with few tiles or many, sorts of two and three passes), and rows whose words begin and end at all places of the pieces in
use: small whole numbers, so that every sum is exact in fp32."""
import pytest

from launches import launched

pytestmark = pytest.mark.gpu


def expected(grad, tokens, rows, scale):
    import torch
    named = (tokens >= 0) & (tokens < rows)
    out = torch.zeros(rows + 1, grad.shape[1], device="cuda")
    out.index_add_(0, torch.where(named, tokens, torch.full_like(tokens, rows)).long(), grad.float())
    assert float(out.abs().max()) < 2 ** 24
    return (out[:rows] * scale).to(grad.dtype)


# Ranks up to 4096 tokens where one pass of 10 bits would sort them (tables of up to 1023 rows), up to 12 288 where it takes more;
# a pass has few tiles up to 32 768 tokens.
LINES = ([(rows, tokens, tokens <= 4096) for rows in (517, 1023) for tokens in (4095, 4096, 4097, 32767, 32768, 32769, 120_000)] +
         [(rows, tokens, tokens <= 12_288) for rows in (1024, 70_000, (1 << 20) - 1, (1 << 20) + 5)
          for tokens in (12_287, 12_288, 12_289, 32_768, 32_769, 100_003)])


@pytest.mark.parametrize("rows,tokens,ranked", LINES)
@pytest.mark.parametrize("dtype,channels,wide", [("float32", 8, False), ("bfloat16", 33, True)])
def test_every_way_to_order_the_tokens(gpu_handle, dtype, channels, wide, rows, tokens, ranked):
    import torch
    import mluop_hip
    print("embedding order", dtype, channels, rows, tokens, flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows + tokens)
    # a third all over the table, a third a few rows, the ends of the table, some of no row
    t = torch.randint(0, rows, (tokens,), device="cuda", generator=g)
    pick = torch.rand(tokens, device="cuda", generator=g)
    t = torch.where(pick < 0.33, t % 5, t)
    t = torch.where((pick >= 0.33) & (pick < 0.4), rows - 1 - t % 3, t)
    t = torch.where(pick > 0.9, torch.where(pick > 0.95, rows, -1), t)
    t = t if wide else t.to(torch.int32)
    grad = torch.randint(-2, 3, (tokens, channels), device="cuda", generator=g).to(getattr(torch, dtype))
    got, names = launched(gpu_handle, lambda: mluop_hip.embedding_backward(gpu_handle, grad, t, rows, 0.5))
    assert torch.equal(got, expected(grad, t, rows, 0.5))
    assert names[0] == ("embeddingRankWords" if ranked else "embeddingSort")
    # (where one pass sorts, it leaves the rows' first words too)
    assert ("embeddingRowStarts" in names) == (ranked or rows >= 1024)


def lengths_around(p):
    """lengths of rows' runs in pieces of p words"""
    return [[p, p, p], [p + 1], [p - 1, p + 1, p, 1, 2 * p, 2 * p + 1], [1, p, 1, p, 3 * p + 8], [2 * p - 1, 1, p + 2],
            [p * 40 + 1, 1, 7 * p - 1], [p // 2, 3 * p // 2, p // 2, 3 * p // 2], [1] * p + [p + 1] + [1] * (p - 1),
            # long rows that begin with the first word of a later piece, and with its last
            [p, 2 * p + 3, 1], [2 * p, 5 * p, 1], [p // 2, p - p // 2, 3 * p], [p - 1, p + 1, p - 1, 3 * p], [3 * p - 1, 2 * p]]


@pytest.mark.parametrize("case", range(13))
@pytest.mark.parametrize("channels,shared,piece", [(40, True, 200), (8, True, 1024), (4, True, 2048), (512, True, 64),
                                                   (40, False, 32), (520, False, 32), (1024, False, 64), (1032, False, 64)])
def test_rows_around_the_pieces_in_use(gpu_handle, channels, shared, piece, case):
    """pieces are of 8 words for every row of threads where a workgroup shares a row (24 words a row or more, below 1024
    channels), else of 32 or 64"""
    import torch
    import mluop_hip
    lengths = lengths_around(piece)[case]
    print("embedding pieces", channels, shared, piece, case, flush=True)
    tokens = torch.arange(len(lengths), device="cuda").repeat_interleave(torch.tensor(lengths, device="cuda")).to(torch.int32)
    n = tokens.numel()
    rows = len(lengths) if shared else max(len(lengths) + 3, n // 24 + 1)
    if shared and n < 24 * rows:   # (rows of one word: more words of the last row)
        tokens = torch.cat([tokens, torch.full((24 * rows - n,), rows - 1, dtype=torch.int32, device="cuda")])
        n = tokens.numel()
    assert (n >= 24 * rows and channels < 1024) == shared
    g = torch.Generator(device="cuda").manual_seed(case)
    grad = torch.randint(-8, 9, (n, channels), device="cuda", generator=g).float()
    want = expected(grad, tokens, rows, 1.0)
    for order in (torch.arange(n, device="cuda"), torch.randperm(n, generator=g, device="cuda")):
        got = mluop_hip.embedding_backward(gpu_handle, grad[order].contiguous(), tokens[order].contiguous(), rows)
        assert torch.equal(got, want)
