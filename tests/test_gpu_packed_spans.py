"""Packed prompts whose launch is cut into key spans give the precision of one that is not: results do not depend on whether a
workspace was passed, nor on how the device cuts the prompts.

Inputs that leave the second product nothing to round: the queries are zero, so every score is 0, every probability is exactly
1 in the cache's type, and a row's result is the mean of the values it sees.  What is left of the tolerance of
tests/paged_helpers.py is the fp32 sums, (n + 8) 2^-23 A over n keys with A the mean of |v|, the weight and the division that
join the spans (a handful of fp32 roundings: in the + 8), and the rounding of the result itself, 2^-24 |o| for an fp32 ``o``.
Spans kept in 16 bits would be off by u A, u = 2^-8 in bfloat16 and 2^-11 in float16: at 1024 keys, where (n + 8) 2^-23 is
1.2e-4, 32 and 4 times the tolerance.  Then the same with random queries, a span's worth of probabilities to round, against
the tolerance of tests/test_gpu_query_rounding.py: no 16-bit rounding but that of the probabilities."""

import pytest
import torch

from paged_helpers import U16, attend64, causal_hidden

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def packed(gpu_device):
    from g4b_amd.kernels import packed

    return packed


def means64(v, lens, window, H):
    """Mean over the values each row sees, and of their magnitudes: [T, H, D] in 64 bits; and the number of keys [T]."""
    v = v.double().cpu()
    G = v.shape[1]
    out, mag, n = [], [], []
    start = 0
    for length in lens:
        x = v[start:start + length]
        hi = torch.arange(1, length + 1)
        lo = (hi - window).clamp(min=0) if window else torch.zeros_like(hi)
        for values, into in ((x, out), (x.abs(), mag)):
            c = torch.cat([torch.zeros(1, *x.shape[1:], dtype=torch.float64), values.cumsum(0)])
            into.append((c[hi] - c[lo]) / (hi - lo)[:, None, None])
        n.append(hi - lo)
        start += length
    return torch.cat(out).repeat_interleave(H // G, 1), torch.cat(mag).repeat_interleave(H // G, 1), torch.cat(n)


# one prompt whose spans differ in number from tile to tile, two unequal ones, and a window that begins inside a span
CASES = {128: [([2048], None), ([1700, 300], None), ([2400], 1900)], 256: [([1024], None), ([1100, 500], None), ([1300], 1000)]}
CASES[512] = CASES[256]


def was_cut(ws):
    """Whether rows of spans, which come first, were written into a workspace that held nothing but 0x7F."""
    return bool((ws[: ws.numel() // 2] != 0x7F).any())


@pytest.mark.parametrize("case", [0, 1, 2], ids=["one", "two", "window"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D,heads", [(128, (8, 2)), (256, (8, 2)), (256, (3, 3)), (512, (4, 1))], ids=str)
@pytest.mark.parametrize("unrounded", [False, True], ids=["rounded_q", "unrounded_q"])
def test_spans_lose_nothing(packed, case, dtype, D, heads, unrounded):
    (lens, window), (H, G) = CASES[D][case], heads
    T = sum(lens)
    gen = torch.Generator().manual_seed(T + D)
    q = torch.zeros(T, H, D, dtype=torch.float32, device="cuda")
    k = torch.randn(T, G, D, generator=gen).to(dtype).cuda()
    v = (1.0 + 0.1 * torch.randn(T, G, D, generator=gen)).to(dtype).cuda()
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0)], dtype=torch.int32, device="cuda")
    ref, mag, n = means64(v, lens, window, H)
    tol = (n + 8)[:, None, None] * 2.0**-23 * mag + 2.0**-24 * ref.abs()
    size = packed.packed_workspace_bytes(T, len(lens), H, G, D)
    assert size > 0
    for ws in (None, torch.full((size,), 0x7F, dtype=torch.uint8, device="cuda")):
        o = torch.full((T, H, D), 777.0, device="cuda")
        packed.packed_attention(q, k, v, o, cu, query_window=window, use_fp32_dot=unrounded, workspace=ws)
        torch.cuda.synchronize()
        # (at head dimension 128 a launch with an unrounded query has 256 places, of which 75 tiles of two kv heads take more than half)
        assert ws is None or was_cut(ws) == (not (D == 128 and unrounded and window))
        over = ((o.double().cpu() - ref).abs() / tol).max().item()
        assert over <= 1.0, f"{'whole' if ws is None else 'cut'}: {over:.2f} times the tolerance"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_rows_computed_again_lose_nothing(packed, dtype, D):
    """An infinity in the last value row, which only the last query sees: the rows beside it take the plain body, span by span."""
    T, H, G = 2048 if D == 128 else 1024, 8, 2
    gen = torch.Generator().manual_seed(D)
    q = torch.zeros(T, H, D, dtype=torch.float32, device="cuda")
    k = torch.randn(T, G, D, generator=gen).to(dtype).cuda()
    v = (1.0 + 0.1 * torch.randn(T, G, D, generator=gen)).to(dtype).cuda()
    ref, mag, n = means64(v, [T], None, H)
    v[-1, 0, 3] = float("inf")
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    o = torch.full((T, H, D), 777.0, device="cuda")
    ws = torch.full((packed.packed_workspace_bytes(T, 1, H, G, D),), 0x7F, dtype=torch.uint8, device="cuda")
    packed.packed_attention(q, k, v, o, cu, workspace=ws)
    torch.cuda.synchronize()
    assert was_cut(ws)
    tol = (n + 8)[:, None, None] * 2.0**-23 * mag + 2.0**-24 * ref.abs()
    over = ((o.double().cpu() - ref).abs() / tol)[:-1].max().item()
    assert over <= 1.0, f"{over:.2f} times the tolerance"
    assert bool(torch.isinf(o[-1, : H // G, 3]).all())


@pytest.mark.parametrize("case", [0, 1, 2], ids=["one", "two", "window"])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_spans_of_random_queries(packed, D, case):
    (lens, window), H, G = CASES[D][case], 8, 2
    T, dtype = sum(lens), torch.bfloat16
    gen = torch.Generator().manual_seed(D + case)
    q, k, v = ((torch.randn(T, n, D, generator=gen) + mean).to(dtype).cuda() for n, mean in ((H, 0), (G, 0), (G, 1)))
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0)], dtype=torch.int32, device="cuda")
    ws = torch.full((packed.packed_workspace_bytes(T, len(lens), H, G, D),), 0x7F, dtype=torch.uint8, device="cuda")
    o = torch.full((T, H, D), 777.0, device="cuda")
    packed.packed_attention(q, k, v, o, cu, scale=D**-0.5, query_window=window, workspace=ws)
    torch.cuda.synchronize()
    assert was_cut(ws)
    start = 0
    for n in lens:
        rows = slice(start, start + n)
        start += n
        for h in (0, H - 1):
            g = h * G // H
            ref, mag, qk = attend64(q[rows, h], k[rows, g], v[rows, g], causal_hidden(n, window), D**-0.5)
            rel = 2 * U16[dtype] + 2 * (D + 4) * 2.0**-24 * qk + (n + 8) * 2.0**-23
            tol = rel[:, None] * mag * 1.0001 + 2.0**-24 * ref.abs()
            over = ((o[rows, h].double().cpu() - ref).abs() / tol).max().item()
            assert over <= 1.0, f"head {h}: {over:.2f} times the tolerance"
