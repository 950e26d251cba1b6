"""``use_fp32_dot`` over packed prompts and pages: with it the scores are those of the query as it was passed, without it those
of the query rounded once to the cache's type.

Inputs that make the difference plain and everything else exact.  A query's elements are 256 + r with r a multiple of a power
of two in [-1, 1), representable in the query's type; the keys' elements are -1, 0 and 1, equal numbers of each sign in a
row, so the 256 cancels and a score is sum r k.  All products and sums are multiples of 1/8 (1/4 for a float16 query) below
2^17, which fp32 holds exactly in any order, and the two 16-bit operands that an unrounded query is split into (a multiple of
the type's step at 256 and a remainder of four bits) hold it exactly.  What is left of a score's error is its scaling, two
fp32 roundings of a score of at most qk' = scale sum |r| |k|; the rest of the tolerance is that of tests/paged_helpers.py with
the probabilities' rounding (2 u A: the sum and the numerator) and no other 16-bit one.  Rounding the query moves r by up to
half of the type's step at 256 (1/8 in float16, 1 in bfloat16) and thus the scores by more than 0.1.

A float16 probability below 2^-14 is rounded to a multiple of 2^-24, so by up to 2^-25 whatever its size: the largest of a row
is at least 1 in the units that the kernels round in, so the row's sum is, and n of them move the numerator by at most
2^-25 sum |v| and, through the sum, the result by 2^-25 n |o|.  It shows where one key has nearly all of the weight and an
element of its value row is next to zero: with 31 keys, p = 1 at v = -1.9e-5 and 7.4e-6 at the next, p rounded on the CPU
gives 1.2e-7 of error against 2 u A = 1.9e-8."""

import pytest
import torch

from paged_helpers import U16, attend64, causal_hidden, make_tables

pytestmark = pytest.mark.gpu

TYPES = [(torch.float32, torch.float16), (torch.float32, torch.bfloat16), (torch.float16, torch.bfloat16)]
SCALE = 0.5


def queries(n, H, D, q_dtype, gen):
    step = 8 if q_dtype == torch.float32 else 4
    r = torch.randint(-step, step, (n, H, D), generator=gen).float() / step
    q = (256.0 + r).to(q_dtype)
    assert bool((q.float() - 256.0 == r).all())
    return q


def keys(shape, dtype, gen):
    half = torch.randint(-1, 2, (*shape[:-1], shape[-1] // 2), generator=gen).float()
    return torch.cat([half, -half], -1).to(dtype)


def worst(got, q, k, v, hidden, dtype):
    """The largest error of got [n, D] in units of the tolerance, against rows q [n, D] in 64 bits."""
    ref, mag, _ = attend64(q, k, v, hidden, SCALE)
    r = q.double().cpu() - 256.0
    qk = (r.abs() @ k.double().cpu().abs().T * SCALE).masked_fill(hidden.cpu(), 0.0).amax(-1)
    n = hidden.shape[1]
    rel = 2 * U16[dtype] + 2 * (2 * 2.0**-23) * qk + (n + 8) * 2.0**-23
    tol = rel[:, None] * mag * 1.0001 + U16[got.dtype] * ref.abs() + 1e-30
    if dtype == torch.float16:
        seen = (~hidden.cpu()).double()
        tol = tol + 2.0**-25 * (seen @ v.double().cpu().abs() + seen.sum(-1, keepdim=True) * ref.abs())
    return ((got.double().cpu() - ref).abs() / tol).max().item()


def judge(fp32_dot, got, q, k, v, hidden, dtype, what):
    as_passed, rounded = worst(got, q, k, v, hidden, dtype), worst(got, q.to(dtype), k, v, hidden, dtype)
    want, other = (as_passed, rounded) if fp32_dot else (rounded, as_passed)
    assert want <= 1.0, f"{what}: {want:.2f} times the tolerance"
    return other


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("heads", [(8, 2), (2, 2), (32, 2)], ids=str)
@pytest.mark.parametrize("q_dtype,dtype", TYPES, ids=str)
@pytest.mark.parametrize("fp32_dot", [False, True])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
def test_packed_prompts(gpu_device, D, heads, q_dtype, dtype, fp32_dot, ws):
    from g4b_amd.kernels import packed

    H, G = heads
    lens = [65, 1600 if D == 128 else 640] if ws else [65, 150]
    T = sum(lens)
    gen = torch.Generator().manual_seed(D + H)
    q = queries(T, H, D, q_dtype, gen).cuda()
    k, v = keys((T, G, D), dtype, gen).cuda(), torch.randn(T, G, D, generator=gen).to(dtype).cuda()
    o = torch.full((T, H, D), 777.0, device="cuda")
    cu = torch.tensor([0, lens[0], T], dtype=torch.int32, device="cuda")
    n = packed.packed_workspace_bytes(T, 2, H, G, D) if ws else 0
    w = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda") if n else None
    packed.packed_attention(q, k, v, o, cu, scale=SCALE, use_fp32_dot=fp32_dot, workspace=w)
    torch.cuda.synchronize()
    for a, b in ((0, lens[0]), (lens[0], T)):
        hidden = causal_hidden(b - a, None)
        other = max(judge(fp32_dot, o[a:b, h], q[a:b, h], k[a:b, h * G // H], v[a:b, h * G // H], hidden, dtype, f"rows {a}.. head {h}")
                    for h in (0, H - 1))
        assert other > 4.0, "the two readings of the query cannot be told apart"


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("heads", [(8, 2), (16, 2), (32, 2)], ids=str)
@pytest.mark.parametrize("q_dtype,dtype", TYPES, ids=str)
@pytest.mark.parametrize("fp32_dot", [False, True])
@pytest.mark.parametrize("window", [None, 300], ids=["all", "window"])
def test_pages(gpu_device, D, heads, q_dtype, dtype, fp32_dot, window):
    from g4b_amd.kernels import paged

    H, G = heads
    lens, page = [2100, 333, 64], 16
    gen = torch.Generator().manual_seed(D + H)
    tables, P = make_tables(lens, page, gen)
    q = queries(len(lens), H, D, q_dtype, gen).cuda()
    kp, vp = keys((P, G, page, D), dtype, gen).cuda(), torch.randn(P, G, page, D, generator=gen).to(dtype).cuda()
    len_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    size = paged.paged_workspace_bytes(len(lens), H, G, D)
    for ws in (None, torch.full((size,), 0x7F, dtype=torch.uint8, device="cuda")):
        o = torch.full((len(lens), H, D), 777.0, device="cuda")
        paged.paged_attention(q, kp, vp, o, tables, len_t, window_size=window, scale=SCALE, use_fp32_dot=fp32_dot, workspace=ws)
        torch.cuda.synchronize()
        for b, n in enumerate(lens):
            lo = max(0, n - window) if window else 0
            at = tables[b].long().repeat_interleave(page)[lo:n]
            row = torch.arange(lo, n, device="cuda") % page
            hidden = torch.zeros(H // G, n - lo, dtype=torch.bool)
            other = 0.0
            for g in range(G):
                hs = slice(g * (H // G), (g + 1) * (H // G))
                other = max(other, judge(fp32_dot, o[b, hs], q[b, hs], kp[at, g, row], vp[at, g, row], hidden, dtype, f"sequence {b} head {g}"))
            assert other > 4.0, "the two readings of the query cannot be told apart"


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("q_dtype,dtype", TYPES, ids=str)
@pytest.mark.parametrize("fp32_dot", [False, True])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
def test_packed_rows_beside_an_infinity(gpu_device, D, q_dtype, dtype, fp32_dot, ws):
    """An infinity that only the prompt's last row sees does not change how the queries of the other rows are read."""
    from g4b_amd.kernels import packed

    H, G, T = 8, 2, (1600 if D == 128 else 800) if ws else 150
    gen = torch.Generator().manual_seed(D)
    q = queries(T, H, D, q_dtype, gen).cuda()
    k, v = keys((T, G, D), dtype, gen).cuda(), torch.randn(T, G, D, generator=gen).to(dtype).cuda()
    v[T - 1] = float("inf")
    o = torch.full((T, H, D), 777.0, device="cuda")
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    n = packed.packed_workspace_bytes(T, 1, H, G, D) if ws else 0
    w = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda") if n else None
    packed.packed_attention(q, k, v, o, cu, scale=SCALE, use_fp32_dot=fp32_dot, workspace=w)
    torch.cuda.synchronize()
    rows = slice(T - 8, T - 1)  # of the last row's tile: 16 tokens in the smallest
    hidden = causal_hidden(T, None)[rows, :T - 1]
    other = max(judge(fp32_dot, o[rows, h], q[rows, h], k[:T - 1, h * G // H], v[:T - 1, h * G // H], hidden, dtype, f"head {h}") for h in range(H))
    assert other > 4.0, "the two readings of the query cannot be told apart"
