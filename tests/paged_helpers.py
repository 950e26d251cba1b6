"""References in 64 bits, tolerances and inputs of the tests of packed prompts and the paged cache.

Tolerance of an attention output, element by element.  With u the rounding of the 16-bit type that the probabilities are
multiplied in (``eps / 2``), A = sum_j p_j |v_j| / sum_j p_j and n keys:

* every probability is rounded once: at most u A in the numerator, and again u A through the sum of probabilities;
* partial results that are kept in 16 bits (a key split of a packed prompt) add one more u A;
* a score is off by at most d = (D + 4) 2^-24 scale sum |q| |k| (a dot product and its scaling in fp32), which moves a
  probability and the sum by a factor exp(+-d): 2 d A;
* fp32 sums over n keys and the exponential's last place: (n + 8) 2^-23 A;
* a query that is rounded to the cache's type moves a score by at most u scale sum |q| |k|: 2 of those times A, when it is;
* the result is rounded once to its own type: u_o |o|.
"""

from __future__ import annotations

import torch

U16 = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


def attend64(q, k, v, hidden, scale):
    """softmax(scale q k^T) v and the same with |v|, in 64 bits: q [n, D], k, v [m, D], hidden [n, m]; also sum |q| |k|.
    Rows that see nothing are zeros; hidden values take no part, whatever they are."""
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    hidden = hidden.cpu()
    unseen = hidden.all(0)
    k = k.masked_fill(unseen[:, None], 0.0)
    s = (q @ k.T * scale).masked_fill(hidden, -torch.inf)
    m = s.amax(-1, keepdim=True) if s.shape[1] else s.new_full((s.shape[0], 1), -torch.inf)
    p = torch.exp(s - m.masked_fill(m == -torch.inf, 0.0))
    p = p / p.sum(-1, keepdim=True).masked_fill(hidden.all(-1)[:, None], 1.0)
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    finite = torch.isfinite(v).all(-1)
    if bool(finite.all()):
        return p @ v, p @ v.abs(), (q.abs() @ k.abs().T * scale).masked_fill(hidden, 0.0).amax(-1) if k.shape[0] else out[:, 0]
    for i in range(q.shape[0]):  # (rows that see different keys: a hidden value must not take part as 0 * inf)
        seen = ~hidden[i]
        out[i] = p[i, seen] @ v[seen]
        mag[i] = p[i, seen] @ v[seen].abs()
    return out, mag, (q.abs() @ k.nan_to_num().abs().T * scale).masked_fill(hidden, 0.0).amax(-1)


def check_attention(got, ref, mag, qk, n_keys, D, kv_dtype, q_rounded=False, what=""):
    """got [n, D] against the reference's rows, inside the tolerance at the head of this file."""
    u, uo = U16[kv_dtype], U16[got.dtype]
    d = (D + 4) * 2.0**-24 * qk + (u * qk if q_rounded else 0.0)
    rel = 3 * u + 2 * d + (n_keys + 8) * 2.0**-23
    tol = rel[:, None] * mag * 1.0001 + uo * ref.abs() + 1e-30
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    over = ((got - ref).abs() / tol).max().item() if got.numel() else 0.0
    assert over <= 1.0, f"{what}: {over:.2f} times the tolerance"


def causal_hidden(n, window):
    i = torch.arange(n)
    hidden = i[None] > i[:, None]
    if window:
        hidden |= i[:, None] - i[None] >= window
    return hidden


def make_tables(lens, page_size, gen, extra=3, width=None, device="cuda"):
    """Block tables that hold ``lens`` positions, on pages in random order: (tables [S, M], number of pages)."""
    held = [-(-n // page_size) for n in lens]
    P = sum(held) + extra
    order = torch.randperm(P, generator=gen).tolist()
    M = width or max(max(held), 1)
    rows = [[order.pop() for _ in range(h)] + [-1] * (M - h) for h in held]
    return torch.tensor(rows, dtype=torch.int32, device=device).view(len(lens), M), P
