"""A paged KV cache: attention of one new token per sequence over it, and the append that feeds it.

The reference's cache is one ring of rows per slot (``g4b/models/gemma4e.py:702-717``); here K and V live in pools of pages
``[P, G, page_size, D]`` (``page_size`` a multiple of 16) and ``block_tables[s, e]`` names the page that holds positions
``[e * page_size, (e + 1) * page_size)`` of sequence ``s``.  An entry outside ``[0, P)`` names no page: attention does not
see its positions and the append drops rows that would go there.  Entries past a sequence's length are never read.
:mod:`.pages` hands pages out and takes them back.
"""

from __future__ import annotations

import ctypes as C

from .. import _native
from . import utils as U


def _pools(k_pages, v_pages, G: int, D: int):
    """Checked pools ``[P, G, page_size, D]``: (dtype code, P, page_size, page strides)."""
    U.require_tensor(k_pages, "k_pages", 4)
    U.require_tensor(v_pages, "v_pages", 4)
    P, Gp, page_size, Dp = U.shape_of(k_pages)
    if U.shape_of(v_pages) != [P, Gp, page_size, Dp]:
        raise ValueError("k_pages and v_pages must have the same shape")
    if (Gp, Dp) != (G, D):
        raise ValueError(f"the pools {tuple(k_pages.shape)} must have G = {G} kv heads of D = {D}")
    dt = U.float_dtype_code(k_pages, "k_pages")
    if U.float_dtype_code(v_pages, "v_pages") != dt:
        raise ValueError("k_pages and v_pages must have the same dtype")
    strides = []
    for name, c in (("k_pages", k_pages), ("v_pages", v_pages)):
        s = U.strides_of(c)
        if s[3] != 1 or s[2] != D or s[1] != page_size * D:
            raise ValueError(f"{name} must be contiguous inside a page")
        # (the stride of a dimension of size one says nothing: a pool of one page is a page apart from nobody)
        strides.append(s[0] if P > 1 else max(s[0], G * page_size * D))
    return dt, P, page_size, strides


def _table(block_tables, rows: int):
    U.require_tensor(block_tables, "block_tables", 2)
    U.int_itemsize(block_tables, "block_tables", {"int32"})
    S, M = U.shape_of(block_tables)
    s = U.strides_of(block_tables)
    if S != rows:
        raise ValueError(f"block_tables must have one row per sequence ({rows}), got {S}")
    if M > 1 and s[1] != 1:
        raise ValueError("block_tables must have unit stride along its rows")
    return M, s[0]


def _per_sequence(t, what: str, n: int, dtype: str = "int32"):
    U.require_tensor(t, what, 1)
    U.int_itemsize(t, what, {dtype})
    if U.shape_of(t) != [n]:
        raise ValueError(f"{what} must have shape [{n}], got {tuple(t.shape)}")
    return t.data_ptr(), U.strides_of(t)[0]


def paged_workspace_bytes(B: int, H: int, G: int, D: int, num_workers: int = 0) -> int:
    """Bytes of scratch that let :func:`paged_attention` split the keys of ``B`` sequences over ``num_workers`` waves
    (0 = the library's default); 0 for shapes that never split."""
    return int(_native.load().g4b_paged_attn_workspace_bytes(B, H, G, D, num_workers))


def paged_attention(
    q, k_pages, v_pages, o, block_tables, seq_lens, user_phase=None, phase: int = 0, *, window_size: int | None = None,
    scale: float = 1.0, use_fp32_dot: bool = False, workspace=None, num_workers: int = 0, stream=None,
):
    """``o[b, h] = softmax(scale * q[b, h] . K_b^T) V_b``: one new token per sequence over the sequence's pages.

    * ``q``, ``o``: ``[B, H, D]`` (strided views allowed, unit stride in ``D``); ``block_tables``: ``[B, M]`` int32;
      ``seq_lens``: ``[B]`` int32, the new token included (append first): the query stands at position
      ``seq_lens[b] - 1``.  Lengths above ``M * page_size`` count as that, negative ones as 0.
    * ``user_phase`` / ``phase``: with ``user_phase`` (``[B]`` uint8) given, sequences whose phase differs are skipped and
      their rows of ``o`` stay untouched, as in :func:`.fa2.flash_attention`.
    * ``window_size``: only the last ``window_size`` positions are seen (a sliding-window layer); ``None``: all of them.
    * a sequence that sees no key (length 0, or nothing but absent pages) gets zeros.
    * ``scale``, ``use_fp32_dot``, ``num_workers``: as in :func:`.fa2.flash_attention`.  ``workspace``: a uint8 tensor of
      :func:`paged_workspace_bytes` bytes, used by one launch at a time; without it one wave reads all keys of a
      (sequence, kv head).

    Head dimensions 128, 256 and 512 with float16 / bfloat16 pools and up to 16 query heads per kv head take the streaming
    kernel; other multiples of 8 up to 1024, larger groups and float32 pools a plain fp32 kernel.
    """
    assert isinstance(phase, int)
    U.require_tensor(q, "q", 3)
    U.require_tensor(o, "o", 3)
    B, H, D = U.shape_of(q)
    if U.shape_of(o) != [B, H, D]:
        raise ValueError(f"o shape {tuple(o.shape)} must equal q shape {tuple(q.shape)}")
    U.require_tensor(k_pages, "k_pages", 4)
    G = U.shape_of(k_pages)[1]
    if G == 0 or H == 0 or H % G:
        raise ValueError("number of query heads must be a multiple of the number of kv heads")
    a = _native.PagedAttnArgs()
    a.kv_dtype, a.num_pages, a.page_size, (a.k_page_stride, a.v_page_stride) = _pools(k_pages, v_pages, G, D)
    a.max_pages, a.block_tables_stride = _table(block_tables, B)
    a.seq_lens, a.seq_lens_stride = _per_sequence(seq_lens, "seq_lens", B)
    if user_phase is not None:
        a.user_phase, a.user_phase_stride = _per_sequence(user_phase, "user_phase", B, "uint8")
    if window_size is not None and int(window_size) < 1:
        raise ValueError("window_size must be a positive int or None")
    a.q, a.k_pages, a.v_pages, a.o, a.block_tables = (t.data_ptr() for t in (q, k_pages, v_pages, o, block_tables))
    a.q_stride, a.o_stride = (U.row_strides(t) for t in (q, o))
    a.q_dtype, a.o_dtype = U.float_dtype_code(q, "q"), U.float_dtype_code(o, "o")
    a.B, a.H, a.G, a.D = B, H, G, D
    a.window_size = 0 if window_size is None else min(int(window_size), 0x7FFFFFFF)
    a.phase = phase
    a.num_workers = int(num_workers)
    a.use_fp32_dot = 1 if use_fp32_dot else 0
    a.scale = float(scale)
    a.workspace, a.workspace_bytes = U.workspace_of(workspace)
    U.require_one_gpu(q=q, k_pages=k_pages, v_pages=v_pages, o=o, block_tables=block_tables, seq_lens=seq_lens,
                      user_phase=user_phase, workspace=workspace)
    _native.check(_native.load().g4b_paged_attn(C.byref(a), U.stream_arg(stream)))
    return None


def add_kv_to_pages(
    k, v, k_pages, v_pages, block_tables, cache_offsets, rmsnorm_eps: float, k_rsos=None, v_rsos=None, user_phase=None,
    phase: int = 0, *, cu_seqlens=None, stream=None,
):
    """New K and V rows into their pages, the paged counterpart of two :func:`.add_kv_to_cache.add_kv_to_cache` calls.

    ``k``, ``v``: ``[T, G, D]`` strided views.  Sequence ``s`` brings rows ``cu_seqlens[s] .. cu_seqlens[s + 1] - 1``
    (``[N + 1]`` int32), or, without ``cu_seqlens``, the one row ``s``; they go to positions ``cache_offsets[s]``,
    ``cache_offsets[s] + 1``, ... (``[N]`` int32).  ``k_rsos`` / ``v_rsos``: optional ``[T, G]`` fp32 row sums of squares
    that turn the copy into the weightless RMSNorm ``x * rsqrt(rsos / D + rmsnorm_eps)``
    (``add_kv_to_cache.py:148-151``).  With ``user_phase`` (``[N]`` uint8) given, sequences whose phase differs from
    ``phase`` are skipped.  Rows that fall outside the table or on an absent page are dropped.
    """
    assert isinstance(phase, int)
    U.require_tensor(k, "k", 3)
    U.require_tensor(v, "v", 3)
    T, G, D = U.shape_of(k)
    if U.shape_of(v) != [T, G, D]:
        raise ValueError(f"v shape {tuple(v.shape)} must equal k shape {tuple(k.shape)}")
    a = _native.PagedAppendArgs()
    a.cache_dtype, a.num_pages, a.page_size, (a.k_page_stride, a.v_page_stride) = _pools(k_pages, v_pages, G, D)
    U.require_tensor(cache_offsets, "cache_offsets", 1)
    N = U.shape_of(cache_offsets)[0]
    a.cache_offsets, a.cache_offsets_stride = _per_sequence(cache_offsets, "cache_offsets", N)
    a.max_pages, a.block_tables_stride = _table(block_tables, N)
    if cu_seqlens is not None:
        a.cu_seqlens, a.cu_seqlens_stride = _per_sequence(cu_seqlens, "cu_seqlens", N + 1)
    elif T != N:
        raise ValueError(f"without cu_seqlens every sequence brings one row: got {T} rows and {N} sequences")
    for name, t in (("k_rsos", k_rsos), ("v_rsos", v_rsos)):
        if t is None:
            continue
        U.require_tensor(t, name, 2)
        if U.shape_of(t) != [T, G]:
            raise ValueError(f"{name} must have shape {[T, G]}, got {tuple(t.shape)}")
        if U.float_dtype_code(t, name) != _native.DT_F32:
            raise ValueError(f"{name} must be float32")
        setattr(a, name, t.data_ptr())
        setattr(a, name + "_stride", (C.c_int64 * 2)(*U.strides_of(t)))
    if user_phase is not None:
        a.user_phase, a.user_phase_stride = _per_sequence(user_phase, "user_phase", N, "uint8")
    a.k, a.v, a.k_pages, a.v_pages, a.block_tables = (t.data_ptr() for t in (k, v, k_pages, v_pages, block_tables))
    a.k_stride, a.v_stride = (U.row_strides(t) for t in (k, v))
    a.k_dtype, a.v_dtype = U.float_dtype_code(k, "k"), U.float_dtype_code(v, "v")
    a.T, a.N, a.G, a.D = T, N, G, D
    a.phase = phase
    a.rmsnorm_eps = float(rmsnorm_eps)
    U.require_one_gpu(k=k, v=v, k_pages=k_pages, v_pages=v_pages, block_tables=block_tables, cache_offsets=cache_offsets,
                      cu_seqlens=cu_seqlens, k_rsos=k_rsos, v_rsos=v_rsos, user_phase=user_phase)
    _native.check(_native.load().g4b_paged_append(C.byref(a), U.stream_arg(stream)))
    return None
