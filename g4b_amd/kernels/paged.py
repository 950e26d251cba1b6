"""A paged KV cache: attention of one new token per sequence over it, and the append that feeds it.

The reference's cache is one ring of rows per slot (``g4b/models/gemma4e.py:702-717``); here K and V live in pools of pages
``[P, G, page_size, D]`` (``page_size`` a multiple of 16) and ``block_tables[s, e]`` names the page that holds positions
``[e * page_size, (e + 1) * page_size)`` of sequence ``s``.  An entry outside ``[0, P)`` names no page: attention does not
see its positions and the append drops rows that would go there.  Entries past a sequence's length are never read.
:mod:`.pages` hands pages out and takes them back.
"""

from __future__ import annotations

from .. import _native
from . import utils as U


def _pools(k_pages, v_pages, D: int):
    """Checked pools ``[P, G, page_size, D]``: (K pointer, V pointer, dtype code, P, G, page_size, K and V page stride)."""
    k_ptr, ks, k_st, dt = U.float_meta(k_pages, "k_pages", 4)
    v_ptr, vs, v_st, v_dt = U.float_meta(v_pages, "v_pages", 4)
    if ks != vs:
        raise ValueError("k_pages and v_pages must have the same shape")
    P, G, page_size, Dp = ks
    if Dp != D:
        raise ValueError(f"the pools {tuple(ks)} must have rows of D = {D}")
    if v_dt != dt:
        raise ValueError("k_pages and v_pages must have the same dtype")
    inside = (page_size * D, D, 1)
    if k_st[1:] != inside or v_st[1:] != inside:
        for name, st in (("k_pages", tuple(k_st)), ("v_pages", tuple(v_st))):
            if st[3] != 1 or st[2] != D or (G > 1 and st[1] != page_size * D):
                raise ValueError(f"{name} must be contiguous inside a page")
    k_stride, v_stride = k_st[0], v_st[0]
    if P == 1:  # (the stride of a dimension of size one says nothing)
        k_stride = v_stride = G * page_size * D
    return k_ptr, v_ptr, dt, P, G, page_size, k_stride, v_stride


def _table(block_tables, rows: int):
    ptr, (S, M), stride, code = U.meta(block_tables, "block_tables", 2)
    if code != "int32":
        raise ValueError(f"block_tables: dtype must be int32, got {U.dtype_name(block_tables)}")
    if S != rows:
        raise ValueError(f"block_tables must have one row per sequence ({rows}), got {S}")
    if M > 1 and stride[1] != 1:
        raise ValueError("block_tables must have unit stride along its rows")
    return ptr, M, stride[0]


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
    * a sequence that sees no key (length 0, or nothing but absent pages), or none with a score above minus infinity, gets zeros.
    * ``scale``, ``use_fp32_dot``, ``num_workers``: as in :func:`.fa2.flash_attention`.  ``workspace``: a uint8 tensor of
      :func:`paged_workspace_bytes` bytes, used by one launch at a time; without it one wave reads all keys of a
      (sequence, kv head).
    * a row that is hidden (in front of the window, behind the length, on an absent page) never enters a result, whatever
      it holds.

    At most 65535 sequences; ``B * G * ceil(M * page_size / 32)`` must stay below 2^31, one kv head of a page below 2 GiB,
    ``B * G`` below 2^23 in the streaming kernels.

    Head dimensions 128, 256 and 512 with float16 / bfloat16 pools and up to 16 query heads per kv head take the streaming
    kernel; other multiples of 8 up to 1024, larger groups and float32 pools a plain fp32 kernel.
    """
    assert isinstance(phase, int)
    q_ptr, qs, q_st, q_dt = U.float_meta(q, "q", 3)
    o_ptr, os_, o_st, o_dt = U.float_meta(o, "o", 3)
    if os_ != qs:
        raise ValueError(f"o shape {tuple(os_)} must equal q shape {tuple(qs)}")
    B, H, D = qs
    k_ptr, v_ptr, kv_dt, P, G, page_size, k_stride, v_stride = _pools(k_pages, v_pages, D)
    if G == 0 or H == 0 or H % G:
        raise ValueError("number of query heads must be a multiple of the number of kv heads")
    t_ptr, M, t_stride = _table(block_tables, B)
    len_ptr, len_st, _ = U.int_vector(seq_lens, "seq_lens", B)
    ph_ptr, ph_st, _ = (0, 0, 0) if user_phase is None else U.int_vector(user_phase, "user_phase", B, "uint8")
    if window_size is not None and window_size < 1:
        raise ValueError("window_size must be a positive int or None")
    ws, ws_bytes = U.workspace_of(workspace)
    st = U.launch_on(stream, "q k_pages v_pages o block_tables seq_lens user_phase workspace", q, k_pages, v_pages, o, block_tables,
                     seq_lens, user_phase, workspace)
    _native.call("g4b_paged_attn", st, q_ptr, k_ptr, v_ptr, o_ptr, t_ptr, len_ptr, ph_ptr, ws, ws_bytes, *U.row_strides(qs, q_st),
                 *U.row_strides(os_, o_st), k_stride, v_stride, t_stride, len_st, ph_st, q_dt, o_dt, kv_dt, B, H, G, D, P, page_size,
                 M, 0 if window_size is None else min(int(window_size), 0x7FFFFFFF), phase, num_workers, 1 if use_fp32_dot else 0, scale)
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
    ``phase`` are skipped.  Rows that fall outside the table or on an absent page are dropped.  ``G * D`` must stay below 2^24.
    """
    assert isinstance(phase, int)
    k_ptr, ks, k_st, k_dt = U.float_meta(k, "k", 3)
    v_ptr, vs, v_st, v_dt = U.float_meta(v, "v", 3)
    if vs != ks:
        raise ValueError(f"v shape {tuple(vs)} must equal k shape {tuple(ks)}")
    T, G, D = ks
    kp_ptr, vp_ptr, cache_dt, P, Gp, page_size, kp_stride, vp_stride = _pools(k_pages, v_pages, D)
    if Gp != G:
        raise ValueError(f"the pools have {Gp} kv heads, k and v {G}")
    off_ptr, off_st, N = U.int_vector(cache_offsets, "cache_offsets", None)
    t_ptr, M, t_stride = _table(block_tables, N)
    cu_ptr, cu_st = 0, 0
    if cu_seqlens is not None:
        cu_ptr, cu_st, _ = U.int_vector(cu_seqlens, "cu_seqlens", N + 1)
    elif T != N:
        raise ValueError(f"without cu_seqlens every sequence brings one row: got {T} rows and {N} sequences")
    kr_ptr, kr_st = (0, (0, 0)) if k_rsos is None else _rsos(k_rsos, "k_rsos", T, G)
    vr_ptr, vr_st = (0, (0, 0)) if v_rsos is None else _rsos(v_rsos, "v_rsos", T, G)
    ph_ptr, ph_st, _ = (0, 0, 0) if user_phase is None else U.int_vector(user_phase, "user_phase", N, "uint8")
    st = U.launch_on(stream, "k v k_pages v_pages block_tables cache_offsets cu_seqlens k_rsos v_rsos user_phase", k, v, k_pages,
                     v_pages, block_tables, cache_offsets, cu_seqlens, k_rsos, v_rsos, user_phase)
    _native.call("g4b_paged_append", st, k_ptr, v_ptr, kp_ptr, vp_ptr, t_ptr, off_ptr, cu_ptr, kr_ptr, vr_ptr, ph_ptr,
                 *U.row_strides(ks, k_st), *U.row_strides(vs, v_st), *kr_st, *vr_st, kp_stride, vp_stride, t_stride, off_st, cu_st,
                 ph_st, k_dt, v_dt, cache_dt, T, N, G, D, P, page_size, M, phase, rmsnorm_eps)
    return None


def _rsos(t, what: str, T: int, G: int):
    ptr, shape, stride, code = U.meta(t, what, 2)
    if tuple(shape) != (T, G):
        raise ValueError(f"{what} must have shape {[T, G]}, got {tuple(shape)}")
    if code != _native.DT_F32:
        raise ValueError(f"{what} must be float32")
    return ptr, stride
