"""Causal attention over packed prompts: sequences of different lengths one after the other, without padding.

The reference prefills one slot at a time into that slot's ring (``g4b/scheduler.py:66``,
``g4b/kernels/fa2.py:634-715``) and has no counterpart; the conventions (outputs passed in, nothing allocated, explicit
``scale``, ``query_window``, ``use_fp32_dot``, ``workspace``) are those of :mod:`.fa2`.
"""

from __future__ import annotations

from .. import _native
from . import utils as U


def packed_workspace_bytes(T: int, N: int, H: int, G: int, D: int) -> int:
    """Bytes of scratch that let a launch over ``T`` rows of ``N`` sequences split the keys of its query tiles when they are
    fewer than the chip has compute units (0: such a launch never splits)."""
    return int(_native.load().g4b_packed_attn_workspace_bytes(T, N, H, G, D))


def packed_attention(
    q, k, v, o, cu_seqlens, *, query_window: int | None = None, scale: float = 1.0, use_fp32_dot: bool = False,
    workspace=None, stream=None,
):
    """``o[t, h] = softmax(scale * q[t, h] . k[j, g]^T) v[j, g]`` over the rows ``j <= t`` of the row's own sequence.

    * ``q``, ``o``: ``[T, H, D]``; ``k``, ``v``: ``[T, G, D]`` (strided views allowed, unit stride in ``D``, strides
      multiples of 8 elements); query head ``h`` reads kv head ``h // (H // G)``.
    * ``cu_seqlens``: ``[N + 1]`` int32, ascending: sequence ``s`` owns rows ``cu_seqlens[s] .. cu_seqlens[s + 1] - 1``.
      Empty sequences are allowed; rows of ``o`` outside every sequence (a buffer longer than its prompts) stay as they are.
    * ``query_window``: an int hides keys with ``t - j >= query_window`` (a sliding-window layer), ``None`` hides none.
    * ``scale`` (1.0 as in the reference, ``fa2.py:89``); ``use_fp32_dot``: a query wider than ``k``'s 16-bit type enters
      the first product unrounded (``fa2.py:85-88``), as the sum of two 16-bit operands; by default it is rounded once.
    * ``workspace``: a uint8 tensor of :func:`packed_workspace_bytes` bytes, used by one launch at a time, or ``None``.
    * a row that is hidden (a later one, one in front of the window, another sequence's) never enters a result, whatever it
      holds: infinities and NaN there are as good as any number.
    * a score of minus infinity is a weight of zero; a row with no other score becomes zeros.

    ``T * H`` must stay below 2^31; on the matrix cores the token strides of ``k`` and ``v`` below 2^24 elements, and the query
    tiles that the prompts can have, ``(T // t + min(N, T)) * G`` with ``t = 128 // (H // G)`` tokens (half of it at ``D = 512``
    with an unrounded query), below 2^24 - 16.

    Head dimensions 128, 256 and 512 with float16 / bfloat16 ``k`` and ``v`` and ``H / G`` dividing 128 run on the matrix
    cores; other multiples of 8 up to 1024, other groups and float32 ``k`` and ``v`` on a plain fp32 kernel.
    """
    q_ptr, qs, q_st, q_dt = U.float_meta(q, "q", 3)
    k_ptr, ks, k_st, kv_dt = U.float_meta(k, "k", 3)
    v_ptr, vs, v_st, v_dt = U.float_meta(v, "v", 3)
    o_ptr, os_, o_st, o_dt = U.float_meta(o, "o", 3)
    cu_ptr, cu_st, n_cu = U.int_vector(cu_seqlens, "cu_seqlens", None)
    T, H, D = qs
    G = ks[1]
    if os_ != qs:
        raise ValueError(f"o shape {tuple(os_)} must equal q shape {tuple(qs)}")
    if ks != vs or ks[0] != T or ks[2] != D:
        raise ValueError("k and v must have shape [T, G, D] with q's T and D")
    if G == 0 or H == 0 or H % G:
        raise ValueError("number of query heads must be a multiple of the number of kv heads")
    if n_cu < 1:
        raise ValueError("cu_seqlens must have shape [N + 1]")
    if v_dt != kv_dt:
        raise ValueError("k and v must have the same dtype")
    if query_window is not None and query_window < 1:
        raise ValueError("query_window must be a positive int or None")
    ws, ws_bytes = U.workspace_of(workspace)
    st = U.launch_on(stream, "q k v o cu_seqlens workspace", q, k, v, o, cu_seqlens, workspace)
    _native.call("g4b_packed_attn", st, q_ptr, k_ptr, v_ptr, o_ptr, cu_ptr, ws, ws_bytes, *U.row_strides(qs, q_st),
                 *U.row_strides(ks, k_st), *U.row_strides(vs, v_st), *U.row_strides(os_, o_st), cu_st, q_dt, o_dt, kv_dt, T,
                 n_cu - 1, H, G, D, 0 if query_window is None else min(int(query_window), 0x7FFFFFFF), 1 if use_fp32_dot else 0, scale)
    return None
