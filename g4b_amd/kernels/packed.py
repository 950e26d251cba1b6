"""Causal attention over packed prompts: sequences of different lengths one after the other, without padding.

The reference prefills one slot at a time into that slot's ring (``g4b/scheduler.py:66``,
``g4b/kernels/fa2.py:634-715``) and has no counterpart; the conventions (outputs passed in, nothing allocated, explicit
``scale``, ``query_window``, ``use_fp32_dot``, ``workspace``) are those of :mod:`.fa2`.
"""

from __future__ import annotations

import ctypes as C

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
      the first product unrounded (``fa2.py:85-88``), by default it is rounded once.
    * ``workspace``: a uint8 tensor of :func:`packed_workspace_bytes` bytes, used by one launch at a time, or ``None``.

    Head dimensions 128, 256 and 512 with float16 / bfloat16 ``k`` and ``v`` and ``H / G`` dividing 128 run on the matrix
    cores; other multiples of 8 up to 1024, other groups and float32 ``k`` and ``v`` on a plain fp32 kernel.
    """
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o)):
        U.require_tensor(t, name, 3)
    U.require_tensor(cu_seqlens, "cu_seqlens", 1)
    U.int_itemsize(cu_seqlens, "cu_seqlens", {"int32"})
    T, H, D = U.shape_of(q)
    G = U.shape_of(k)[1]
    if U.shape_of(o) != [T, H, D]:
        raise ValueError(f"o shape {tuple(o.shape)} must equal q shape {tuple(q.shape)}")
    if U.shape_of(k) != [T, G, D] or U.shape_of(v) != [T, G, D]:
        raise ValueError("k and v must have shape [T, G, D] with q's T and D")
    if G == 0 or H == 0 or H % G:
        raise ValueError("number of query heads must be a multiple of the number of kv heads")
    if U.shape_of(cu_seqlens)[0] < 1:
        raise ValueError("cu_seqlens must have shape [N + 1]")
    kv_dt = U.float_dtype_code(k, "k")
    if U.float_dtype_code(v, "v") != kv_dt:
        raise ValueError("k and v must have the same dtype")
    if query_window is not None and int(query_window) < 1:
        raise ValueError("query_window must be a positive int or None")

    a = _native.PackedAttnArgs()
    a.q, a.k, a.v, a.o, a.cu_seqlens = (t.data_ptr() for t in (q, k, v, o, cu_seqlens))
    a.q_stride, a.k_stride, a.v_stride, a.o_stride = (U.row_strides(t) for t in (q, k, v, o))
    a.cu_seqlens_stride = U.strides_of(cu_seqlens)[0]
    a.q_dtype, a.o_dtype, a.kv_dtype = U.float_dtype_code(q, "q"), U.float_dtype_code(o, "o"), kv_dt
    a.T, a.N, a.H, a.G, a.D = T, U.shape_of(cu_seqlens)[0] - 1, H, G, D
    a.query_window = 0 if query_window is None else int(query_window)
    a.use_fp32_dot = 1 if use_fp32_dot else 0
    a.scale = float(scale)
    a.workspace, a.workspace_bytes = U.workspace_of(workspace)
    U.require_one_gpu(q=q, k=k, v=v, o=o, cu_seqlens=cu_seqlens, workspace=workspace)
    _native.check(_native.load().g4b_packed_attn(C.byref(a), U.stream_arg(stream)))
    return None
