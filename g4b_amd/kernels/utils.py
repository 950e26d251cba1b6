"""Tensor protocol and stream plumbing shared by the kernel wrappers.

The reference's launch adapter accepts its own ``Tensor`` dataclass or any object with
``shape``, ``stride`` (sequence or callable), ``dtype`` and ``data_ptr()``
(``g4b/kernels/utils.py:51-60,87-127``); strides are in elements.  The same objects are
accepted here and reduced to (pointer, shape, strides, dtype code).
"""

from __future__ import annotations

import ctypes as C

from .. import _native

_DTYPE_NAMES = {
    "float16": _native.DT_F16,
    "half": _native.DT_F16,
    "bfloat16": _native.DT_BF16,
    "float32": _native.DT_F32,
    "float": _native.DT_F32,
}
_INT_NAMES = {"int32": 4, "int64": 8, "uint8": 1, "int8": 1}


def _is_tensor_like(t) -> bool:
    return hasattr(t, "shape") and hasattr(t, "stride") and hasattr(t, "dtype") and hasattr(t, "data_ptr")


def dtype_name(t) -> str:
    """'float16', 'int32', ... for torch dtypes (``torch.float16``) and g4b DTypes (``.name``)."""
    dt = t.dtype
    name = getattr(dt, "name", None)
    if not isinstance(name, str):
        name = str(dt)
    return name.rsplit(".", 1)[-1]


def float_dtype_code(t, what: str) -> int:
    name = dtype_name(t)
    if name not in _DTYPE_NAMES:
        raise ValueError(f"{what}: unsupported dtype {name}")
    return _DTYPE_NAMES[name]


def int_itemsize(t, what: str, allowed) -> int:
    name = dtype_name(t)
    if name not in allowed:
        raise ValueError(f"{what}: dtype must be one of {sorted(allowed)}, got {name}")
    return _INT_NAMES[name]


def strides_of(t) -> list[int]:
    s = t.stride
    if isinstance(s, (list, tuple)):
        return [int(x) for x in s]
    if callable(s):
        return [int(s(i)) for i in range(len(t.shape))]
    raise RuntimeError("Failed to normalize tensor stride into list[int]")


def shape_of(t) -> list[int]:
    return [int(x) for x in t.shape]


def require_tensor(t, what: str, ndim: int):
    if not _is_tensor_like(t):
        raise TypeError(f"{what} must expose shape, stride, dtype and data_ptr()")
    if len(t.shape) != ndim:
        raise ValueError(f"{what} must have {ndim} dimensions, got shape {tuple(t.shape)}")


_stream_override = None


def set_stream(stream) -> None:
    """Pin the HIP stream kernels are enqueued on (an int / hipStream_t handle, or None).

    The reference launches everything on one engine-owned stream (``g4b/device.py:99,117-124``).
    Without an override the current PyTorch stream is used when torch has a GPU, else the
    default stream.
    """
    global _stream_override
    _stream_override = stream


def stream_handle(stream) -> int:
    """hipStream_t of a ``stream=`` argument: an int, a ``torch.cuda.Stream`` (``cuda_stream``) or a g4b stream
    (``handle``, ``g4b/device.py:99``)."""
    return int(getattr(stream, "cuda_stream", getattr(stream, "handle", stream)))


def current_stream() -> int:
    if _stream_override is not None:
        return stream_handle(_stream_override)
    try:
        import torch

        if torch.cuda.is_available():
            return int(torch.cuda.current_stream().cuda_stream)
    except ImportError:
        pass
    return 0


def row_strides(t):
    """Strides of ``t`` as a ctypes int64 array; a dimension of size one is never stepped over, so its stride (which may
    be anything) counts as 0."""
    dims = list(zip(shape_of(t), strides_of(t)))
    out = [0 if n == 1 else s for n, s in dims[:-1]] + [dims[-1][1]]
    return (C.c_int64 * len(out))(*out)


def stream_arg(stream):
    """The ``stream=`` argument of a wrapper (None: :func:`current_stream`) as the C ABI takes it."""
    return C.c_void_p(current_stream() if stream is None else stream_handle(stream))


def workspace_of(workspace):
    """(pointer, bytes) of a ``workspace=`` argument: a contiguous tensor of any dtype, or None."""
    if workspace is None:
        return None, 0
    if not _is_tensor_like(workspace):
        raise ValueError("workspace must be a tensor or None")
    if not getattr(workspace, "is_contiguous", lambda: True)():
        raise ValueError("workspace must be contiguous")
    return workspace.data_ptr(), int(workspace.numel()) * int(workspace.element_size())


def require_one_gpu(**tensors) -> None:
    """Torch tensors of a call must all live on the current GPU: the kernels are launched there and take their pointers as
    they are.  (Other tensor types do not say where they live.)"""
    seen = {}
    for name, t in tensors.items():
        device = getattr(t, "device", None)
        if device is None or not hasattr(device, "type"):
            continue
        if device.type != "cuda":
            raise ValueError(f"{name} must be on the GPU, it is on {device}")
        seen.setdefault(device.index, name)
    if len(seen) > 1:
        raise ValueError("all tensors of a call must be on one GPU: " + ", ".join(f"{n} is on cuda:{i}" for i, n in seen.items()))
    if seen:
        import torch

        index, name = next(iter(seen.items()))
        if index != torch.cuda.current_device():
            raise ValueError(f"{name} is on cuda:{index}, the current device is cuda:{torch.cuda.current_device()}")
