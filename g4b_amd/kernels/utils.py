"""Tensor protocol and stream plumbing shared by the kernel wrappers.

The reference's launch adapter accepts its own ``Tensor`` dataclass or any object with
``shape``, ``stride`` (sequence or callable), ``dtype`` and ``data_ptr()``
(``g4b/kernels/utils.py:51-60,87-127``); strides are in elements.  The same objects are
accepted here and reduced to (pointer, shape, strides, dtype code).
"""

from __future__ import annotations

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

        if torch.cuda.is_initialized():  # (a third of the time of the general way below)
            return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
        if torch.cuda.is_available():
            return int(torch.cuda.current_stream().cuda_stream)
    except ImportError:
        pass
    return 0


# ---- arguments of the calls that a serving step makes many of --------------------------------------------------------

_CODES = {}  # dtype object -> DT_* of a float type, or the name of an integer type


def meta(t, what: str, ndim: int):
    """(pointer, shape, strides, dtype) of a tensor in one go; dtype is a DT_* code or the name of any other type."""
    try:
        shape, stride, dtype, ptr = t.shape, t.stride, t.dtype, t.data_ptr()
    except AttributeError:
        raise TypeError(f"{what} must expose shape, stride, dtype and data_ptr()") from None
    if len(shape) != ndim:
        raise ValueError(f"{what} must have {ndim} dimensions, got shape {tuple(shape)}")
    try:
        code = _CODES[dtype]
    except (KeyError, TypeError):
        name = dtype_name(t)
        code = _DTYPE_NAMES.get(name, name)
        try:
            _CODES[dtype] = code
        except TypeError:
            pass
    try:
        stride = stride()  # a torch tensor's
    except TypeError:
        stride = strides_of(t)
    return ptr, shape, stride, code


def float_meta(t, what: str, ndim: int):
    m = meta(t, what, ndim)
    if m[3].__class__ is not int:
        raise ValueError(f"{what}: unsupported dtype {m[3]}")
    return m


def int_vector(t, what: str, n: int | None, dtype: str = "int32"):
    """(pointer, stride, size) of a one-dimensional integer tensor (of size n)."""
    ptr, shape, stride, code = meta(t, what, 1)
    if code != dtype:
        raise ValueError(f"{what}: dtype must be {dtype}, got {dtype_name(t)}")
    size = shape[0]
    if n is not None and size != n:
        raise ValueError(f"{what} must have shape [{n}], got {tuple(shape)}")
    return ptr, stride[0], size


def row_strides(shape, stride):
    """Strides of a [rows, heads, D] tensor; a dimension of size one is never stepped over, so its stride (which may be
    anything) counts as 0."""
    return (0 if shape[0] == 1 else stride[0]), (0 if shape[1] == 1 else stride[1]), stride[2]


def workspace_of(workspace):
    """(pointer, bytes) of a ``workspace=`` argument: a contiguous tensor of any dtype, or None."""
    if workspace is None:
        return 0, 0
    if not _is_tensor_like(workspace):
        raise ValueError("workspace must be a tensor or None")
    if not getattr(workspace, "is_contiguous", lambda: True)():
        raise ValueError("workspace must be contiguous")
    return workspace.data_ptr(), int(workspace.numel()) * int(workspace.element_size())


def launch_on(stream, what: str, *tensors) -> int:
    """The stream to launch on, after a check that torch tensors all live on the current GPU: the kernels run there and take
    the pointers as they are.  ``what``: the tensors' names.  (Other tensor types do not say where they live.)"""
    try:
        import torch

        here = torch._C._cuda_getDevice() if torch.cuda.is_initialized() else -2
        for t in tensors:
            if t is not None and t.get_device() != here:
                _explain_devices(what.split(), tensors)
    except (ImportError, AttributeError):
        _explain_devices(what.split(), tensors)
    return current_stream() if stream is None else stream_handle(stream)


def _explain_devices(names, tensors) -> None:
    seen = {}
    for name, t in zip(names, tensors):
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
