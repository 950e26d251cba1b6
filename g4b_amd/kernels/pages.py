"""Page management of a paged KV cache, on the device: copy, free, fork, allocate, compact.

The reference reserves a full ring per slot and has no counterpart (``g4b/scheduler.py:133-212`` only resets a slot's
integers).  ``ref_counts`` (``[P]`` int32: how many holders a page has) is the allocator's only state: a page is free while
its count is 0, and whoever needs pages gets the lowest-numbered free ones, so results do not depend on timing.
``block_tables`` is ``[S, M]`` int32, ``seq_lens`` ``[S]`` int32; sequence ``s`` holds the first
``ceil(seq_lens[s] / page_size)`` entries of its row.  Pools are ``[P, G, page_size, D]`` or, with every layer following
the same tables, ``[L, P, G, page_size, D]``.

Nothing here waits for the device, so every call can be recorded into a graph; what can only be seen there ends up in
``status`` (an int32 tensor of one element).  Calls on the same tables belong on one stream.
"""

from __future__ import annotations

import ctypes as C

from .. import _native
from . import utils as U

MAX_LIST = 8192  # pairs of pages, or sequences, that one call takes


def page_workspace_bytes(num_pages: int, num_seqs: int) -> int:
    """Bytes of scratch that fork, allocate and compact need (one call at a time)."""
    return int(_native.load().g4b_pages_workspace_bytes(num_pages, num_seqs))


def _vector(t, what: str, n: int | None = None):
    U.require_tensor(t, what, 1)
    U.int_itemsize(t, what, {"int32"})
    size = U.shape_of(t)[0]
    if n is not None and size != n:
        raise ValueError(f"{what} must have shape [{n}], got {tuple(t.shape)}")
    if size > 1 and U.strides_of(t)[0] != 1:
        raise ValueError(f"{what} must be contiguous")
    return t.data_ptr(), size


def _pools(a, k_pages, v_pages):
    shape = U.shape_of(k_pages) if U._is_tensor_like(k_pages) else []
    if len(shape) not in (4, 5):
        raise ValueError("k_pages must be [P, G, page_size, D] or [L, P, G, page_size, D]")
    U.require_tensor(v_pages, "v_pages", len(shape))
    if U.shape_of(v_pages) != shape:
        raise ValueError("k_pages and v_pages must have the same shape")
    a.cache_dtype = U.float_dtype_code(k_pages, "k_pages")
    if U.float_dtype_code(v_pages, "v_pages") != a.cache_dtype:
        raise ValueError("k_pages and v_pages must have the same dtype")
    L = shape[0] if len(shape) == 5 else 1
    P, G, page_size, D = shape[-4:]
    a.page_elems = G * page_size * D
    for name, t in (("k", k_pages), ("v", v_pages)):
        s = U.strides_of(t)
        if s[-1] != 1 or s[-2] != D or s[-3] != page_size * D:
            raise ValueError(f"{name}_pages must be contiguous inside a page")
        setattr(a, name + "_pages", t.data_ptr())
        setattr(a, name + "_page_stride", s[-4] if P > 1 else max(s[-4], a.page_elems))
        setattr(a, name + "_layer_stride", s[0] if L > 1 else 0)
    a.layers, a.num_pages = L, P
    return page_size


def _tables(a, block_tables, seq_lens, ref_counts, page_size: int):
    U.require_tensor(block_tables, "block_tables", 2)
    U.int_itemsize(block_tables, "block_tables", {"int32"})
    S, M = U.shape_of(block_tables)
    s = U.strides_of(block_tables)
    if M > 1 and s[1] != 1:
        raise ValueError("block_tables must have unit stride along its rows")
    a.block_tables, a.block_tables_stride, a.S, a.max_pages = block_tables.data_ptr(), s[0] if S > 1 else max(s[0], M), S, M
    a.seq_lens, _ = _vector(seq_lens, "seq_lens", S)
    a.ref_counts, P = _vector(ref_counts, "ref_counts")
    if a.num_pages and a.num_pages != P:
        raise ValueError(f"ref_counts must have one count per page ({a.num_pages}), got {P}")
    a.num_pages = P
    if int(page_size) < 1:
        raise ValueError("page_size must be positive")
    a.page_size = int(page_size)


def _list(t, what: str, n: int | None = None):
    ptr, size = _vector(t, what, n)
    if size > MAX_LIST:
        raise ValueError(f"{what} holds {size} entries, at most {MAX_LIST} fit one call")
    return ptr, size


def _call(entry: str, a, stream, **tensors):
    U.require_one_gpu(**tensors)
    _native.check(getattr(_native.load(), entry)(C.byref(a), U.stream_arg(stream)))
    return None


def copy_pages(k_pages, v_pages, src, dst, status, *, stream=None):
    """``pool[..., dst[i], ...] = pool[..., src[i], ...]`` for every pair, in both pools and every layer.

    ``src``, ``dst``: ``[n]`` int32 on the device, ``n <= 8192``.  Every source is read as it was before the call: a pair
    whose destination is also read by a pair of the list, or was named by an earlier pair, or with a page outside
    ``[0, P)``, is dropped and counted by adding 1 to ``status``.
    """
    a = _native.PagesArgs()
    _pools(a, k_pages, v_pages)
    a.src, a.n = _list(src, "src")
    a.dst, _ = _list(dst, "dst", a.n)
    a.status, _ = _vector(status, "status", 1)
    return _call("g4b_pages_copy", a, stream, k_pages=k_pages, v_pages=v_pages, src=src, dst=dst, status=status)


def free_sequences(block_tables, seq_lens, ref_counts, seqs, page_size: int, *, stream=None):
    """Sequences ``seqs`` (``[n]`` int32) give up their pages: counts go down by one (never below 0), the entries that were
    held become -1 and the lengths 0.  Indices outside ``[0, S)`` and repeated ones do nothing."""
    a = _native.PagesArgs()
    _tables(a, block_tables, seq_lens, ref_counts, page_size)
    a.src, a.n = _list(seqs, "seqs")
    return _call("g4b_pages_free", a, stream, block_tables=block_tables, seq_lens=seq_lens, ref_counts=ref_counts, seqs=seqs)


def fork_sequences(k_pages, v_pages, block_tables, seq_lens, ref_counts, src, dst, status, *, workspace, stream=None):
    """Sequence ``dst[i]`` becomes a copy of ``src[i]``: full pages are shared (their counts go up), a partly filled last
    page is copied, in every layer, to a free page of its own (an absent one stays absent).

    ``src``, ``dst``: ``[n]`` int32.  Sources are read as they were before the call.  ``status`` becomes 0; or the number
    of free pages that were missing; or -1 when an index is outside ``[0, S)``, a destination is named twice or not empty,
    or a source is longer than its table.  Unless it is 0 nothing has changed.
    """
    a = _native.PagesArgs()
    page_size = _pools(a, k_pages, v_pages)
    _tables(a, block_tables, seq_lens, ref_counts, page_size)
    a.src, a.n = _list(src, "src")
    a.dst, _ = _list(dst, "dst", a.n)
    a.status, _ = _vector(status, "status", 1)
    a.workspace, a.workspace_bytes = U.workspace_of(workspace)
    return _call("g4b_pages_fork", a, stream, k_pages=k_pages, v_pages=v_pages, block_tables=block_tables, seq_lens=seq_lens,
                 ref_counts=ref_counts, src=src, dst=dst, status=status, workspace=workspace)


def allocate_pages(block_tables, seq_lens, ref_counts, num_new, page_size: int, status, *, workspace, stream=None):
    """Every sequence ``s`` grows by ``num_new[s]`` (``[S]`` int32) positions and gets the pages for them: sequences in
    ascending order, pages in ascending order.  ``status`` becomes 0; or the number of free pages that were missing; or
    -1 when a ``num_new`` is negative or a sequence would outgrow its table.  Unless it is 0 nothing has changed."""
    a = _native.PagesArgs()
    _tables(a, block_tables, seq_lens, ref_counts, page_size)
    a.num_new, _ = _vector(num_new, "num_new", a.S)
    a.status, _ = _vector(status, "status", 1)
    a.workspace, a.workspace_bytes = U.workspace_of(workspace)
    return _call("g4b_pages_allocate", a, stream, block_tables=block_tables, seq_lens=seq_lens, ref_counts=ref_counts,
                 num_new=num_new, status=status, workspace=workspace)


def compact_pages(k_pages, v_pages, block_tables, seq_lens, ref_counts, page_map, num_live, *, workspace, stream=None):
    """The pages in use move to the front of the pool: with n of them, those at or above n move, in ascending order, into
    the free ones below n.  Tables, counts and both pools follow.  ``page_map`` (``[P]`` int32) receives every page's new
    index, -1 for free ones (for holders other than the tables), ``num_live`` (``[1]`` int32) n."""
    a = _native.PagesArgs()
    page_size = _pools(a, k_pages, v_pages)
    _tables(a, block_tables, seq_lens, ref_counts, page_size)
    a.page_map, _ = _vector(page_map, "page_map", a.num_pages)
    a.status, _ = _vector(num_live, "num_live", 1)
    a.workspace, a.workspace_bytes = U.workspace_of(workspace)
    return _call("g4b_pages_compact", a, stream, k_pages=k_pages, v_pages=v_pages, block_tables=block_tables, seq_lens=seq_lens,
                 ref_counts=ref_counts, page_map=page_map, num_live=num_live, workspace=workspace)
