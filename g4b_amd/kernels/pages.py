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

from .. import _native
from . import utils as U

MAX_LIST = 8192  # pairs of pages, or sequences, that one call takes


def page_workspace_bytes(num_pages: int, num_seqs: int) -> int:
    """Bytes of scratch that fork, allocate and compact need (one call at a time)."""
    return int(_native.load().g4b_pages_workspace_bytes(num_pages, num_seqs))


def _vector(t, what: str, n: int | None = None):
    ptr, stride, size = U.int_vector(t, what, n)
    if stride != 1 and size > 1:
        raise ValueError(f"{what} must be contiguous")
    return ptr, size


def _list(t, what: str, n: int | None = None):
    ptr, size = _vector(t, what, n)
    if size > MAX_LIST:
        raise ValueError(f"{what} holds {size} entries, at most {MAX_LIST} fit one call")
    return ptr, size


class _Pools:
    """Checked pools ``[L, P, G, page_size, D]`` or ``[P, G, page_size, D]``."""

    __slots__ = ("k", "v", "strides", "elems", "dtype", "layers", "P", "page_size")

    def __init__(self, k_pages, v_pages):
        ndim = len(getattr(k_pages, "shape", ()))
        if ndim not in (4, 5):
            raise ValueError("k_pages must be [P, G, page_size, D] or [L, P, G, page_size, D]")
        self.k, shape, k_st, self.dtype = U.float_meta(k_pages, "k_pages", ndim)
        self.v, v_shape, v_st, v_dt = U.float_meta(v_pages, "v_pages", ndim)
        if shape != v_shape:
            raise ValueError("k_pages and v_pages must have the same shape")
        if v_dt != self.dtype:
            raise ValueError("k_pages and v_pages must have the same dtype")
        P, G, page_size, D = shape[-4:]
        for name, st in (("k_pages", k_st), ("v_pages", v_st)):
            if st[-1] != 1 or st[-2] != D or (G > 1 and st[-3] != page_size * D):
                raise ValueError(f"{name} must be contiguous inside a page")
        self.layers, self.P, self.page_size, self.elems = shape[0] if ndim == 5 else 1, P, page_size, G * page_size * D
        one, single = P == 1, self.layers == 1  # (the stride of a dimension of size one says nothing)
        self.strides = (0 if single else k_st[0], 0 if single else v_st[0], self.elems if one else k_st[-4], self.elems if one else v_st[-4])


def _tables(block_tables, seq_lens, ref_counts, page_size: int, pools=None):
    """(table pointer, row stride, S, M, lengths pointer, counts pointer, P)."""
    ptr, (S, M), stride, code = U.meta(block_tables, "block_tables", 2)
    if code != "int32":
        raise ValueError(f"block_tables: dtype must be int32, got {U.dtype_name(block_tables)}")
    if M > 1 and stride[1] != 1:
        raise ValueError("block_tables must have unit stride along its rows")
    lens, _ = _vector(seq_lens, "seq_lens", S)
    refs, P = _vector(ref_counts, "ref_counts")
    if pools is not None and pools.P != P:
        raise ValueError(f"ref_counts must have one count per page ({pools.P}), got {P}")
    if page_size < 1:
        raise ValueError("page_size must be positive")
    return ptr, (M if S == 1 else stride[0]), S, M, lens, refs, P


_NO_POOLS = (0, 0, 0, 0)


def copy_pages(k_pages, v_pages, src, dst, status, *, stream=None):
    """``pool[..., dst[i], ...] = pool[..., src[i], ...]`` for every pair, in both pools and every layer.

    ``src``, ``dst``: ``[n]`` int32 on the device, ``n <= 8192``.  Every source is read as it was before the call: a pair
    whose destination is also read by a pair of the list, or was named by an earlier pair, or with a page outside
    ``[0, P)``, is dropped and counted by adding 1 to ``status``.  A pair of a page with itself moves nothing and stands in
    no other pair's way.
    """
    p = _Pools(k_pages, v_pages)
    src_ptr, n = _list(src, "src")
    dst_ptr, _ = _list(dst, "dst", n)
    st_ptr, _ = _vector(status, "status", 1)
    at = U.launch_on(stream, "k_pages v_pages src dst status", k_pages, v_pages, src, dst, status)
    _native.call("g4b_pages_copy", at, p.k, p.v, 0, 0, 0, src_ptr, dst_ptr, 0, 0, st_ptr, 0, 0, *p.strides, p.elems, 0, p.dtype,
                 p.layers, p.P, p.page_size, 0, 0, n)


def free_sequences(block_tables, seq_lens, ref_counts, seqs, page_size: int, *, stream=None):
    """Sequences ``seqs`` (``[n]`` int32) give up their pages: counts go down by one (never below 0), the entries that were
    held become -1 and the lengths 0.  Indices outside ``[0, S)`` and repeated ones do nothing."""
    t_ptr, t_st, S, M, lens, refs, P = _tables(block_tables, seq_lens, ref_counts, page_size)
    src_ptr, n = _list(seqs, "seqs")
    at = U.launch_on(stream, "block_tables seq_lens ref_counts seqs", block_tables, seq_lens, ref_counts, seqs)
    _native.call("g4b_pages_free", at, 0, 0, t_ptr, lens, refs, src_ptr, 0, 0, 0, 0, 0, 0, *_NO_POOLS, 0, t_st, 0, 0, P, page_size, S, M, n)


def fork_sequences(k_pages, v_pages, block_tables, seq_lens, ref_counts, src, dst, status, *, workspace, stream=None):
    """Sequence ``dst[i]`` becomes a copy of ``src[i]``: full pages are shared (their counts go up), a partly filled last
    page is copied, in every layer, to a free page of its own (an absent one stays absent).

    ``src``, ``dst``: ``[n]`` int32.  Sources are read as they were before the call.  ``status`` becomes 0; or the number
    of free pages that were missing; or -1 when an index is outside ``[0, S)``, a destination is named twice or not empty,
    or a source is longer than its table.  Unless it is 0 nothing has changed.
    """
    p = _Pools(k_pages, v_pages)
    t_ptr, t_st, S, M, lens, refs, P = _tables(block_tables, seq_lens, ref_counts, p.page_size, p)
    src_ptr, n = _list(src, "src")
    dst_ptr, _ = _list(dst, "dst", n)
    st_ptr, _ = _vector(status, "status", 1)
    ws, ws_bytes = U.workspace_of(workspace)
    at = U.launch_on(stream, "k_pages v_pages block_tables seq_lens ref_counts src dst status workspace", k_pages, v_pages, block_tables,
                     seq_lens, ref_counts, src, dst, status, workspace)
    _native.call("g4b_pages_fork", at, p.k, p.v, t_ptr, lens, refs, src_ptr, dst_ptr, 0, 0, st_ptr, ws, ws_bytes, *p.strides, p.elems,
                 t_st, p.dtype, p.layers, P, p.page_size, S, M, n)


def allocate_pages(block_tables, seq_lens, ref_counts, num_new, page_size: int, status, *, workspace, stream=None):
    """Every sequence ``s`` grows by ``num_new[s]`` (``[S]`` int32) positions and gets the pages for them: sequences in
    ascending order, pages in ascending order.  ``status`` becomes 0; or the number of free pages that were missing; or
    -1 when a ``num_new`` is negative or a sequence would outgrow its table.  Unless it is 0 nothing has changed."""
    t_ptr, t_st, S, M, lens, refs, P = _tables(block_tables, seq_lens, ref_counts, page_size)
    new_ptr, _ = _vector(num_new, "num_new", S)
    st_ptr, _ = _vector(status, "status", 1)
    ws, ws_bytes = U.workspace_of(workspace)
    at = U.launch_on(stream, "block_tables seq_lens ref_counts num_new status workspace", block_tables, seq_lens, ref_counts, num_new,
                     status, workspace)
    _native.call("g4b_pages_allocate", at, 0, 0, t_ptr, lens, refs, 0, 0, new_ptr, 0, st_ptr, ws, ws_bytes, *_NO_POOLS, 0, t_st, 0, 0, P,
                 page_size, S, M, 0)


def compact_pages(k_pages, v_pages, block_tables, seq_lens, ref_counts, page_map, num_live, *, workspace, stream=None):
    """The pages in use move to the front of the pool: with n of them, those at or above n move, in ascending order, into
    the free ones below n.  Tables, counts and both pools follow.  ``page_map`` (``[P]`` int32) receives every page's new
    index, -1 for free ones (for holders other than the tables), ``num_live`` (``[1]`` int32) n."""
    p = _Pools(k_pages, v_pages)
    t_ptr, t_st, S, M, lens, refs, P = _tables(block_tables, seq_lens, ref_counts, p.page_size, p)
    map_ptr, _ = _vector(page_map, "page_map", P)
    live_ptr, _ = _vector(num_live, "num_live", 1)
    ws, ws_bytes = U.workspace_of(workspace)
    at = U.launch_on(stream, "k_pages v_pages block_tables seq_lens ref_counts page_map num_live workspace", k_pages, v_pages,
                     block_tables, seq_lens, ref_counts, page_map, num_live, workspace)
    _native.call("g4b_pages_compact", at, p.k, p.v, t_ptr, lens, refs, 0, 0, 0, map_ptr, live_ptr, ws, ws_bytes, *p.strides, p.elems,
                 t_st, p.dtype, p.layers, P, p.page_size, S, M, 0)
