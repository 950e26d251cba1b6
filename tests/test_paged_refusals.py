"""What the operators over packed prompts and pages refuse, on the host: nothing here reaches a GPU."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def K():
    import g4b_amd.kernels as kernels

    return kernels


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def packed_args(T=10, H=4, G=2, D=64, dtype=torch.float16):
    return dict(q=torch.zeros(T, H, D, dtype=dtype), k=torch.zeros(T, G, D, dtype=dtype), v=torch.zeros(T, G, D, dtype=dtype),
                o=torch.zeros(T, H, D, dtype=dtype), cu_seqlens=i32(0, 4, T))


def paged_args(B=2, H=4, G=2, D=64, P=6, page=16, M=3, dtype=torch.float16):
    return dict(q=torch.zeros(B, H, D, dtype=dtype), k_pages=torch.zeros(P, G, page, D, dtype=dtype),
                v_pages=torch.zeros(P, G, page, D, dtype=dtype), o=torch.zeros(B, H, D, dtype=dtype),
                block_tables=torch.zeros(B, M, dtype=torch.int32), seq_lens=i32(*[1] * B))


def append_args(N=2, G=2, D=64, P=6, page=16, M=3, dtype=torch.float16):
    return dict(k=torch.zeros(N, G, D, dtype=dtype), v=torch.zeros(N, G, D, dtype=dtype),
                k_pages=torch.zeros(P, G, page, D, dtype=dtype), v_pages=torch.zeros(P, G, page, D, dtype=dtype),
                block_tables=torch.zeros(N, M, dtype=torch.int32), cache_offsets=i32(*[0] * N), rmsnorm_eps=1e-6)


CASES = {
    "packed": (packed_args, "packed_attention", [
        (dict(o=torch.zeros(10, 4, 32).half()), ValueError, "must equal q shape"),
        (dict(k=torch.zeros(9, 2, 64).half()), ValueError, "shape"),
        (dict(v=torch.zeros(10, 2, 64).bfloat16()), ValueError, "same dtype"),
        (dict(k=torch.zeros(10, 3, 64).half(), v=torch.zeros(10, 3, 64).half()), ValueError, "multiple"),
        (dict(q=torch.zeros(10, 64).half()), ValueError, "3 dimensions"),
        (dict(q=[1]), TypeError, "data_ptr"),
        (dict(cu_seqlens=torch.zeros(3, dtype=torch.int64)), ValueError, "dtype"),
        (dict(cu_seqlens=i32()), ValueError, "N \\+ 1"),
        (dict(query_window=0), ValueError, "positive"),
        (dict(query_window=-4), ValueError, "positive"),
        (dict(q=torch.zeros(10, 4, 64).int()), ValueError, "dtype"),
        (dict(workspace="static"), ValueError, "workspace"),
        (dict(), ValueError, "on the GPU"),
    ]),
    "paged": (paged_args, "paged_attention", [
        (dict(o=torch.zeros(2, 4, 32).half()), ValueError, "must equal q shape"),
        (dict(v_pages=torch.zeros(6, 2, 32, 64).half()), ValueError, "same shape"),
        (dict(v_pages=torch.zeros(6, 2, 16, 64)), ValueError, "same dtype"),
        (dict(k_pages=torch.zeros(6, 16, 2, 64).half().transpose(1, 2), v_pages=torch.zeros(6, 16, 2, 64).half().transpose(1, 2)),
         ValueError, "contiguous inside a page"),
        (dict(k_pages=torch.zeros(6, 2, 16, 32).half(), v_pages=torch.zeros(6, 2, 16, 32).half()), ValueError, "D = 64"),
        (dict(block_tables=torch.zeros(3, 3, dtype=torch.int32)), ValueError, "one row per sequence"),
        (dict(block_tables=torch.zeros(3, 2, dtype=torch.int32).t()), ValueError, "unit stride"),
        (dict(block_tables=torch.zeros(2, 3, dtype=torch.int64)), ValueError, "dtype"),
        (dict(seq_lens=i32(1)), ValueError, "shape"),
        (dict(user_phase=i32(1, 1)), ValueError, "dtype"),
        (dict(phase=1.0), AssertionError, None),
        (dict(window_size=0), ValueError, "positive"),
        (dict(), ValueError, "on the GPU"),
    ]),
    "append": (append_args, "add_kv_to_pages", [
        (dict(v=torch.zeros(2, 2, 32).half()), ValueError, "must equal k shape"),
        (dict(k=torch.zeros(3, 2, 64).half(), v=torch.zeros(3, 2, 64).half()), ValueError, "one row"),
        (dict(cu_seqlens=i32(0, 1)), ValueError, "shape"),
        (dict(k_rsos=torch.zeros(2, 2).half()), ValueError, "float32"),
        (dict(v_rsos=torch.zeros(2, 3)), ValueError, "shape"),
        (dict(cache_offsets=torch.zeros(2, dtype=torch.int64)), ValueError, "dtype"),
        (dict(user_phase=torch.zeros(3, dtype=torch.uint8)), ValueError, "shape"),
        (dict(), ValueError, "on the GPU"),
    ]),
}


@pytest.mark.parametrize("name,i", [(n, i) for n, c in CASES.items() for i in range(len(c[2]))])
def test_wrappers_refuse(K, name, i):
    make, fn, cases = CASES[name]
    change, error, match = cases[i]
    args = make()
    args.update(change)
    with pytest.raises(error, match=match):
        getattr(K, fn)(**args)


def pages_state(P=8, S=4, M=3, page=16):
    pool = torch.zeros(P, 2, page, 64).half()
    return dict(k=pool, v=pool.clone(), tables=torch.zeros(S, M, dtype=torch.int32), lens=i32(*[0] * S), refs=i32(*[0] * P),
                ws=torch.zeros(4096, dtype=torch.uint8), status=i32(0), page=page)


def test_page_management_refuses(K):
    from g4b_amd.kernels import pages

    s = pages_state()
    t = (s["tables"], s["lens"], s["refs"])

    def bad(match, fn, *a, **kw):
        with pytest.raises(ValueError, match=match):
            fn(*a, **kw)

    long = torch.zeros(pages.MAX_LIST + 1, dtype=torch.int32)
    bad("at most", pages.copy_pages, s["k"], s["v"], long, long, s["status"])
    bad("shape", pages.copy_pages, s["k"], s["v"], i32(0, 1), i32(2), s["status"])
    bad("shape", pages.copy_pages, s["k"], s["v"], i32(0), i32(2), i32(0, 0))
    bad("same shape", pages.copy_pages, s["k"], s["v"][:4], i32(0), i32(2), s["status"])
    bad("contiguous inside a page", pages.copy_pages, s["k"][..., :32], s["v"][..., :32], i32(0), i32(2), s["status"])
    bad("P, G, page_size, D", pages.copy_pages, s["k"][0], s["v"][0], i32(0), i32(2), s["status"])
    bad("on the GPU", pages.copy_pages, s["k"], s["v"], i32(0), i32(2), s["status"])
    bad("at most", pages.free_sequences, *t, long, 16)
    bad("page_size", pages.free_sequences, *t, i32(0), 0)
    bad("dtype", pages.free_sequences, *t, i32(0).long(), 16)
    bad("shape", pages.free_sequences, s["tables"], i32(0), s["refs"], i32(0), 16)
    bad("on the GPU", pages.free_sequences, *t, i32(0), 16)
    bad("one count per page", pages.fork_sequences, s["k"], s["v"], s["tables"], s["lens"], i32(0, 0), i32(0), i32(1), s["status"], workspace=s["ws"])
    bad("contiguous", pages.fork_sequences, s["k"], s["v"], s["tables"], s["lens"], torch.zeros(16, dtype=torch.int32)[::2], i32(0), i32(1),
        s["status"], workspace=s["ws"])
    bad("shape", pages.allocate_pages, *t, i32(0), 16, s["status"], workspace=s["ws"])
    bad("workspace", pages.allocate_pages, *t, i32(0, 0, 0, 0), 16, s["status"], workspace="static")
    bad("shape", pages.compact_pages, s["k"], s["v"], *t, i32(0), s["status"], workspace=s["ws"])
    bad("on the GPU", pages.compact_pages, s["k"], s["v"], *t, i32(*[0] * 8), s["status"], workspace=s["ws"])


def test_struct_layouts_match_the_header(K):
    """Field order and sizes of the ctypes mirrors follow the header's structs."""
    from g4b_amd import _native as native

    header = (ROOT / "include" / "g4b_attn.h").read_text()
    size = {"void*": 8, "int32_t*": 8, "uint8_t*": 8, "float*": 8, "uint64_t": 8, "int64_t": 8, "int32_t": 4, "float": 4}
    for cname, mirror in (("g4b_packed_attn_args", native.PackedAttnArgs), ("g4b_paged_attn_args", native.PagedAttnArgs),
                          ("g4b_paged_append_args", native.PagedAppendArgs), ("g4b_pages_args", native.PagesArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), header, re.S).group(1)
        want = []
        for line in body.splitlines():
            line = line.strip().rstrip(";")
            if line:
                m = re.match(r"(?:const\s+)?([a-z0-9_]+\s*\*?)\s*(.*)", line)
                for decl in m.group(2).split(","):
                    arr = re.match(r"(\w+)(?:\[(\d+)\])?", decl.strip())
                    want.append((arr.group(1), size[m.group(1).replace(" ", "")] * int(arr.group(2) or 1)))
        assert [(n, ctypes.sizeof(t)) for n, t in mirror._fields_] == want, cname


FAKE = 4096  # an aligned address: every block below is refused before anything looks at it


def refused(fn, block, want, /, **change):
    from g4b_amd import _native as native

    for name, value in change.items():
        old = getattr(block, name)
        if hasattr(old, "__len__"):
            value = type(old)(*value)
        setattr(block, name, value)
    assert getattr(native.load(), fn)(ctypes.byref(block), None) == want, change
    assert native.last_error(), change


def packed_block():
    from g4b_amd import _native as native

    a = native.PackedAttnArgs()
    a.q = a.k = a.v = a.o = a.cu_seqlens = FAKE
    for n in ("q", "k", "v", "o"):
        setattr(a, n + "_stride", (ctypes.c_int64 * 3)(512, 128, 1))
    a.cu_seqlens_stride, a.T, a.N, a.H, a.G, a.D, a.scale = 1, 10, 2, 4, 2, 128, 1.0
    return a


def paged_block():
    from g4b_amd import _native as native

    a = native.PagedAttnArgs()
    a.q = a.o = a.k_pages = a.v_pages = a.block_tables = a.seq_lens = FAKE
    a.q_stride = a.o_stride = (ctypes.c_int64 * 3)(512, 128, 1)
    a.k_page_stride = a.v_page_stride = 2 * 16 * 128
    a.block_tables_stride, a.seq_lens_stride = 4, 1
    a.B, a.H, a.G, a.D, a.num_pages, a.page_size, a.max_pages, a.scale = 3, 4, 2, 128, 10, 16, 4, 1.0
    return a


def append_block():
    from g4b_amd import _native as native

    a = native.PagedAppendArgs()
    a.k = a.v = a.k_pages = a.v_pages = a.block_tables = a.cache_offsets = FAKE
    a.k_stride = a.v_stride = (ctypes.c_int64 * 3)(256, 128, 1)
    a.k_page_stride = a.v_page_stride = 2 * 16 * 128
    a.block_tables_stride = a.cache_offsets_stride = 1
    a.T, a.N, a.G, a.D, a.num_pages, a.page_size, a.max_pages = 3, 3, 2, 128, 10, 16, 4
    return a


def pages_block():
    from g4b_amd import _native as native

    a = native.PagesArgs()
    for n in ("k_pages", "v_pages", "block_tables", "seq_lens", "ref_counts", "src", "dst", "num_new", "page_map", "status", "workspace"):
        setattr(a, n, FAKE)
    a.workspace_bytes = 1 << 20
    a.k_page_stride = a.v_page_stride = a.page_elems = 4096
    a.block_tables_stride, a.layers, a.num_pages, a.page_size, a.S, a.max_pages, a.n = 4, 1, 10, 16, 5, 4, 2
    return a


INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("change,status", [
    (dict(T=-1), INVALID), (dict(N=-1), INVALID), (dict(H=0), INVALID), (dict(G=3), INVALID), (dict(D=12), UNSUPPORTED), (dict(D=1032), UNSUPPORTED),
    (dict(q=0), INVALID), (dict(cu_seqlens=0), INVALID), (dict(v=FAKE + 8), INVALID), (dict(o=FAKE + 2), INVALID), (dict(q_dtype=3), INVALID),
    (dict(kv_dtype=-1), INVALID), (dict(q_stride=(512, 128, 2)), INVALID), (dict(k_stride=(4, 128, 1)), INVALID), (dict(o_stride=(-512, 128, 1)), INVALID),
    (dict(query_window=-1), INVALID), (dict(scale=0.0), INVALID), (dict(scale=-1.0), INVALID), (dict(scale=NAN), INVALID), (dict(scale=INF), INVALID),
    (dict(T=1 << 30), UNSUPPORTED)], ids=str)
def test_packed_entry_point_refuses(K, change, status):
    refused("g4b_packed_attn", packed_block(), status, **change)


@pytest.mark.parametrize("change,status", [
    (dict(B=-1), INVALID), (dict(B=70000), UNSUPPORTED), (dict(H=5), INVALID), (dict(D=100), UNSUPPORTED), (dict(page_size=8), UNSUPPORTED),
    (dict(page_size=24), UNSUPPORTED), (dict(page_size=0), UNSUPPORTED), (dict(page_size=-16), UNSUPPORTED), (dict(num_pages=0), INVALID),
    (dict(max_pages=0), INVALID), (dict(max_pages=1 << 28), UNSUPPORTED), (dict(k_page_stride=16), INVALID), (dict(v_page_stride=2 * 16 * 128 + 4), INVALID),
    (dict(k_pages=FAKE + 8), INVALID), (dict(block_tables=0), INVALID), (dict(seq_lens=0), INVALID), (dict(o=0), INVALID), (dict(window_size=-2), INVALID),
    (dict(phase=256), INVALID), (dict(num_workers=-1), INVALID), (dict(num_workers=1 << 21), INVALID), (dict(scale=NAN), INVALID),
    (dict(kv_dtype=7), INVALID), (dict(workspace=FAKE, workspace_bytes=64), WORKSPACE), (dict(workspace=FAKE + 8, workspace_bytes=1 << 30), INVALID),
    (dict(B=65535, G=4, H=4, max_pages=1 << 20, k_page_stride=1 << 20, v_page_stride=1 << 20), UNSUPPORTED)], ids=str)
def test_paged_entry_point_refuses(K, change, status):
    refused("g4b_paged_attn", paged_block(), status, **change)


@pytest.mark.parametrize("change,status", [
    (dict(T=-1), INVALID), (dict(T=4), INVALID), (dict(D=12), UNSUPPORTED), (dict(G=0), INVALID), (dict(page_size=10), UNSUPPORTED), (dict(phase=-1), INVALID),
    (dict(rmsnorm_eps=NAN), INVALID), (dict(k=0), INVALID), (dict(v=FAKE + 4), INVALID), (dict(v_stride=(256, 100, 1)), INVALID), (dict(cache_dtype=9), INVALID),
    (dict(cache_offsets=0), INVALID), (dict(v_page_stride=100), INVALID)], ids=str)
def test_append_entry_point_refuses(K, change, status):
    refused("g4b_paged_append", append_block(), status, **change)


@pytest.mark.parametrize("fn,change,status", [
    ("copy", dict(n=-1), INVALID), ("copy", dict(n=8193), INVALID), ("copy", dict(num_pages=0), INVALID), ("copy", dict(k_pages=0), INVALID),
    ("copy", dict(page_elems=4), INVALID), ("copy", dict(k_page_stride=4000), INVALID), ("copy", dict(v_layer_stride=4), INVALID), ("copy", dict(src=0), INVALID),
    ("copy", dict(status=0), INVALID), ("copy", dict(layers=0), INVALID), ("copy", dict(cache_dtype=4), INVALID), ("copy", dict(v_pages=FAKE + 8), INVALID),
    ("free", dict(S=0), INVALID), ("free", dict(S=1 << 19), INVALID), ("free", dict(max_pages=(1 << 20) + 1), INVALID), ("free", dict(ref_counts=FAKE + 4), INVALID),
    ("free", dict(block_tables_stride=3), INVALID), ("free", dict(src=0), INVALID), ("free", dict(seq_lens=0), INVALID), ("free", dict(page_size=0), INVALID),
    ("fork", dict(n=6), INVALID), ("fork", dict(workspace=0), WORKSPACE), ("fork", dict(workspace_bytes=8), WORKSPACE), ("fork", dict(dst=0), INVALID),
    ("fork", dict(status=0), INVALID), ("fork", dict(workspace=FAKE + 4), INVALID), ("allocate", dict(num_new=0), INVALID), ("allocate", dict(workspace=0), WORKSPACE),
    ("allocate", dict(num_pages=1 << 28), INVALID), ("compact", dict(page_map=0), INVALID), ("compact", dict(workspace_bytes=0), WORKSPACE),
    ("compact", dict(v_pages=0), INVALID)], ids=str)
def test_page_entry_points_refuse(K, fn, change, status):
    refused("g4b_pages_" + fn, pages_block(), status, **change)


def test_null_blocks_are_refused(K):
    from g4b_amd import _native as native

    for fn in ("g4b_packed_attn", "g4b_paged_attn", "g4b_paged_append", "g4b_pages_copy", "g4b_pages_free", "g4b_pages_fork",
               "g4b_pages_allocate", "g4b_pages_compact"):
        assert getattr(native.load(), fn)(None, None) == INVALID


def test_sizes(K):
    from g4b_amd.kernels import packed, paged, pages

    assert paged.paged_workspace_bytes(64, 8, 2, 256) == K.fa2.workspace_bytes(64, 8, 2, 1, 256)
    assert paged.paged_workspace_bytes(64, 8, 2, 64) == 0 == paged.paged_workspace_bytes(0, 8, 2, 256)
    assert packed.packed_workspace_bytes(0, 0, 8, 2, 256) == 0 == packed.packed_workspace_bytes(100, 2, 8, 2, 64)
    assert pages.page_workspace_bytes(0, 4) == 0 == pages.page_workspace_bytes(4, 0)
    assert pages.page_workspace_bytes(1000, 8) >= 4 * (1000 + 16)


def test_packed_kernels_keep_foreign_memory_traffic_out_of_their_wait_regions():
    """As for the kernels that share their bodies: a compiler-made memory access between the first and the last MFMA would
    break the hand-counted waits."""
    from g4b_amd.build import PACKED_SOURCES, check_wait_discipline

    seen = check_wait_discipline(PACKED_SOURCES)
    # head dims 128, 256 and 512, fp16 and bf16, the query rounded or split into two operands
    assert len(seen) == 12, seen
    assert all(n >= 48 for n in seen.values()), seen


@pytest.mark.parametrize("entry,value", [(e, v) for e in ("g4b_packed_attn", "g4b_paged_attn", "g4b_paged_append") for v in (1e50, -1e50, None)]
                         + [("g4b_pages_free", v) for v in (1 << 40, -(1 << 40), 1.5, None)], ids=str)
def test_numbers_that_do_not_fit_their_field_are_refused(K, entry, value):
    """The last field of every block is a 32-bit number."""
    from g4b_amd import _native as native

    n = sum(getattr(t, "_length_", 1) for _, t in native.PACKED_ENTRIES[entry]._fields_)
    with pytest.raises(ValueError):
        native.call(entry, 0, *[0] * (n - 1), value)
