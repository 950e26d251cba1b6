"""The paged cache: decode attention and append against a plain implementation in 64 bits."""

import random

import pytest
import torch

from paged_helpers import U16, attend64, check_attention, make_tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged(gpu_device):
    from g4b_amd.kernels import paged

    return paged


class Case:
    def __init__(self, lens, H, G, D, page, dtype=torch.float16, seed=0, q_dtype=None, fill=None):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.D, self.H, self.G = lens, page, D, H, G
        self.tables, P = make_tables([max(n, 0) for n in lens], page, gen)
        self.k, self.v = (torch.randn(P, G, page, D, generator=gen).to(dtype).cuda() for _ in range(2))
        if fill is not None:  # what is not part of a sequence holds this
            held = torch.zeros(P, page, dtype=torch.bool)
            for b, n in enumerate(lens):
                for j in range(n):
                    held[self.tables[b, j // page], j % page] = True
            for x in (self.k, self.v):
                x.masked_fill_(~held.cuda()[:, None, :, None], fill)
        self.q = torch.randn(len(lens), H, D, generator=gen).to(q_dtype or dtype).cuda()
        self.o = torch.full((len(lens), H, D), 777.0, dtype=q_dtype or dtype, device="cuda")
        self.len_t = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def run(self, paged, ws=True, num_workers=0, **kw):
        w = None
        if ws:
            n = paged.paged_workspace_bytes(len(self.lens), self.H, self.G, self.D, num_workers)
            w = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda") if n else None
        paged.paged_attention(self.q, self.k, self.v, self.o, self.tables, self.len_t, scale=self.D**-0.5, workspace=w,
                              num_workers=num_workers, **kw)
        torch.cuda.synchronize()
        return self

    def rows(self, pool, b, g, n):
        """(rows [n, D], absent [n]) of a sequence."""
        pages = self.tables[b].long().repeat_interleave(self.page)[:n]
        absent = (pages < 0) | (pages >= pool.shape[0])
        return pool[pages.masked_fill(absent, 0), g, torch.arange(n, device="cuda") % self.page], absent.cpu()

    def check(self, window=None, q_rounded=False, seqs=None):
        for b, n in enumerate(self.lens):
            if seqs is not None and b not in seqs:
                continue
            n = min(max(n, 0), self.tables.shape[1] * self.page)
            for g in range(self.G):
                (k, absent), (v, _) = self.rows(self.k, b, g, n), self.rows(self.v, b, g, n)
                hidden = absent.clone()
                if window:
                    hidden |= torch.arange(n) < n - window
                R = self.H // self.G
                heads = slice(g * R, (g + 1) * R)
                if n == 0 or bool(hidden.all()):
                    assert bool((self.o[b, heads] == 0).all()), f"sequence {b}: not zeros"
                    continue
                ref, mag, qk = attend64(self.q[b, heads], k, v, hidden[None].expand(R, n), self.D**-0.5)
                check_attention(self.o[b, heads], ref, mag, qk, n, self.D, self.k.dtype, q_rounded, f"sequence {b} kv head {g}")


@pytest.mark.parametrize("lens", [[1], [2], [15, 16, 17], [31, 32, 33], [0, 1, 0], [47, 0, 64, 700], [1025]], ids=str)
@pytest.mark.parametrize("page", [16, 32, 48, 64, 256])
@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
def test_lengths(paged, lens, page, D, ws):
    Case(lens, 8, 2, D, page, seed=sum(lens) + page, fill=float("nan")).run(paged, ws).check()


@pytest.mark.parametrize("window", [1, 2, 16, 17, 31, 33, 100, 512, 513, 100000])
@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
def test_windows(paged, window, page, D, ws):
    c = Case([1, 40, 0, 700, 1100], 4, 2, D, page, torch.bfloat16, seed=window, fill=float("nan"))
    c.run(paged, ws, window_size=window).check(window)


@pytest.mark.parametrize("window", [5, 16, 33, 200])
@pytest.mark.parametrize("D", [128, 256, 512, 64])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
def test_pages_behind_the_window_may_be_gone(paged, window, D, ws):
    """Rows before the window hold NaN where their page is still there, and most of their pages are gone."""
    lens, page = [300, 95, 1, 513], 16
    c = Case(lens, 8, 2, D, page, seed=window)
    for b, n in enumerate(lens):
        lo = max(0, n - window)
        for x in (c.k, c.v):
            pages = c.tables[b].long().repeat_interleave(page)[:lo]
            x[pages, :, torch.arange(lo, device="cuda") % page] = float("nan")
        c.tables[b, : max(lo // page - 1, 0)] = -1
        c.tables[b, -(-n // page):] = 1 << 30  # (past the sequence: never read)
    c.run(paged, ws, window_size=window).check(window)


@pytest.mark.parametrize("D", [128, 256, 512, 64])
@pytest.mark.parametrize("page", [16, 32, 80])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
def test_absent_pages_hide_their_keys(paged, D, page, ws):
    """Absent pages anywhere, named by negative and by too large entries, next to pages of NaN that nobody holds."""
    lens = [500, 33, 16, 260, 700]
    c = Case(lens, 4, 2, D, page, seed=page, fill=float("nan"))
    P = c.k.shape[0]
    gen = torch.Generator().manual_seed(page)
    for b, n in enumerate(lens):
        held = -(-n // page)
        gone = torch.rand(held, generator=gen) < 0.4
        if b == 1:
            gone[:] = True
        bad = torch.tensor([-1, P, P + 7, -(1 << 31), (1 << 31) - 1])[torch.randint(0, 5, (held,), generator=gen)]
        c.tables[b, :held] = torch.where(gone, bad, c.tables[b, :held].cpu().long()).int().cuda()
    c.run(paged, ws).check()


@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (4, 1), (8, 1), (16, 1), (12, 4), (10, 2), (32, 8), (17, 1), (40, 2)], ids=str)
@pytest.mark.parametrize("D", [128, 256, 512])
def test_head_layouts(paged, heads, D):
    Case([100, 5, 333], *heads, D, 32, torch.bfloat16, seed=heads[0]).run(paged).check()


@pytest.mark.parametrize("D", [8, 64, 80, 1024])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_other_head_dims(paged, D, dtype):
    Case([70, 0, 129], 4, 2, D, 16, dtype, seed=D, fill=float("nan")).run(paged, window_size=100).check(100)


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("q_dtype,dtype", [(torch.float32, torch.float16), (torch.float32, torch.bfloat16),
                                           (torch.float16, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("fp32_dot", [False, True])
def test_query_types(paged, D, q_dtype, dtype, fp32_dot):
    c = Case([333, 64, 1], 8, 2, D, 16, dtype, seed=4, q_dtype=q_dtype)
    c.run(paged, use_fp32_dot=fp32_dot).check(q_rounded=True)


@pytest.mark.parametrize("num_workers", [1, 2, 3, 7, 64, 1000, 5000])
@pytest.mark.parametrize("D", [128, 256, 512])
def test_worker_counts(paged, num_workers, D):
    Case([1, 800, 0, 333, 64, 65], 8, 2, D, 32, seed=num_workers).run(paged, num_workers=num_workers).check()


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
def test_phases_and_odd_lengths(paged, D, ws):
    """Skipped sequences keep their rows; lengths below 0 count as 0 and lengths past the table as all of it."""
    c = Case([64, 64, 64, 64], 4, 2, D, 16, seed=1)
    c.lens = [64, -7, 5000, 64]
    c.len_t.copy_(torch.tensor(c.lens, dtype=torch.int32))
    phase = torch.tensor([2, 2, 2, 1], dtype=torch.uint8, device="cuda")
    c.run(paged, ws, user_phase=phase, phase=2).check(seqs=(0, 1, 2))
    assert bool((c.o[3] == 777.0).all())


@pytest.mark.parametrize("D", [128, 256])
def test_more_sequences_than_lanes(paged, D):
    gen = torch.Generator().manual_seed(3)
    lens = [int(x) for x in torch.randint(0, 90, (150,), generator=gen)]
    for ws in (False, True):
        Case(lens, 4, 2, D, 16, seed=2).run(paged, ws).check()
        Case(lens, 4, 2, D, 16, seed=2).run(paged, ws, window_size=20).check(20)


@pytest.mark.parametrize("D", [128, 256])
def test_views(paged, D):
    """Pools that are interleaved in one buffer with a gap between pages, tables and lengths with strides, q and o as views."""
    c = Case([100, 17, 250], 8, 2, D, 16, seed=5)
    P, G, page, _ = c.k.shape
    both = torch.full((P, 2 * G * page * D + 64), float("nan"), dtype=torch.float16, device="cuda")
    k = both[:, : G * page * D].unflatten(1, (G, page, D))
    v = both[:, G * page * D:2 * G * page * D].unflatten(1, (G, page, D))
    k.copy_(c.k), v.copy_(c.v)
    c.k, c.v = k, v
    wide = torch.full((3, 2 * c.tables.shape[1]), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, : c.tables.shape[1]] = c.tables
    c.tables = wide[:, : c.tables.shape[1]]
    c.len_t = torch.stack([c.len_t, c.len_t + 99], 1)[:, 0]
    c.q = torch.cat([c.q, c.q], 1)[:, :8]
    out = torch.full((3, 9, D + 16), 777.0, dtype=torch.float16, device="cuda")
    c.o = out[:, :8, :D]
    c.run(paged).check()
    assert bool((out[:, 8] == 777.0).all()) and bool((out[:, :, D:] == 777.0).all())


@pytest.mark.parametrize("window", [1, 5, 16, 33, 200, 700])
@pytest.mark.parametrize("D", [128, 256, 512, 64])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_hidden_rows_may_hold_anything(paged, window, D, ws, dtype):
    """K and V rows in front of the window and behind the length hold infinities and NaN."""
    c = Case([1000, 217, 33, 750], 8, 2, D, 48, dtype, seed=11, fill=float("nan"))
    for b, n in enumerate(c.lens):
        for j in range(max(n - window, 0)):
            page = int(c.tables[b, j // c.page])
            c.k[page, :, j % c.page] = (float("inf"), float("nan"), float("-inf"))[j % 3]
            c.v[page, :, j % c.page] = (float("nan"), float("-inf"), float("inf"))[j % 3]
    c.run(paged, ws, window_size=window)
    for b, n in enumerate(c.lens):
        seen = torch.arange(max(n - window, 0), n, device="cuda")
        hidden = torch.zeros(4, seen.numel(), dtype=torch.bool)
        for g in range(2):
            (k, _), (v, _) = c.rows(c.k, b, g, n), c.rows(c.v, b, g, n)
            heads = slice(g * 4, (g + 1) * 4)
            ref, mag, qk = attend64(c.q[b, heads], k[seen], v[seen], hidden, D**-0.5)
            check_attention(c.o[b, heads], ref, mag, qk, n, D, dtype, what=f"sequence {b} kv head {g}")


@pytest.mark.parametrize("D", [128, 256, 512, 64])
@pytest.mark.parametrize("ws,window", [(False, None), (True, None), (True, 100), (True, 1)], ids=str)
def test_nan_that_is_seen_is_not_lost(paged, D, ws, window):
    """A NaN in a query, in a visible key or in a visible value reaches the rows that see it, and no others."""
    c = Case([300, 33, 1, 64], 8, 2, D, 16, seed=13)
    c.q[0, 1] = float("nan")
    c.k[c.tables[1, 32 // 16], 0, 32 % 16] = float("nan")
    c.v[c.tables[2, 0], 1, 0] = float("nan")
    c.run(paged, ws, window_size=window)
    bad = torch.zeros(4, 8, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[1, :4] = bad[2, 4:] = True
    assert bool((torch.isfinite(c.o).all(-1) == ~bad).all())
    assert not bool(torch.isfinite(c.o[bad]).any())
    want = c.o.clone()
    c.q[0, 1] = 0
    for x in (c.k, c.v):
        x.nan_to_num_(0.0)
    c.run(paged, ws, window_size=window).check(window)
    assert torch.equal(want[~bad], c.o[~bad])


@pytest.mark.parametrize("seed", range(48))
def test_random_caches(paged, seed):
    """Head layouts, types, page sizes, windows, lengths and workers drawn at random."""
    rng = random.Random(seed)
    D = rng.choice([128, 128, 256, 256, 512, 64])
    G = rng.choice([1, 2, 3, 8])
    H = G * rng.choice([1, 2, 4, 8, 5, 16])
    dtype = rng.choice([torch.float16, torch.bfloat16])
    q_dtype = rng.choice([None, None, torch.float32])
    fp32_dot = q_dtype is not None and rng.random() < 0.5
    window = rng.choice([None, None, rng.randint(1, 64), rng.randint(65, 600)])
    page = 16 * rng.randint(1, 20)
    lens = [rng.choice([0, 1, rng.randint(1, 70), rng.randint(1, 700), rng.randint(700, 2500)]) for _ in range(rng.randint(1, 6))]
    workers = rng.choice([0, 0, 1, rng.randint(2, 40), rng.randint(41, 3000)])
    print(f"D {D} H {H} G {G} {dtype} q {q_dtype} {fp32_dot} window {window} page {page} lens {lens} workers {workers}", flush=True)
    c = Case(lens, H, G, D, page, dtype, seed, q_dtype, fill=float("nan"))
    for ws in (True, False):
        c.o.fill_(777.0)
        c.run(paged, ws, workers, window_size=window, use_fp32_dot=fp32_dot).check(window, q_dtype is not None and not fp32_dot)


def test_offsets_past_32_bits(paged):
    """A pool of more than 8 GiB whose pages at both ends belong to one sequence."""
    G, page, D = 2, 256, 256
    P = (9 << 30) // (G * page * D * 2)
    k = torch.zeros(P, G, page, D, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    c = Case([700, 300], 8, G, D, page, seed=6)
    far = [0, P - 1, P // 2, P - 2, 1]
    order = torch.arange(c.k.shape[0])
    new = torch.tensor(far + list(range(10, 10 + c.k.shape[0] - len(far))))[: c.k.shape[0]]
    k[new], v[new] = c.k[order], c.v[order]
    t = c.tables.long().cpu()
    c.tables = torch.where(t >= 0, new[t.clamp(0)], t).int().cuda()
    c.k, c.v = k, v
    c.run(paged).check()
    c.o.fill_(0)
    c.run(paged, window_size=400).check(400)


def test_captured_and_replayed(paged):
    c = Case([900, 900, 900], 8, 2, 256, 16, seed=7)
    n = paged.paged_workspace_bytes(3, 8, 2, 256)
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    eager = torch.empty_like(c.o)

    def call(o, w):
        paged.paged_attention(c.q, c.k, c.v, o, c.tables, c.len_t, scale=1 / 16, workspace=w)

    call(c.o, ws[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(c.o, ws[0])
    for lens in ([1, 2, 3], [900, 0, 31], [450, 451, 452], [0, 0, 0], [16, 900, 32], [17, 33, 65]):
        c.len_t.copy_(torch.tensor(lens, dtype=torch.int32))
        c.q.add_(0.01)
        c.o.fill_(777.0), eager.fill_(777.0)
        graph.replay()
        call(eager, ws[1])
        torch.cuda.synchronize()
        assert torch.equal(c.o, eager), lens


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("o_dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["f16", "bf16", "f32"])
def test_result_types(paged, D, o_dtype):
    c = Case([1000, 0, 33], 8, 2, D, 32, torch.bfloat16, seed=15)
    c.o = torch.full((3, 8, D), 777.0, dtype=o_dtype, device="cuda")
    for ws in (True, False):
        c.run(paged, ws).check()
        c.run(paged, ws, window_size=100).check(100)


def test_two_recorded_launches_with_a_workspace_each(paged):
    """Two graphs on streams of their own, replayed beside an eager launch on a third workspace."""
    cases = [Case([700, 900, 40], 8, 2, 256, 16, seed=16 + i) for i in range(2)]
    n = paged.paged_workspace_bytes(3, 8, 2, 256)
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(3)]

    def call(c, o, w):
        paged.paged_attention(c.q, c.k, c.v, o, c.tables, c.len_t, scale=1 / 16, workspace=w)

    want = []
    for c in cases:
        call(c, c.o, ws[2])
        torch.cuda.synchronize()
        want.append(c.o.clone())
    graphs = [torch.cuda.CUDAGraph() for _ in cases]
    for graph, c, w in zip(graphs, cases, ws):
        with torch.cuda.graph(graph):
            call(c, c.o, w)
    side = torch.cuda.Stream()
    eager = torch.empty_like(cases[0].o)
    for step in range(6):
        for c in cases:
            c.o.fill_(777.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[step % 2].replay()
        graphs[1 - step % 2].replay()
        call(cases[0], eager, ws[2])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        for c, w in zip(cases, want):
            assert torch.equal(c.o, w), step


def test_no_sequences(paged):
    c = Case([16], 4, 2, 128, 16)
    paged.paged_attention(c.q[:0], c.k, c.v, c.o[:0], c.tables[:0], c.len_t[:0])
    torch.cuda.synchronize()
    assert bool((c.o == 777.0).all())


# ---- append --------------------------------------------------------------------------------------------------------


def append_reference(k, v, kp, vp, tables, offsets, cu, page, skip=(), k_rsos=None, v_rsos=None, eps=1e-6):
    kp, vp = kp.double().cpu().clone(), vp.double().cpu().clone()
    D = k.shape[2]
    for s, off in enumerate(offsets):
        for i, row in enumerate(range(cu[s], cu[s + 1])):
            pos = off + i
            if s in skip or pos < 0 or pos >= tables.shape[1] * page:
                continue
            pg = int(tables[s, pos // page])
            if not 0 <= pg < kp.shape[0]:
                continue
            for x, pool, rs in ((k, kp, k_rsos), (v, vp, v_rsos)):
                y = x[row].double().cpu()
                if rs is not None:
                    y = y / (rs[row].double().cpu()[:, None] / D + eps).sqrt()
                pool[pg, :, pos % page] = y
    return kp, vp


def same(got, ref, exact):
    """Bit for bit, or within one rounding of the pool's type on top of four fp32 roundings of the scaling."""
    g = got.double().cpu()
    if exact:
        assert torch.equal(g, ref)
    else:
        tol = (U16[got.dtype] + 6 * 2.0**-24) * ref.abs() + 1e-7
        assert bool(((g - ref).abs() <= tol).all())


@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("x_dtype,dtype", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16),
                                           (torch.float32, torch.float32), (torch.bfloat16, torch.float16)], ids=str)
@pytest.mark.parametrize("norm", [False, True])
def test_append(paged, page, x_dtype, dtype, norm):
    gen = torch.Generator().manual_seed(page)
    G, D = 2, 256
    lens, offsets = [5, 0, 1, 100, 17], [3, 40, 15, 30, 0]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    tables, P = make_tables([a + b for a, b in zip(lens, offsets)], page, gen)
    kp, vp = (torch.randn(P, G, page, D, generator=gen).to(dtype).cuda() for _ in range(2))
    T = cu[-1] + 3  # rows behind the last sequence belong to nobody
    kv = torch.randn(T, 2 * G, D, generator=gen).to(x_dtype).cuda()
    k, v = kv[:, :G], kv[:, G:]
    rs = dict(k_rsos=k.float().square().sum(-1), v_rsos=v.float().square().sum(-1)) if norm else {}
    ref = append_reference(k, v, kp, vp, tables, offsets, cu, page, **rs)
    off_t, cu_t = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (offsets, cu))
    paged.add_kv_to_pages(k, v, kp, vp, tables, off_t, 1e-6, **rs, cu_seqlens=cu_t)
    torch.cuda.synchronize()
    exact = not norm and (x_dtype == dtype)
    same(kp, ref[0], exact), same(vp, ref[1], exact)


@pytest.mark.parametrize("D", [8, 64, 512])
def test_append_one_row_each_and_what_is_dropped(paged, D):
    """One row per sequence: skipped phases, positions outside the table, absent pages, the last slot of a page."""
    gen = torch.Generator().manual_seed(D)
    G, page, N = 3, 16, 8
    tables, P = make_tables([48] * N, page, gen)
    tables[4, 1] = -1
    tables[5, 0] = P
    offsets = [0, 15, 47, 48, 20, 0, -1, 31]
    kp, vp = (torch.randn(P, G, page, D, generator=gen).half().cuda() for _ in range(2))
    k, v = (torch.randn(N, G, D, generator=gen).half().cuda() for _ in range(2))
    phase = torch.tensor([2, 2, 2, 2, 2, 2, 2, 1], dtype=torch.uint8, device="cuda")
    ref = append_reference(k, v, kp, vp, tables, offsets, list(range(N + 1)), page, skip=(7,))
    off_t = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    paged.add_kv_to_pages(k, v, kp, vp, tables, off_t, 1e-6, user_phase=phase, phase=2)
    torch.cuda.synchronize()
    same(kp, ref[0], True), same(vp, ref[1], True)
    before = kp.clone()
    paged.add_kv_to_pages(k[:0], v[:0], kp, vp, tables[:0], off_t[:0], 1e-6)
    torch.cuda.synchronize()
    assert torch.equal(before, kp)


# ---- the operators together -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("D,page,window", [(256, 16, None), (128, 48, 40), (512, 32, None), (64, 16, 30)])
def test_prompts_then_tokens(gpu_device, paged, D, page, window):
    """A server's path: pages for packed prompts, their attention and append, a fork, then tokens one at a time, a sequence
    that leaves, a compaction in between; every result against a token stream kept on the side."""
    from g4b_amd.kernels import packed, pages

    gen = torch.Generator().manual_seed(D + page)
    H, G, S, M, P = 8, 2, 5, 24, 60
    kp, vp = (torch.full((P, G, page, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    tables, lens, refs = torch.full((S, M), -1, dtype=torch.int32, device="cuda"), i32(*[0] * S), i32(*[0] * P)
    ws = torch.empty(pages.page_workspace_bytes(P, S), dtype=torch.uint8, device="cuda")
    aw = torch.empty(max(paged.paged_workspace_bytes(S, H, G, D), 16), dtype=torch.uint8, device="cuda")
    status = i32(0)
    stream = {s: [torch.zeros(0, G, D).half().cuda()] * 2 for s in range(S)}

    prompt = [37, 0, 100, 1, 0]
    cu = [0]
    for n in prompt:
        cu.append(cu[-1] + n)
    q, k, v = (torch.randn(cu[-1], n, D, generator=gen).half().cuda() for n in (H, G, G))
    o = torch.empty_like(q)
    pages.allocate_pages(tables, lens, refs, i32(*prompt), page, status, workspace=ws)
    assert status.item() == 0 and lens.tolist() == prompt
    paged.add_kv_to_pages(k, v, kp, vp, tables, lens - i32(*prompt), 1e-6, cu_seqlens=i32(*cu))
    packed.packed_attention(q, k, v, o, i32(*cu), scale=D**-0.5, query_window=window)
    torch.cuda.synchronize()
    for s in range(S):
        a, b = cu[s], cu[s + 1]
        stream[s] = [k[a:b], v[a:b]]
        if b > a:
            i = torch.arange(b - a)
            hidden = (i[None] > i[:, None]) | ((i[:, None] - i[None] >= window) if window else False)
            for h in range(H):
                ref, mag, qk = attend64(q[a:b, h], k[a:b, h // 4], v[a:b, h // 4], hidden, D**-0.5)
                check_attention(o[a:b, h], ref, mag, qk, b - a, D, torch.float16, what=f"prompt {s} head {h}")
    pages.fork_sequences(kp, vp, tables, lens, refs, i32(2, 0), i32(1, 4), status, workspace=ws)
    assert status.item() == 0
    stream[1], stream[4] = list(stream[2]), list(stream[0])
    for step in range(20):
        if step == 7:
            pages.free_sequences(tables, lens, refs, i32(0), page)
            stream[0] = [x[:0] for x in stream[0]]
        if step == 11:
            page_map, live = i32(*[0] * P), i32(0)
            pages.compact_pages(kp, vp, tables, lens, refs, page_map, live, workspace=ws)
            assert int((refs > 0).sum()) == live.item() and bool((refs[: live.item()] > 0).all())
        new = [0 if step >= 7 and s == 0 else 1 for s in range(S)]
        pages.allocate_pages(tables, lens, refs, i32(*new), page, status, workspace=ws)
        assert status.item() == 0
        q, k, v = (torch.randn(S, n, D, generator=gen).half().cuda() for n in (H, G, G))
        phase = torch.tensor([2 if n else 0 for n in new], dtype=torch.uint8, device="cuda")
        paged.add_kv_to_pages(k, v, kp, vp, tables, lens - 1, 1e-6, user_phase=phase, phase=2)
        o = torch.full_like(q, 777.0)
        paged.paged_attention(q, kp, vp, o, tables, lens, phase, 2, scale=D**-0.5, window_size=window, workspace=aw)
        torch.cuda.synchronize()
        for s in range(S):
            if not new[s]:
                assert bool((o[s] == 777.0).all())
                continue
            stream[s] = [torch.cat([old, x[s:s + 1]]) for old, x in zip(stream[s], (k, v))]
            n = stream[s][0].shape[0]
            hidden = (torch.arange(n) < n - window)[None].expand(4, n) if window else torch.zeros(4, n, dtype=torch.bool)
            for g in range(G):
                ref, mag, qk = attend64(q[s, 4 * g:4 * g + 4], stream[s][0][:, g], stream[s][1][:, g], hidden, D**-0.5)
                check_attention(o[s, 4 * g:4 * g + 4], ref, mag, qk, n, D, torch.float16, what=f"step {step} sequence {s}")


def test_append_and_copy_past_32_bits_on_another_stream(gpu_device, paged):
    """Pools of more than 8 GiB, rows to their last page and pages from there to the first, on a stream that is not the
    current one."""
    from g4b_amd.kernels import pages

    G, page, D = 2, 256, 256
    P = (9 << 30) // (G * page * D * 2)
    k, v = (torch.empty(P, G, page, D, dtype=torch.float16, device="cuda") for _ in range(2))
    for x in (k, v):
        x[[0, 1, P - 2, P - 1]] = 0
    rows = [torch.randn(page + 3, G, D, device="cuda").half() for _ in range(2)]
    tables = torch.tensor([[P - 1, 1], [P - 2, -1]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, page + 1, page + 3], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, page - 2], dtype=torch.int32, device="cuda")
    status, src, dst = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (0, P - 1, 0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    paged.add_kv_to_pages(*rows, k, v, tables, offsets, 1e-6, cu_seqlens=cu, stream=side)
    pages.copy_pages(k, v, src, dst, status, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    for x, pool in zip(rows, (k, v)):
        assert torch.equal(pool[P - 1].transpose(0, 1), x[:page]) and torch.equal(pool[0], pool[P - 1])
        assert torch.equal(pool[1, :, 0], x[page]) and not bool(pool[1, :, 1:].any())
        assert torch.equal(pool[P - 2, :, page - 2:].transpose(0, 1), x[page + 1:]) and not bool(pool[P - 2, :, :page - 2].any())
    assert status.item() == 0


@pytest.mark.parametrize("window", [None, 300])
def test_two_recorded_launches_share_a_workspace_in_turn(paged, window):
    """Recorded launches of different shapes that use one workspace, replayed one after the other on one stream."""
    a, b = Case([700, 900, 40], 8, 2, 256, 16, seed=18), Case([2500], 8, 2, 128, 32, seed=19)
    size = max(paged.paged_workspace_bytes(3, 8, 2, 256), paged.paged_workspace_bytes(1, 8, 2, 128))
    ws = torch.full((size,), 0x7F, dtype=torch.uint8, device="cuda")

    def call(c):
        paged.paged_attention(c.q, c.k, c.v, c.o, c.tables, c.len_t, scale=c.D**-0.5, workspace=ws, window_size=window)

    call(a), call(b)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, c in zip(graphs, (a, b)):
        with torch.cuda.graph(graph):
            call(c)
    for step in range(4):
        for c in (a, b):
            c.q.mul_(0.9), c.o.fill_(777.0)
        graphs[step % 2].replay()
        graphs[1 - step % 2].replay()
        torch.cuda.synchronize()
        a.check(window), b.check(window)
