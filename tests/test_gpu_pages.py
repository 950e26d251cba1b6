"""Page management against a model in plain Python: whole numbers and page contents have to be equal."""

import random

import pytest
import torch

pytestmark = pytest.mark.gpu
G, D = 2, 64


@pytest.fixture(scope="module")
def ops(gpu_device):
    from g4b_amd.kernels import pages

    return pages


def i32(vals):
    return torch.tensor(list(vals), dtype=torch.int32, device="cuda")


class Model:
    """What the operators are meant to do, one step after the other."""

    def __init__(self, S, M, P, page):
        self.S, self.M, self.P, self.page = S, M, P, page
        self.tables = [[-1] * M for _ in range(S)]
        self.lens, self.refs = [0] * S, [0] * P
        self.content = list(range(P))  # a page's contents, by a mark

    def held(self, n):
        return -(-n // self.page)

    def allocate(self, num_new):
        if any(n < 0 or self.lens[s] + n > self.M * self.page for s, n in enumerate(num_new)):
            return -1
        wants = [self.held(self.lens[s] + n) - self.held(self.lens[s]) for s, n in enumerate(num_new)]
        free = [p for p in range(self.P) if self.refs[p] == 0]
        if sum(wants) > len(free):
            return sum(wants) - len(free)
        for s, w in enumerate(wants):
            for e in range(w):
                p = free.pop(0)
                self.tables[s][self.held(self.lens[s]) + e] = p
                self.refs[p] = 1
            self.lens[s] += num_new[s]
        return 0

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < self.S:
                for e in range(self.held(self.lens[s])):
                    p = self.tables[s][e]
                    self.tables[s][e] = -1
                    if 0 <= p < self.P:
                        self.refs[p] = max(self.refs[p] - 1, 0)
                self.lens[s] = 0

    def fork(self, src, dst):
        if any(not (0 <= s < self.S and 0 <= d < self.S) for s, d in zip(src, dst)) or len(set(dst)) < len(dst):
            return -1
        if any(self.lens[d] for d in dst) or any(self.lens[s] > self.M * self.page for s in src):
            return -1
        before = [(self.lens[s], list(self.tables[s])) for s in src]
        part = [n % self.page > 0 and 0 <= row[n // self.page] < self.P for n, row in before]
        free = [p for p in range(self.P) if self.refs[p] == 0]
        if sum(part) > len(free):
            return sum(part) - len(free)
        for (n, row), d, tail in zip(before, dst, part):
            full = n // self.page
            self.tables[d][:full] = row[:full]
            for p in row[:full]:
                if 0 <= p < self.P:
                    self.refs[p] += 1
            if n % self.page:
                self.tables[d][full] = -1
            if tail:
                p = free.pop(0)
                self.tables[d][full], self.refs[p], self.content[p] = p, 1, self.content[row[full]]
            self.lens[d] = n
        return 0

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        to = [p for p in range(n) if self.refs[p] <= 0]
        frm = [p for p in range(n, self.P) if self.refs[p] > 0]
        page_map = [p if self.refs[p] > 0 else -1 for p in range(self.P)]
        for a, b in zip(frm, to):
            page_map[a] = b
            self.refs[b], self.refs[a], self.content[b] = self.refs[a], 0, self.content[a]
        for s in range(self.S):
            for e in range(self.held(self.lens[s])):
                p = self.tables[s][e]
                if 0 <= p < self.P and page_map[p] >= 0:
                    self.tables[s][e] = page_map[p]
        return n, page_map


class Device:
    def __init__(self, m, layers=1, dtype=torch.float16, gap=0):
        P, page = m.P, m.page
        elems = G * page * D
        self.bufs = [torch.zeros(layers, P, elems + gap, dtype=dtype, device="cuda") for _ in range(2)]
        mark = (torch.arange(P, device="cuda")[None, :, None] + 1000 * torch.arange(layers, device="cuda")[:, None, None]).expand(layers, P, elems)
        wave = torch.arange(elems, device="cuda") % 7
        for i, b in enumerate(self.bufs):
            b[:, :, :elems] = (mark % 509 + wave + 500 * i).to(dtype)
        self.start = [b.clone() for b in self.bufs]
        self.elems = elems
        pools = [b[:, :, :elems].unflatten(2, (G, page, D)) for b in self.bufs]
        self.k, self.v = pools if layers > 1 else [p[0] for p in pools]
        self.push(m)
        self.status = i32([-99])
        self.m = m

    def push(self, m):
        self.tables, self.lens, self.refs = torch.tensor(m.tables, dtype=torch.int32, device="cuda").view(m.S, m.M), i32(m.lens), i32(m.refs)

    def check(self, what=""):
        torch.cuda.synchronize()
        m = self.m
        assert self.lens.tolist() == m.lens, what
        assert self.refs.tolist() == m.refs, what
        assert self.tables.tolist() == m.tables, what
        live = [p for p in range(m.P) if m.refs[p] > 0]
        for now, start in zip(self.bufs, self.start):
            # what a page holds is a page of the start; free pages may hold anything
            assert torch.equal(now[:, live, : self.elems], start[:, [m.content[p] for p in live], : self.elems]), what
            assert bool((now[:, :, self.elems:] == 0).all()), what


def workspace(ops, m):
    return torch.full((ops.page_workspace_bytes(m.P, m.S),), 0x7F, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("S,M,P,page,layers,gap", [(1, 1, 1, 16, 1, 0), (3, 5, 9, 16, 2, 8), (12, 8, 50, 48, 1, 0), (70, 20, 600, 16, 3, 0),
                                                   (1500, 4, 5000, 32, 1, 0)], ids=str)
def test_a_server_in_random_steps(ops, S, M, P, page, layers, gap):
    rng = random.Random(S * P)
    m = Model(S, M, P, page)
    d = Device(m, layers, gap=gap)
    ws = workspace(ops, m)
    for step in range(24):
        kind = rng.choice(["allocate", "allocate", "fork", "free", "compact"])
        if kind == "allocate":
            new = [rng.choice([0, 0, 1, rng.randrange(1, 2 * page)]) if m.lens[s] + 2 * page <= M * page else 0 for s in range(S)]
            if rng.random() < 0.15:
                new[rng.randrange(S)] = rng.choice([-1, M * page + 1, (1 << 31) - 1])
            want = m.allocate(new)
            ops.allocate_pages(d.tables, d.lens, d.refs, i32(new), page, d.status, workspace=ws)
            assert d.status.item() == want, step
        elif kind == "fork":
            empty = [s for s in range(S) if not m.lens[s]]
            dst = rng.sample(empty, rng.randrange(min(len(empty), 40) + 1))
            src = [rng.randrange(S) for _ in dst]
            if dst and rng.random() < 0.2:
                if rng.random() < 0.5:
                    dst[0] = rng.choice([S, -1, dst[-1]])
                else:
                    src[-1] = rng.choice([S, -3])
            want = m.fork(src, dst)
            ops.fork_sequences(d.k, d.v, d.tables, d.lens, d.refs, i32(src), i32(dst), d.status, workspace=ws)
            assert d.status.item() == want, step
        elif kind == "free":
            seqs = [rng.randrange(-1, S + 1) for _ in range(rng.randrange(S // 2 + 2))]
            m.free(seqs)
            ops.free_sequences(d.tables, d.lens, d.refs, i32(seqs), page)
        else:
            page_map = i32([-7] * P)
            n, want_map = m.compact()
            ops.compact_pages(d.k, d.v, d.tables, d.lens, d.refs, page_map, d.status, workspace=ws)
            assert d.status.item() == n and page_map.tolist() == want_map, step
        d.check(f"step {step}: {kind}")


@pytest.mark.parametrize("P", [4095, 4096, 4097, 20000])
def test_lowest_pages_first_in_a_large_pool(ops, P):
    rng = random.Random(P)
    m = Model(3, 4096, P, 16)
    m.refs = [rng.choice([0, 0, 1, 3]) for _ in range(P)]
    d = Device(m)
    ws = workspace(ops, m)
    for new in ([16 * 1000, 5, 0], [1, 16 * 700, 17]):
        want = m.allocate(new)
        ops.allocate_pages(d.tables, d.lens, d.refs, i32(new), 16, d.status, workspace=ws)
        assert d.status.item() == want == 0
        d.check()
    ops.compact_pages(d.k, d.v, d.tables, d.lens, d.refs, i32([0] * P), d.status, workspace=ws)
    assert d.status.item() == m.compact()[0]
    d.check()


def test_too_few_pages_change_nothing(ops):
    m = Model(4, 8, 10, 16)
    d = Device(m)
    ws = workspace(ops, m)
    for new in ([40, 40, 40, 1], [161, 0, 0, 0], [16, 16, 16, 16]):
        want = m.allocate(new)
        ops.allocate_pages(d.tables, d.lens, d.refs, i32(new), 16, d.status, workspace=ws)
        assert d.status.item() == want
        d.check()
    assert m.lens == [40, 40, 40, 1]
    m.free([3]), ops.free_sequences(d.tables, d.lens, d.refs, i32([3]), 16)
    want = m.fork([0], [3])
    ops.fork_sequences(d.k, d.v, d.tables, d.lens, d.refs, i32([0]), i32([3]), d.status, workspace=ws)
    assert d.status.item() == want == 0  # the one free page
    d.check()
    m.free([3]), ops.free_sequences(d.tables, d.lens, d.refs, i32([3]), 16)
    m.refs[9] = 1
    d.refs[9] = 1
    want = m.fork([1], [3])
    ops.fork_sequences(d.k, d.v, d.tables, d.lens, d.refs, i32([1]), i32([3]), d.status, workspace=ws)
    assert d.status.item() == want == 1
    d.check()


def test_absent_pages_stay_absent(ops):
    m = Model(4, 4, 12, 16)
    m.lens = [64, 40, 0, 0]
    m.tables[0] = [3, -1, 12, 5]
    m.tables[1] = [7, 2, -5, -1]
    m.refs = [0, 0, 1, 1, 0, 1, 0, 1, 0, 0, 0, 0]
    d = Device(m)
    ws = workspace(ops, m)
    assert m.fork([0, 1], [2, 3]) == 0
    ops.fork_sequences(d.k, d.v, d.tables, d.lens, d.refs, i32([0, 1]), i32([2, 3]), d.status, workspace=ws)
    assert d.status.item() == 0
    d.check("fork")
    m.compact(), ops.compact_pages(d.k, d.v, d.tables, d.lens, d.refs, i32([0] * 12), d.status, workspace=ws)
    d.check("compact")
    m.free([0, 0, 2, 99, 3]), ops.free_sequences(d.tables, d.lens, d.refs, i32([0, 0, 2, 99, 3]), 16)
    d.check("free")


def test_sources_are_read_as_they_were(ops):
    """A chain 0 -> 1 -> 2 where 1 is empty: 2 becomes a copy of the empty sequence."""
    m = Model(3, 4, 12, 16)
    assert m.allocate([39, 0, 0]) == 0
    d = Device(m)
    ws = workspace(ops, m)
    assert m.fork([0, 1], [1, 2]) == 0
    ops.fork_sequences(d.k, d.v, d.tables, d.lens, d.refs, i32([0, 1]), i32([1, 2]), d.status, workspace=ws)
    d.check()


@pytest.mark.parametrize("layers,page,dtype", [(1, 16, torch.float16), (3, 256, torch.bfloat16), (2, 48, torch.float32)], ids=str)
def test_copy(ops, layers, page, dtype):
    P = 40
    m = Model(1, 1, P, page)
    d = Device(m, layers, dtype, gap=16)
    src = [0, 5, 7, 9, 9, 20, -1, 3, 21, 30, 6, 33]
    dst = [10, 11, 5, 12, 13, 20, 14, P, 10, 31, 32, 30]
    #      ok  ok  11 reads 5: dropped ..., 20 -> 20 moves nothing, two outside, 10 named before, 33 -> 30 is read by 30 -> 31
    dropped = 5
    want = [s.clone() for s in d.start]
    for s, t in zip(src, dst):
        if 0 <= s < P and 0 <= t < P and (s, t) not in ((7, 5), (21, 10), (33, 30)):
            for w, b in zip(want, d.start):
                w[:, t, : d.elems] = b[:, s, : d.elems]
    d.status.fill_(3)
    ops.copy_pages(d.k, d.v, i32(src), i32(dst), d.status)
    torch.cuda.synchronize()
    assert d.status.item() == 3 + dropped
    for w, b in zip(want, d.bufs):
        assert torch.equal(w, b)


def test_copy_a_long_list(ops):
    m = Model(1, 1, 2 * ops.MAX_LIST, 16)
    d = Device(m)
    order = torch.randperm(2 * ops.MAX_LIST, generator=torch.Generator().manual_seed(1))
    src, dst = order[: ops.MAX_LIST], order[ops.MAX_LIST:]
    d.status.zero_()
    ops.copy_pages(d.k, d.v, src.int().cuda(), dst.int().cuda(), d.status)
    torch.cuda.synchronize()
    assert d.status.item() == 0
    for now, start in zip(d.bufs, d.start):
        assert torch.equal(now[:, dst], start[:, src]) and torch.equal(now[:, src], start[:, src])


def test_captured_and_replayed(ops):
    """A round of page management recorded once and replayed on changing tables."""
    rng = random.Random(5)
    S, M, P, page = 20, 6, 90, 16
    m = Model(S, M, P, page)
    d = Device(m, 2)
    ws = workspace(ops, m)
    seqs, src, dst, new, page_map = i32([0] * 3), i32([0] * 3), i32([0] * 3), i32([0] * S), i32([0] * P)
    st = i32([0] * 3)

    def call():
        ops.free_sequences(d.tables, d.lens, d.refs, seqs, page)
        ops.fork_sequences(d.k, d.v, d.tables, d.lens, d.refs, src, dst, st[0:1], workspace=ws)
        ops.allocate_pages(d.tables, d.lens, d.refs, new, page, st[1:2], workspace=ws)
        ops.compact_pages(d.k, d.v, d.tables, d.lens, d.refs, page_map, st[2:3], workspace=ws)

    dst.fill_(-1)  # (refused: the run before the recording changes nothing)
    seqs.fill_(-1)
    call()
    torch.cuda.synchronize()
    m.compact()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(12):
        a = rng.sample(range(S), 3)
        b = [rng.randrange(S) for _ in range(3)]
        grow = [rng.choice([0, 1, 9, 20]) if m.lens[s] + 40 <= M * page and s not in a else 0 for s in range(S)]
        seqs.copy_(i32(a)), src.copy_(i32(b)), dst.copy_(i32(a)), new.copy_(i32(grow))
        graph.replay()
        m.free(a)
        want = [m.fork(b, a), m.allocate(grow), m.compact()[0]]
        assert st.tolist() == want, step
        d.check(f"step {step}")


def test_more_chunks_than_one_dimension_of_a_grid(ops):
    """8192 pairs of 2 MiB pages: more than 2^24 workgroups along one dimension if the pairs were laid out along it, too.
    Most pairs are of a page with itself and move nothing."""
    P, page, heads, wide = 6, 256, 16, 256
    k, v = (torch.randint(-99, 99, (9, P, heads, page, wide), dtype=torch.int16, device="cuda").to(torch.float16) for _ in range(2))
    n = ops.MAX_LIST
    src, dst = [0] * n, [0] * n
    src[5], dst[5], src[n - 1], dst[n - 1] = 1, 4, 2, 5
    want = [x.clone() for x in (k, v)]
    for x in want:
        x[:, 4], x[:, 5] = x[:, 1], x[:, 2]
    status = i32([0])
    ops.copy_pages(k, v, i32(src), i32(dst), status)
    assert status.item() == 0 and torch.equal(k, want[0]) and torch.equal(v, want[1])
