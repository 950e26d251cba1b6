"""The paged key-value cache's operators and the packed prompts' attention, as cases to be measured.

Four operators: attention of one new token per sequence over a paged cache ("decode"), causal attention over packed
prompts of different lengths ("prompts"), the append of new K and V rows into pages ("append") and a round of page
management between two steps ("pages").  ``run`` computes each in plain torch operations, or, where ``own`` is true,
with this package's kernels.
"""

import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # one sequence a step, a few thousand tokens in: a chat with a single user, all latency
        dict(name="decode_one_2k", op="decode", dtype="f16", batch=1, heads=8, kv_heads=2, head_dim=256, page=16,
             min_len=2047, max_len=2047, window=0),
        # a global layer of a full decode batch with contexts from short to long: the cache's whole stream from memory
        dict(name="decode_batch_64", op="decode", dtype="f16", batch=64, heads=8, kv_heads=2, head_dim=256, page=32,
             min_len=128, max_len=32768, window=0),
        # a sliding-window layer of such a batch
        dict(name="decode_window_512", op="decode", dtype="bf16", batch=64, heads=8, kv_heads=2, head_dim=256, page=16,
             min_len=1, max_len=32768, window=512),
        # a batch on wide heads
        dict(name="decode_d512", op="decode", dtype="bf16", batch=32, heads=8, kv_heads=2, head_dim=512, page=64,
             min_len=256, max_len=16384, window=0),
        # one short prompt: the time to a first token
        dict(name="prompt_short", op="prompts", dtype="f16", heads=8, kv_heads=2, head_dim=256, seqs=1, min_len=130,
             max_len=130, window=0, behind=0),
        # a step's worth of prompts of every length on narrow heads, in a buffer that is longer than they are
        dict(name="prompts_ragged", op="prompts", dtype="bf16", heads=16, kv_heads=4, head_dim=128, seqs=24, min_len=1,
             max_len=2048, window=0, behind=37),
        # a long document next to short prompts
        dict(name="prompt_8192", op="prompts", dtype="f16", heads=8, kv_heads=2, head_dim=256, seqs=3, min_len=60,
             max_len=8192, window=0, behind=0),
        # the same on a sliding-window layer
        dict(name="prompt_window_512", op="prompts", dtype="bf16", heads=8, kv_heads=2, head_dim=256, seqs=3, min_len=60,
             max_len=8192, window=512, behind=0),
        # one new token of each of 64 sequences
        dict(name="append_step_64", op="append", dtype="f16", kv_heads=2, head_dim=256, page=16, seqs=64, min_len=1,
             max_len=1, context=4096, norm=False),
        # a step's prompts, V normalised on its way into the cache
        dict(name="append_prompts", op="append", dtype="bf16", kv_heads=2, head_dim=256, page=32, seqs=24, min_len=1,
             max_len=4096, context=2048, norm=True),
        # a few sequences leave, fork and grow between two steps of a small server
        dict(name="pages_small", op="pages", dtype="f16", layers=1, kv_heads=2, head_dim=256, page=16, seqs=16,
             min_len=100, max_len=2048, copies=4),
        # the same in a full server, two layers' pools side by side: the pool is closed up again, most of it data moved
        dict(name="pages_large", op="pages", dtype="bf16", layers=2, kv_heads=2, head_dim=256, page=16, seqs=64,
             min_len=128, max_len=16384, copies=64),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompts", "prompts", "append", "pages"])
    dtype = rng.choice(["f16", "bf16"])
    kv_heads = rng.choice([1, 2, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 8])
    head_dim = rng.choice([128, 256, 256, 512])
    page = rng.choice([16, 32, 64, 128, 48])
    if op == "decode":
        batch = _log(rng, 1, 96)
        # keys of all sequences together, times what a key takes, stay below the largest listed batch
        most = 64 * 8192 * 1024 // (batch * kv_heads * head_dim)
        hi = _log(rng, 16, max(16, min(32768, most)))
        return dict(op=op, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                    min_len=_log(rng, 1, hi), max_len=hi, window=rng.choice([0, 0, _log(rng, 1, 2048)]))
    if op == "prompts":
        if heads > 16:
            heads, kv_heads = 16, min(kv_heads, 4)
        seqs = _log(rng, 1, 32)
        hi = _log(rng, 1, min(4096, 8192 // seqs * 2 * 256 // max(head_dim, 256)))
        return dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim, seqs=seqs,
                    min_len=_log(rng, 1, hi), max_len=hi, window=rng.choice([0, 0, _log(rng, 1, 1024)]),
                    behind=rng.choice([0, 0, rng.randrange(1, 200)]))
    if op == "append":
        seqs = _log(rng, 1, 128)
        hi = _log(rng, 1, min(4096, 12288 * 512 // (seqs * kv_heads * head_dim)) if seqs * kv_heads * head_dim < 12288 * 512 else 1)
        return dict(op=op, dtype=dtype, kv_heads=kv_heads, head_dim=head_dim, page=page, seqs=seqs,
                    min_len=_log(rng, 1, hi), max_len=hi, context=_log(rng, 1, 4096), norm=rng.random() < 0.5)
    seqs = _log(rng, 8, 64)
    hi = _log(rng, 40, max(40, min(8192, 64 * 4096 * 512 // (seqs * kv_heads * head_dim))))
    return dict(op=op, dtype=dtype, layers=rng.choice([1, 2]), kv_heads=kv_heads, head_dim=head_dim, page=page, seqs=seqs,
                min_len=_log(rng, 17, hi), max_len=hi, copies=_log(rng, 1, 64))


def _lengths(case, n):
    """The n lengths of a case, evenly spread between its least and its most, ends included (work() has to know them);
    prepare() shuffles their order."""
    lo, hi = case["min_len"], case["max_len"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


# ------------------------------------------------------------------------------------------------ inputs


def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _pool(gen, shape, dtype):
    """A pool of pages, filled layer by layer and part by part (the random numbers are drawn in 32 bits)."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for part in flat.split(1 << 27):
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda", dtype=torch.float32))
    return out


def _tables(rng, lens, page, num_pages, width):
    """Block tables that hold lens tokens a sequence, on pages in random order; what is not held is -1."""
    free = list(range(num_pages))
    rng.shuffle(free)
    rows = []
    for n in lens:
        held = -(-n // page)
        rows.append([free.pop() for _ in range(held)] + [-1] * (width - held))
    return rows


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case=case)
    dt = DTYPES[case["dtype"]]
    D, G = case["head_dim"], case["kv_heads"]
    if case["op"] == "decode":
        B, H, page = case["batch"], case["heads"], case["page"]
        lens = _lengths(case, B)
        rng.shuffle(lens)
        pages = [-(-n // page) for n in lens]
        num_pages, width = sum(pages) + 8, max(pages)
        st.update(q=_randn(gen, (B, H, D), dt), k=_pool(gen, (num_pages, G, page, D), dt),
                  v=_pool(gen, (num_pages, G, page, D), dt), o=torch.zeros(B, H, D, dtype=dt, device="cuda"),
                  tables=_i32(_tables(rng, lens, page, num_pages, width)), lens=_i32(lens))
        if own:
            from g4b_amd.kernels import paged

            st["workspace"] = torch.empty(paged.paged_workspace_bytes(B, H, G, D), dtype=torch.uint8, device="cuda")
    elif case["op"] == "prompts":
        N, H = case["seqs"], case["heads"]
        lens = _lengths(case, N)
        rng.shuffle(lens)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        T = cu[-1] + case["behind"]
        st.update(q=_randn(gen, (T, H, D), dt), k=_randn(gen, (T, G, D), dt), v=_randn(gen, (T, G, D), dt),
                  o=_randn(gen, (T, H, D), dt), cu=_i32(cu))
        if own:
            from g4b_amd.kernels import packed

            st["workspace"] = torch.empty(packed.packed_workspace_bytes(T, N, H, G, D), dtype=torch.uint8, device="cuda")
    elif case["op"] == "append":
        N, page = case["seqs"], case["page"]
        lens = _lengths(case, N)
        rng.shuffle(lens)
        before = [rng.randrange(case["context"] + 1) for _ in lens]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        after = [b + n for b, n in zip(before, lens)]
        num_pages = sum(-(-(n + case["context"]) // page) for n in lens) + 8  # whatever the contexts turn out to be
        width = max(-(-n // page) for n in after)
        st.update(k=_randn(gen, (cu[-1], G, D), dt), v=_randn(gen, (cu[-1], G, D), dt),
                  k_pages=_pool(gen, (num_pages, G, page, D), dt), v_pages=_pool(gen, (num_pages, G, page, D), dt),
                  tables=_i32(_tables(rng, after, page, num_pages, width)), cu=_i32(cu), offsets=_i32(before))
        # sums of squares of V's rows, as the projection before leaves them
        st["v_rsos"] = st["v"].float().square().sum(-1) if case["norm"] else None
    else:
        S, page, L = case["seqs"], case["page"], case["layers"]
        # a quarter of the slots is free, a quarter of the sequences leaves, a quarter forks into the free slots
        quarter = S // 4
        lens = _lengths(case, S - quarter)
        rng.shuffle(lens)
        lens += [0] * quarter
        grow = [rng.randrange(2 * page) for _ in lens]
        width = max(-(-n // page) for n in lens) + 2
        held = sum(-(-n // page) for n in lens)
        num_pages = held + held // 4 + 4 * S + 2 * case["copies"]
        rows = _tables(rng, lens, page, num_pages, width)
        used = [p for r in rows for p in r if p >= 0]
        order = list(range(S - quarter))
        rng.shuffle(order)
        refs = [0] * num_pages
        for p in used:
            refs[p] = 1
        spare = [p for p in range(num_pages) if not refs[p]]
        rng.shuffle(spare)
        into = spare[: case["copies"]]
        for p in into:  # pages that are kept without being in a table: a prefix that stays
            refs[p] = 1
        leave, fork = order[:quarter], order[quarter:2 * quarter]
        for s in leave:
            grow[s] = 0
        st.update(k_pages=_pool(gen, (L, num_pages, G, page, D), dt), v_pages=_pool(gen, (L, num_pages, G, page, D), dt),
                  tables=_i32(rows), lens=_i32(lens), refs=_i32(refs), leave=_i32(leave), src=_i32(fork),
                  dst=_i32(list(range(S - quarter, S))), grow=_i32(grow), copy_src=_i32([used[i % len(used)] for i in range(len(into))]),
                  copy_dst=_i32(into), status=_i32([0] * 4), page_map=_i32([0] * num_pages))
        if own:
            from g4b_amd.kernels import pages as page_ops

            st["workspace"] = torch.empty(page_ops.page_workspace_bytes(num_pages, S), dtype=torch.uint8, device="cuda")
    return st


# ------------------------------------------------------------------------------------------------ one pass


def run(st):
    return globals()["_own_" + st["case"]["op"] if own else "_plain_" + st["case"]["op"]](st)


def _scale(case):
    return 1.0 / math.sqrt(case["head_dim"])


def _own_decode(st):
    from g4b_amd.kernels import paged

    c = st["case"]
    paged.paged_attention(st["q"], st["k"], st["v"], st["o"], st["tables"], st["lens"], window_size=c["window"] or None,
                          scale=_scale(c), workspace=st["workspace"])
    return st["o"]


def _own_prompts(st):
    from g4b_amd.kernels import packed

    c = st["case"]
    packed.packed_attention(st["q"], st["k"], st["v"], st["o"], st["cu"], query_window=c["window"] or None, scale=_scale(c),
                            workspace=st["workspace"])
    return st["o"]


def _own_append(st):
    from g4b_amd.kernels import paged

    paged.add_kv_to_pages(st["k"], st["v"], st["k_pages"], st["v_pages"], st["tables"], st["offsets"], EPS, v_rsos=st["v_rsos"],
                          cu_seqlens=st["cu"])
    return st["k_pages"], st["v_pages"]


def _own_pages(st):
    from g4b_amd.kernels import pages as ops

    k, v, ws, status = st["k_pages"], st["v_pages"], st["workspace"], st["status"]
    tables, lens, refs = st["tables"].clone(), st["lens"].clone(), st["refs"].clone()
    page = st["case"]["page"]
    ops.copy_pages(k, v, st["copy_src"], st["copy_dst"], status[0:1])
    ops.free_sequences(tables, lens, refs, st["leave"], page)
    ops.fork_sequences(k, v, tables, lens, refs, st["src"], st["dst"], status[1:2], workspace=ws)
    ops.allocate_pages(tables, lens, refs, st["grow"], page, status[2:3], workspace=ws)
    ops.compact_pages(k, v, tables, lens, refs, st["page_map"], status[3:4], workspace=ws)
    return k, v, tables, lens, refs, st["page_map"], status


def _plain_decode(st):
    c = st["case"]
    k, v, lens = st["k"], st["v"], st["lens"].long()
    B, H, D = st["q"].shape
    P, G, page, _ = k.shape
    tables = st["tables"].long()
    width = tables.shape[1] * page

    def rows(pool):  # [B, G, width, D]
        return pool[tables.clamp_min(0)].float().permute(0, 2, 1, 3, 4).reshape(B, G, width, D)

    at = torch.arange(width, device=k.device)
    seen = at < lens[:, None]
    if c["window"]:
        seen = seen & (at >= lens[:, None] - c["window"])
    s = torch.matmul(st["q"].float().view(B, G, H // G, D), rows(k).transpose(-1, -2).contiguous()) * _scale(c)
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    e = (s - m.masked_fill(m == float("-inf"), 0.0)).exp()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, rows(v).masked_fill(~seen[:, None, :, None], 0.0)) / total.masked_fill(total == 0, 1.0)
    st["o"].copy_(o.view(B, H, D))
    return st["o"]


def _plain_prompts(st):
    c = st["case"]
    q, k, v, cu = st["q"], st["k"], st["v"], st["cu"].long()
    T, H, D = q.shape
    G = k.shape[1]
    n = T - c["behind"]
    at = torch.arange(n, device=q.device)
    seq = torch.searchsorted(cu[1:], at, right=True)
    seen = (seq[:, None] == seq[None]) & (at[None] <= at[:, None])
    if c["window"]:
        seen = seen & (at[:, None] - at[None] < c["window"])
    qf = q[:n].float().view(n, G, H // G, D).permute(1, 2, 0, 3).reshape(G, H // G * n, D)
    kf = k[:n].float().permute(1, 2, 0).contiguous()
    vf = v[:n].float().permute(1, 0, 2).contiguous()
    s = torch.matmul(qf, kf).view(G, H // G, n, n) * _scale(c)
    s = s.masked_fill_(~seen, float("-inf"))
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(G, H // G * n, n), vf).view(G, H // G, n, D) / total
    st["o"][:n] = o.permute(2, 0, 1, 3).reshape(n, H, D)
    return st["o"]


def _plain_append(st):
    c = st["case"]
    k, v, cu = st["k"], st["v"], st["cu"].long()
    page = c["page"]
    at = torch.arange(k.shape[0], device=k.device)
    seq = torch.searchsorted(cu[1:], at, right=True)
    pos = st["offsets"].long()[seq] + at - cu[seq]
    pages = st["tables"].long()[seq, pos // page]
    if c["norm"]:
        v = v.float() * (st["v_rsos"] / c["head_dim"] + EPS).rsqrt()[..., None]
    st["k_pages"][pages, :, pos % page] = k
    st["v_pages"][pages, :, pos % page] = v.to(st["v_pages"].dtype)
    return st["k_pages"], st["v_pages"]


def _plain_pages(st):
    k, v = st["k_pages"], st["v_pages"]
    page = st["case"]["page"]
    tables, lens, refs = st["tables"].long(), st["lens"].long(), st["refs"].long()
    status = st["status"]
    S, width = tables.shape
    slot = torch.arange(width, device=k.device)
    # copy
    k[:, st["copy_dst"].long()] = k[:, st["copy_src"].long()]
    v[:, st["copy_dst"].long()] = v[:, st["copy_src"].long()]
    # free
    leave = st["leave"].long()
    gone = torch.zeros(S, dtype=torch.bool, device=k.device)
    gone[leave] = True
    held = gone[:, None] & (slot < ((lens + page - 1) // page)[:, None])
    refs.scatter_add_(0, tables[held], torch.full_like(tables[held], -1))
    tables = tables.masked_fill(held, -1)
    lens = lens.masked_fill(gone, 0)
    # fork: whole pages are shared, the one that is still being filled is copied to the lowest free page
    src, dst = st["src"].long(), st["dst"].long()
    whole = lens[src] // page
    shared = slot < whole[:, None]
    refs.scatter_add_(0, tables[src][shared], torch.ones_like(tables[src][shared]))
    rows = torch.where(shared, tables[src], torch.full_like(tables[src], -1))
    part = (lens[src] % page > 0).nonzero()[:, 0]
    new = (refs == 0).nonzero()[: part.numel(), 0]
    old = tables[src[part], whole[part]]
    rows[part, whole[part]] = new
    refs[new] = 1
    k[:, new] = k[:, old]
    v[:, new] = v[:, old]
    tables[dst] = rows
    lens[dst] = lens[src]
    # grow: the lowest free pages, in the order of the sequences
    have, want = (lens + page - 1) // page, (lens + st["grow"].long() + page - 1) // page
    places = (slot >= have[:, None]) & (slot < want[:, None])
    number = int(places.sum())
    new = (refs == 0).nonzero()[:number, 0]
    tables[places] = new
    refs[new] = 1
    lens = lens + st["grow"].long()
    # compact: the live pages above the number of live pages move into the free ones below it, both in ascending order
    live = refs > 0
    count = live.sum()
    index = torch.arange(refs.numel(), device=k.device)
    high, low = (live & (index >= count)).nonzero()[:, 0], (~live & (index < count)).nonzero()[:, 0]
    k[:, low] = k[:, high]
    v[:, low] = v[:, high]
    page_map = torch.where(live, index, torch.full_like(index, -1))
    page_map[high] = low
    held = slot < ((lens + page - 1) // page)[:, None]
    tables = torch.where(held, page_map[tables.clamp_min(0)], tables)
    refs[low] = refs[high]
    refs[high] = 0
    st["page_map"].copy_(page_map)
    status.zero_()
    status[3] = count
    return k, v, tables.int(), lens.int(), refs.int(), st["page_map"], status


# ------------------------------------------------------------------------------------------------ what a pass needs


def _pairs(n, window):
    """(query, key) pairs of a causal prompt of n tokens."""
    w = min(window or n, n)
    return w * (w + 1) // 2 + (n - w) * w


def work(case):
    D, G = case["head_dim"], case["kv_heads"]
    if case["op"] == "decode":
        B, H = case["batch"], case["heads"]
        keys = sum(min(n, case["window"] or n) for n in _lengths(case, B))
        pages = sum(-(-min(n, case["window"] or n) // case["page"]) for n in _lengths(case, B))
        return {"bytes": keys * G * D * 4 + 2 * B * H * D * 2 + pages * 4 + B * 4, "flops": 4 * keys * H * D}
    if case["op"] == "prompts":
        lens, H = _lengths(case, case["seqs"]), case["heads"]
        return {"bytes": sum(lens) * (2 * H + 2 * G) * D * 2 + 4 * len(lens),
                "flops": 4 * D * H * sum(_pairs(n, case["window"]) for n in lens)}
    if case["op"] == "append":
        tokens = sum(_lengths(case, case["seqs"]))
        return {"bytes": tokens * G * D * 2 * 4 + (tokens * G * 4 if case["norm"] else 0), "flops": tokens * G * D if case["norm"] else 0}
    # pages: the copied, forked and moved pages are read and written once (of those above the live ones, the share that
    # the live pages have of the pool), the tables and counts once
    S, page = case["seqs"], case["page"]
    quarter = S // 4
    held = sum(-(-n // page) for n in _lengths(case, S - quarter))
    pool = held + held // 4 + 4 * S + 2 * case["copies"]
    live = held * 3 // 4 + case["copies"] + quarter + S
    moved = live * (pool - live) // pool if pool > live else 0
    page_bytes = 2 * case["layers"] * G * page * D * 2
    return {"bytes": 2 * (case["copies"] + quarter + moved) * page_bytes + 8 * (pool + S), "flops": 0}


# ------------------------------------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "decode":
        return _exact_decode(st)
    if case["op"] == "prompts":
        return _exact_prompts(st)
    if case["op"] == "append" and case["norm"]:
        return None, _exact_appended(st)
    return None  # pages are copied bit for bit


def _attend(q, k, v, scale, window, first):
    """softmax(scale q k^T) v in 64 bits for the rows of one kv head: q [R, n, D] at positions first .., k and v [m, D]."""
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    k, v = k.double(), v.double()
    keys = torch.arange(k.shape[0], device=q.device)
    for a in range(0, q.shape[1], 1024):
        b = min(a + 1024, q.shape[1])
        lo = max(0, first + a - window + 1) if window else 0
        hi = first + b
        pos = torch.arange(first + a, first + b, device=q.device)[:, None]
        hidden = keys[lo:hi] > pos
        if window:
            hidden = hidden | (keys[lo:hi] <= pos - window)
        w = torch.matmul(q[:, a:b].double(), k[lo:hi].t().contiguous()) * scale
        out[:, a:b] = torch.matmul(torch.softmax(w.masked_fill(hidden, float("-inf")), -1), v[lo:hi])
    return out


def _exact_decode(st):
    c = st["case"]
    o = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    G, R = c["kv_heads"], c["heads"] // c["kv_heads"]
    for b, n in enumerate(st["lens"].tolist()):
        if n:
            held = st["tables"][b, : -(-n // c["page"])].long()
            for g in range(G):
                k, v = (st[x][held, g].reshape(-1, c["head_dim"])[:n] for x in ("k", "v"))
                o[b, g * R:(g + 1) * R] = _attend(st["q"][b, g * R:(g + 1) * R, None], k, v, _scale(c), c["window"], n - 1)[:, 0]
    return o


def _exact_prompts(st):
    c = st["case"]
    o = st["o"].double()
    G, R = c["kv_heads"], c["heads"] // c["kv_heads"]
    ends = st["cu"].tolist()
    for a, b in zip(ends[:-1], ends[1:]):
        for g in range(G):
            q = st["q"][a:b, g * R:(g + 1) * R].transpose(0, 1)
            o[a:b, g * R:(g + 1) * R] = _attend(q, st["k"][a:b, g], st["v"][a:b, g], _scale(c), c["window"], 0).transpose(0, 1)
    return o


def _exact_appended(st):
    c = st["case"]
    pool = st["v_pages"].double()
    ends, before, tables = st["cu"].tolist(), st["offsets"].tolist(), st["tables"].tolist()
    for s, (a, b) in enumerate(zip(ends[:-1], ends[1:])):
        rows = st["v"][a:b].double() / (st["v_rsos"][a:b].double() / c["head_dim"] + EPS).sqrt()[..., None]
        done = 0
        while done < b - a:
            at = before[s] + done
            n = min(c["page"] - at % c["page"], b - a - done)
            pool[tables[s][at // c["page"]], :, at % c["page"]:at % c["page"] + n] = rows[done:done + n].transpose(0, 1)
            done += n
    return pool
