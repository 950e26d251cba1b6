"""Packed prompts: attention against a plain implementation in 64 bits, sequence by sequence (tests/paged_helpers.py has the
tolerance's derivation)."""

import random

import pytest
import torch

from paged_helpers import attend64, causal_hidden, check_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def packed(gpu_device):
    from g4b_amd.kernels import packed

    return packed


def inputs(T, H, G, D, dtype, seed, q_dtype=None, fused=False):
    gen = torch.Generator().manual_seed(seed)
    if fused:  # views into one projection's output, as a model has them
        qkv = torch.randn(T, H + 2 * G, D, generator=gen).to(dtype).cuda()
        q, k, v = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    else:
        q, k, v = (torch.randn(T, n, D, generator=gen).to(d).cuda() for n, d in ((H, q_dtype or dtype), (G, dtype), (G, dtype)))
    o = torch.full((T, H, D), 777.0, dtype=q_dtype or dtype, device="cuda")
    return q, k, v, o


def cu_of(lens, start=0):
    cu = [start]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda"), cu


def check(q, k, v, o, cu, window, scale, q_rounded=False, what="", seqs=None):
    H, G, D = q.shape[1], k.shape[1], q.shape[2]
    for s, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        if b == a or (seqs is not None and s not in seqs):
            continue
        hidden = causal_hidden(b - a, window)
        for h in range(H):
            g = h // (H // G)
            ref, mag, qk = attend64(q[a:b, h], k[a:b, g], v[a:b, g], hidden, scale)
            check_attention(o[a:b, h], ref, mag, qk, b - a, D, k.dtype, q_rounded, f"{what} sequence {s} head {h}")


def run(packed, q, k, v, o, cu, ws=True, **kw):
    T, H, D = q.shape
    n = packed.packed_workspace_bytes(T, cu.numel() - 1, H, k.shape[1], D) if ws else 0
    w = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda") if n else None
    packed.packed_attention(q, k, v, o, cu, workspace=w, **kw)
    torch.cuda.synchronize()


LENS = [[1], [2, 1], [0, 1, 0, 5, 0], [31, 32, 33], [64, 65, 63, 1], [130], [127, 0, 129, 300], [513, 7]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
def test_lengths(packed, lens, dtype, D, ws):
    cu, ends = cu_of(lens)
    q, k, v, o = inputs(ends[-1], 8, 2, D, dtype, seed=len(lens) * 100 + ends[-1])
    run(packed, q, k, v, o, cu, ws, scale=D**-0.5)
    check(q, k, v, o, ends, None, D**-0.5)


@pytest.mark.parametrize("window", [1, 2, 31, 64, 65, 200, 100000])
@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
def test_windows(packed, window, D, ws):
    cu, ends = cu_of([3, 260, 0, 97])
    q, k, v, o = inputs(ends[-1], 4, 1, D, torch.float16, seed=window)
    run(packed, q, k, v, o, cu, ws, scale=D**-0.5, query_window=window)
    check(q, k, v, o, ends, window, D**-0.5)


@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (2, 1), (8, 8), (16, 1), (32, 2), (6, 2), (5, 1), (128, 1)], ids=str)
@pytest.mark.parametrize("D", [128, 256, 512])
def test_head_layouts(packed, heads, D):
    H, G = heads
    cu, ends = cu_of([70, 1, 150])
    q, k, v, o = inputs(ends[-1], H, G, D, torch.bfloat16, seed=H * 10 + G)
    run(packed, q, k, v, o, cu, scale=D**-0.5)
    check(q, k, v, o, ends, None, D**-0.5)


@pytest.mark.parametrize("D", [8, 64, 80, 96, 200, 1024])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_other_head_dims(packed, D, dtype):
    cu, ends = cu_of([1, 66, 0, 40])
    q, k, v, o = inputs(ends[-1], 4, 2, D, dtype, seed=D)
    run(packed, q, k, v, o, cu, scale=D**-0.5, query_window=50)
    check(q, k, v, o, ends, 50, D**-0.5)


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("q_dtype,dtype", [(torch.float32, torch.float16), (torch.float32, torch.bfloat16),
                                           (torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16)], ids=str)
@pytest.mark.parametrize("fp32_dot", [False, True])
def test_query_types(packed, D, q_dtype, dtype, fp32_dot):
    cu, ends = cu_of([90, 200])
    q, k, v, o = inputs(ends[-1], 8, 2, D, dtype, seed=3, q_dtype=q_dtype)
    run(packed, q, k, v, o, cu, scale=D**-0.5, use_fp32_dot=fp32_dot)
    check(q, k, v, o, ends, None, D**-0.5, q_rounded=True)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_views_and_rows_outside_the_sequences(packed, D):
    """q, k and v as views of one buffer, o as a view of a wider one; rows before the first and behind the last sequence hold
    NaN and infinities and are neither read into a result nor written."""
    lens, start, behind = [100, 1, 0, 64, 37], 5, 70
    cu, ends = cu_of(lens, start)
    T = ends[-1] + behind
    q, k, v, _ = inputs(T, 8, 2, D, torch.float16, seed=11, fused=True)
    for x in (q, k, v):
        x[:start], x[ends[-1]:] = float("nan"), float("inf")
    wide = torch.full((T, 8, D + 8), 777.0, dtype=torch.float16, device="cuda")
    o = wide[:, :, :D]
    run(packed, q, k, v, o, cu, scale=D**-0.5)
    check(q, k, v, o, ends, None, D**-0.5)
    assert bool((wide[:start] == 777.0).all()) and bool((wide[ends[-1]:] == 777.0).all()) and bool((wide[:, :, D:] == 777.0).all())


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_a_sequence_of_nan_leaves_its_neighbours_alone(packed, D):
    lens = [40, 50, 60]
    cu, ends = cu_of(lens)
    q, k, v, o = inputs(ends[-1], 4, 2, D, torch.float16, seed=12)
    k[ends[1]:ends[2]] = float("nan")
    v[ends[1]:ends[2]] = float("inf")
    run(packed, q, k, v, o, cu, scale=D**-0.5)
    check(q, k, v, o, ends, None, D**-0.5, seqs=(0, 2))


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("n,window", [(70, None), (130, 40), (700, None), (700, 90)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("fp32_q", [False, True])
def test_hidden_rows_of_the_same_prompt_may_hold_anything(packed, D, n, window, dtype, fp32_q):
    """K and V rows that a row must not see (later ones, and those before its window) hold infinities and NaN: the rows that
    see none of them are right, whole tiles and tiles cut into spans alike, and the others are not finite where a value they
    see is not."""
    cu, ends = cu_of([n])
    q, k, v, o = inputs(n, 8, 2, D, dtype, seed=n, q_dtype=torch.float32 if fp32_q else None)
    bad = [n // 2, n // 2 + 1, n - 1] if window else [n - 7, n - 1]
    for j, x in zip(bad, (float("inf"), float("nan"), float("-inf"))):
        v[j, :, j % 5::5] = x
        k[j] = x
    run(packed, q, k, v, o, cu, scale=D**-0.5, query_window=window, use_fp32_dot=fp32_q)
    hidden = causal_hidden(n, window)
    clean = hidden[:, bad].all(1)
    assert 0 < int(clean.sum()) < n
    rows = clean.nonzero()[:, 0]
    if n > 200:  # the tiles around the bad rows, and a few others
        near = torch.zeros(n, dtype=torch.bool)
        for j in bad + [0, 64, n // 3]:
            near[max(j - 70, 0):j + (window or 0) + 70] = True
        rows = (clean & near).nonzero()[:, 0][::5]
    for h in range(8):
        g = h // 4
        ref, mag, qk = attend64(q[rows, h], k[:, g].nan_to_num(0, 0, 0), v[:, g].nan_to_num(0, 0, 0), hidden[rows], D**-0.5)
        check_attention(o[rows, h], ref, mag, qk, n, D, dtype, what=f"head {h}")
        assert not torch.isfinite(o[~clean.cuda(), h]).all(-1).any()


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_bad_starts_stay_inside_the_buffers(packed, D):
    """Starts below 0 and above T count as 0 and T: the rows of the other sequences are right."""
    q, k, v, o = inputs(100, 4, 2, D, torch.float16, seed=13)
    cu = torch.tensor([-5, 30, 60, 400], dtype=torch.int32, device="cuda")
    run(packed, q, k, v, o, cu, scale=D**-0.5)
    check(q, k, v, o, [0, 30, 60, 100], None, D**-0.5)


def test_nothing_to_do(packed):
    q, k, v, o = inputs(0, 4, 2, 128, torch.float16, seed=1)
    packed.packed_attention(q, k, v, o, torch.zeros(3, dtype=torch.int32, device="cuda"))
    q, k, v, o = inputs(7, 4, 2, 128, torch.float16, seed=1)
    packed.packed_attention(q, k, v, o, torch.zeros(1, dtype=torch.int32, device="cuda"))
    packed.packed_attention(q, k, v, o, torch.zeros(4, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert bool((o == 777.0).all())


@pytest.mark.parametrize("D", [128, 256, 512])
def test_many_sequences(packed, D):
    """More sequences than a wave has lanes, many of them empty."""
    gen = torch.Generator().manual_seed(9)
    lens = [int(x) for x in torch.randint(0, 40, (300,), generator=gen)]
    lens[7] = 333
    cu, ends = cu_of(lens)
    q, k, v, o = inputs(ends[-1], 2, 1, D, torch.bfloat16, seed=5)
    run(packed, q, k, v, o, cu, scale=D**-0.5)
    check(q, k, v, o, ends, None, D**-0.5)


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("big", [30.0, 1e4])
def test_large_scores(packed, D, big):
    """Scores so far apart that a single key takes all of the weight, and growing along the prompt (the running maximum has
    to move): the value rows are reproduced."""
    n = 200
    cu, ends = cu_of([n])
    q, k, v, o = inputs(n, 2, 1, D, torch.float16, seed=6)
    q[:], k[:] = 0.0, 0.0
    q[:, :, 0] = 1.0
    k[:, :, 0] = (torch.arange(n, device="cuda")[:, None] * (big / n)).half()
    run(packed, q, k, v, o, cu, scale=1.0)
    check(q, k, v, o, ends, None, 1.0)


@pytest.mark.parametrize("D", [128, 256])
def test_captured_and_replayed(packed, D):
    """A recorded launch follows the starts that the device holds at each replay."""
    T, H, G = 640, 8, 2
    q, k, v, o = inputs(T, H, G, D, torch.float16, seed=7)
    eager = o.clone()
    splits = [[640], [1, 639], [100, 200, 300], [0, 0, 640], [320, 320], [10, 20, 30]]
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    n = packed.packed_workspace_bytes(T, 3, H, G, D)
    ws = [torch.empty(max(n, 16), dtype=torch.uint8, device="cuda") for _ in range(2)]

    def starts(lens):
        lens = (lens + [0, 0, 0])[:3]
        return torch.tensor([0, lens[0], lens[0] + lens[1], sum(lens)], dtype=torch.int32, device="cuda")

    cu.copy_(starts(splits[0]))
    packed.packed_attention(q, k, v, o, cu, scale=0.1, workspace=ws[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed.packed_attention(q, k, v, o, cu, scale=0.1, workspace=ws[0])
    for lens in splits:
        cu.copy_(starts(lens))
        o.fill_(777.0), eager.fill_(777.0)
        graph.replay()
        packed.packed_attention(q, k, v, eager, cu, scale=0.1, workspace=ws[1])
        torch.cuda.synchronize()
        assert torch.equal(o, eager), lens


def test_on_another_stream(packed):
    cu, ends = cu_of([300, 20])
    q, k, v, o = inputs(320, 8, 2, 256, torch.float16, seed=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    packed.packed_attention(q, k, v, o, cu, scale=1 / 16, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    check(q, k, v, o, ends, None, 1 / 16)


@pytest.mark.parametrize("D,dtype", [(256, torch.float16), (128, torch.bfloat16), (512, torch.float16)], ids=str)
@pytest.mark.parametrize("window", [None, 300])
def test_long_prompt(packed, D, dtype, window):
    """A prompt of several thousand tokens next to short ones: a sample of its rows against the reference."""
    lens = [40, 4099, 3]
    cu, ends = cu_of(lens)
    H, G = 8, 2
    q, k, v, o = inputs(ends[-1], H, G, D, dtype, seed=21)
    run(packed, q, k, v, o, cu, scale=D**-0.5, query_window=window)
    check(q, k, v, o, ends, window, D**-0.5, seqs=(0, 2))
    a, n = ends[1], lens[1]
    rows = torch.tensor([0, 1, 31, 32, 33, 63, 64, 127, 128, 1000, 1023, 1024, 2047, 2500, 4000, 4095, 4096, 4097, 4098])
    hidden = causal_hidden(n, window)[rows]
    for h in range(H):
        g = h // (H // G)
        ref, mag, qk = attend64(q[a + rows, h], k[a:a + n, g], v[a:a + n, g], hidden, D**-0.5)
        check_attention(o[a + rows, h], ref, mag, qk, n, D, dtype, what=f"head {h}")


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("window", [None, 260])
def test_more_sequences_than_lanes_cut_into_spans(packed, D, window):
    lens = [1] * 40 + [700] + [2, 0] * 20
    cu, ends = cu_of(lens)
    q, k, v, o = inputs(ends[-1], 4, 1, D, torch.bfloat16, seed=31)
    run(packed, q, k, v, o, cu, scale=D**-0.5, query_window=window)
    check(q, k, v, o, ends, window, D**-0.5)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("lens", [[3, 60], [40, 800]], ids=str)
def test_nan_that_is_seen_is_not_lost(packed, D, lens):
    """A NaN in a query, a key or a value reaches the rows that see it, and no others."""
    cu, ends = cu_of(lens)
    q, k, v, o = inputs(ends[-1], 8, 2, D, torch.float16, seed=45)
    n = ends[-1]
    run(packed, q, k, v, o, cu, scale=D**-0.5)
    want = o.clone()
    q[5, 3] = float("nan")
    k[n - 30, 0] = float("nan")
    v[n - 20, 1] = float("nan")
    run(packed, q, k, v, o, cu, scale=D**-0.5)
    bad = torch.zeros(n, 8, dtype=torch.bool, device="cuda")
    bad[5, 3] = bad[n - 30:, :4] = bad[n - 20:, 4:] = True
    assert bool((torch.isfinite(o).all(-1) == ~bad).all())
    assert not bool(torch.isfinite(o[bad]).any())
    far = ~bad
    far[max(ends[1], n - 20 - 128):] = False  # (rows of the same query tile may be computed by another body)
    assert torch.equal(o[far], want[far])


@pytest.mark.parametrize("seed", range(48))
def test_random_prompts(packed, seed):
    """Head layouts, types, windows, gaps in front and behind, with and without a workspace, drawn at random."""
    rng = random.Random(seed)
    D = rng.choice([128, 128, 256, 256, 512, 64])
    G = rng.choice([1, 1, 2, 3])
    H = G * rng.choice([1, 2, 4, 8, 5])
    dtype = rng.choice([torch.float16, torch.bfloat16])
    q_dtype = rng.choice([None, None, torch.float32])
    fp32_dot = q_dtype is not None and rng.random() < 0.5
    window = rng.choice([None, None, rng.randint(1, 700)])
    lens = [rng.choice([0, 1, rng.randint(1, 70), rng.randint(1, 300), rng.randint(300, 1200)]) for _ in range(rng.randint(1, 5))]
    start, tail = rng.choice([0, rng.randint(1, 50)]), rng.choice([0, rng.randint(1, 200)])
    cu, ends = cu_of(lens, start)
    q, k, v, o = inputs(ends[-1] + tail, H, G, D, dtype, seed=seed, q_dtype=q_dtype)
    what = f"D {D} H {H} G {G} {dtype} q {q_dtype} {fp32_dot} window {window} lens {lens} start {start} tail {tail}"
    print(what, flush=True)
    for ws in (True, False):
        o.fill_(777.0)
        run(packed, q, k, v, o, cu, ws=ws, scale=D**-0.5, query_window=window, use_fp32_dot=fp32_dot)
        check(q, k, v, o, ends, window, D**-0.5, q_dtype is not None and not fp32_dot, what)
        assert bool((o[:start] == 777.0).all()) and bool((o[ends[-1]:] == 777.0).all())


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_offsets_past_32_bits(packed, D):
    """Rows of k, v, q and o that lie 16 MiB apart: the last ones are more than 4 GiB behind the first."""
    n, pitch = 300, 1 << 23
    cu, ends = cu_of([100, 200])
    near = inputs(n, 4, 1, D, torch.float16, seed=33)
    far = [torch.empty(n * pitch, dtype=torch.float16, device="cuda").as_strided(x.shape, (pitch, D, 1)) for x in near]
    for a, b in zip(far, near):
        a.copy_(b)
    run(packed, *far, cu, scale=D**-0.5)
    check(*near[:3], far[3], ends, None, D**-0.5)


def test_two_recorded_launches_with_a_workspace_each(packed):
    """Two graphs of launches that are cut into spans, replayed in turn with eager launches between them: each keeps its
    spans in its own workspace."""
    T, H, G, D = 1500, 8, 2, 256
    cu, _ = cu_of([1400, 100])
    sets = [inputs(T, H, G, D, torch.float16, seed=40 + i) for i in range(2)]
    size = packed.packed_workspace_bytes(T, 2, H, G, D)
    assert size > 0
    ws = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(3)]
    want = []
    for q, k, v, o in sets:
        packed.packed_attention(q, k, v, o, cu, scale=0.1, workspace=ws[2])
        torch.cuda.synchronize()
        want.append(o.clone())
    graphs = [torch.cuda.CUDAGraph() for _ in sets]
    for graph, (q, k, v, o), w in zip(graphs, sets, ws):
        with torch.cuda.graph(graph):
            packed.packed_attention(q, k, v, o, cu, scale=0.1, workspace=w)
    side = torch.cuda.Stream()
    eager = torch.empty_like(sets[0][3])
    for step in range(6):
        for q, k, v, o in sets:
            o.fill_(777.0)
        torch.cuda.synchronize()
        graphs[step % 2].replay()
        with torch.cuda.stream(side):
            graphs[1 - step % 2].replay()
        packed.packed_attention(*sets[0][:3], eager, cu, scale=0.1, workspace=ws[2])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        for (q, k, v, o), w in zip(sets, want):
            assert torch.equal(o, w), step


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("window", [None, 7, 48])
def test_thousands_of_sequences(packed, D, window):
    """More sequences than the threads of a workgroup hold at once, with long ones at both ends."""
    gen = torch.Generator().manual_seed(10)
    lens = [int(x) for x in torch.randint(0, 3, (2600,), generator=gen)]
    lens[3], lens[1024], lens[2599] = 150, 70, 200
    cu, ends = cu_of(lens)
    q, k, v, o = inputs(ends[-1], 2, 1, D, torch.float16, seed=51)
    run(packed, q, k, v, o, cu, scale=D**-0.5, query_window=window)
    check(q, k, v, o, ends, window, D**-0.5, seqs=set(range(0, 2600, 13)) | {3, 4, 1023, 1024, 1025, 2598, 2599})


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("o_dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["f16", "bf16", "f32"])
def test_result_types(packed, D, o_dtype):
    cu, ends = cu_of([90, 700])
    q, k, v, _ = inputs(790, 4, 2, D, torch.bfloat16, seed=52)
    o = torch.full((790, 4, D), 777.0, dtype=o_dtype, device="cuda")
    for ws in (True, False):
        run(packed, q, k, v, o, cu, ws=ws, scale=D**-0.5)
        check(q, k, v, o, ends, None, D**-0.5)


@pytest.mark.parametrize("D", [128, 256, 512])
def test_starts_with_a_stride_and_the_result_in_the_query_s_place(packed, D):
    cu, ends = cu_of([90, 33, 800])
    wide = torch.full((4, 3), -5, dtype=torch.int32, device="cuda")
    wide[:, 0] = cu
    q, k, v, _ = inputs(923, 8, 2, D, torch.float16, seed=53)
    o = q.clone()
    run(packed, o, k, v, o, wide[:, 0], scale=D**-0.5)
    check(q, k, v, o, ends, None, D**-0.5)


def test_two_recorded_launches_share_a_workspace_in_turn(packed):
    """Recorded launches of different shapes, cut into spans, that use one workspace, replayed in turn on one stream."""
    shapes = [([1400, 100], 256), ([900], 512)]
    sets = [(cu_of(lens), inputs(sum(lens), 8, 2, D, torch.float16, seed=60 + D)) for lens, D in shapes]
    ws = torch.full((max(packed.packed_workspace_bytes(sum(lens), len(lens), 8, 2, D) for lens, D in shapes),), 0x7F, dtype=torch.uint8, device="cuda")

    def call(cu, q, k, v, o):
        packed.packed_attention(q, k, v, o, cu, scale=q.shape[2]**-0.5, workspace=ws)

    graphs = []
    for (cu, _), t in sets:
        call(cu, *t)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(cu, *t)
    for step in range(4):
        for _, (q, k, v, o) in sets:
            q.mul_(0.9), o.fill_(777.0)
        graphs[step % 2].replay()
        graphs[1 - step % 2].replay()
        torch.cuda.synchronize()
        for (_, ends), (q, k, v, o) in sets:
            check(q, k, v, o, ends, None, q.shape[2]**-0.5)
