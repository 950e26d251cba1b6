"""Scores of minus infinity over packed prompts and pages: such a key has a weight of zero.  Rows with a finite score beside them
are those of the other keys, and rows with nothing else are zeros, in every kernel: whole tiles of 64 keys and whole pages of
such keys, spans and splits with nothing else, and rows that are computed again because of a value that another row of their
tile must not see.  Tolerances: tests/paged_helpers.py."""

import pytest
import torch

from paged_helpers import attend64, causal_hidden, check_attention, make_tables

pytestmark = pytest.mark.gpu
INF = float("inf")


def check_rows(o, q, k, v, hidden, dark, scale, what):
    """Rows o [n, D] against the reference with the keys of `dark` hidden; rows that see no other key are zeros."""
    hidden = hidden | dark.cpu()[None]
    ref, mag, qk = attend64(q, k.masked_fill(dark[:, None], 0.0), v, hidden, scale)
    check_attention(o, ref, mag, qk, hidden.shape[1], q.shape[1], k.dtype, what=what)
    assert bool((o[hidden.all(-1).cuda()] == 0.0).all()), f"{what}: rows of nothing but minus infinity"


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("dark", [(0, 1), (0, 130), (130, 400), (64, 1000)], ids=str)
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
@pytest.mark.parametrize("window", [None, 100], ids=["all", "window"])
def test_packed(gpu_device, D, dark, ws, window):
    from g4b_amd.kernels import packed

    H, G, lens = 4, 2, [70, 2048 if D == 128 else 1100]
    if D == 64 or window:
        lens = [70, 500]
    T = sum(lens)
    gen = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn(T, n, D, generator=gen).half().cuda() for n in (H, G, G))
    q[:, :, 5] = q[:, :, 5].abs() + 0.1
    gone = torch.zeros(T, dtype=torch.bool, device="cuda")
    gone[lens[0] + dark[0]:lens[0] + dark[1]] = True
    k[gone, :, 5] = -INF
    o = torch.full_like(q, 777.0)
    cu = torch.tensor([0, lens[0], T], dtype=torch.int32, device="cuda")
    n = packed.packed_workspace_bytes(T, 2, H, G, D) if ws else 0
    w = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda") if n else None
    packed.packed_attention(q, k, v, o, cu, scale=D**-0.5, query_window=window, workspace=w)
    torch.cuda.synchronize()
    for a, b in ((0, lens[0]), (lens[0], T)):
        for h in (0, H - 1):
            g = h * G // H
            check_rows(o[a:b, h], q[a:b, h], k[a:b, g], v[a:b, g], causal_hidden(b - a, window), gone[a:b], D**-0.5, f"rows {a}.. head {h}")


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
def test_packed_rows_computed_again(gpu_device, D, ws):
    from g4b_amd.kernels import packed

    H, G, T = 4, 2, 2048 if D == 128 else 1100
    gen = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn(T, n, D, generator=gen).half().cuda() for n in (H, G, G))
    q[:, :, 5] = q[:, :, 5].abs() + 0.1
    gone = torch.zeros(T, dtype=torch.bool, device="cuda")
    gone[:700] = True
    k[gone, :, 5] = -INF
    for t in (40, T - 1):  # only the last row of its tile, and of the prompt, sees the infinity
        v[t] = INF
    o = torch.full_like(q, 777.0)
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    n = packed.packed_workspace_bytes(T, 1, H, G, D) if ws else 0
    w = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda") if n else None
    packed.packed_attention(q, k, v, o, cu, scale=D**-0.5, workspace=w)
    torch.cuda.synchronize()
    clean = v.clone()
    clean[[40, T - 1]] = 0.0
    for h in (0, H - 1):  # (the rows behind 40 see an infinity with a weight of zero: not a number)
        g = h * G // H
        check_rows(o[:40, h], q[:40, h], k[:40, g], clean[:40, g], causal_hidden(40, None), gone[:40], D**-0.5, f"head {h}")
    assert not bool(torch.isfinite(o[T - 1]).any())


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
def test_packed_rows_computed_again_beside_a_dark_stretch(gpu_device, D, ws):
    """As above with nothing but the prompt's last value row infinite, so that all other rows of its tile are finite."""
    from g4b_amd.kernels import packed

    H, G, T = 4, 2, 2048 if D == 128 else 1100
    gen = torch.Generator().manual_seed(D + 1)
    q, k, v = (torch.randn(T, n, D, generator=gen).half().cuda() for n in (H, G, G))
    q[:, :, 5] = q[:, :, 5].abs() + 0.1
    gone = torch.zeros(T, dtype=torch.bool, device="cuda")
    gone[:700] = True
    k[gone, :, 5] = -INF
    clean = v.clone()
    v[T - 1] = INF
    o = torch.full_like(q, 777.0)
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    n = packed.packed_workspace_bytes(T, 1, H, G, D) if ws else 0
    w = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda") if n else None
    packed.packed_attention(q, k, v, o, cu, scale=D**-0.5, workspace=w)
    torch.cuda.synchronize()
    for h in (0, H - 1):
        g, m = h * G // H, T - 1
        check_rows(o[:m, h], q[:m, h], k[:m, g], clean[:m, g], causal_hidden(m, None), gone[:m], D**-0.5, f"head {h}")
    assert bool(torch.isinf(o[T - 1]).all())


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("H", [4, 32])
@pytest.mark.parametrize("ws", [False, True], ids=["unsplit", "workspace"])
@pytest.mark.parametrize("window", [None, 200], ids=["all", "window"])
def test_pages(gpu_device, D, H, ws, window):
    from g4b_amd.kernels import paged

    G, page, lens = 2, 32, [1500, 40, 300, 1]
    dark = [(0, 1000), (0, 40), (150, 300), (0, 1)]
    gen = torch.Generator().manual_seed(D)
    tables, P = make_tables(lens, page, gen)
    q = torch.randn(len(lens), H, D, generator=gen).half().cuda()
    q[:, :, 5] = q[:, :, 5].abs() + 0.1
    kp, vp = (torch.randn(P, G, page, D, generator=gen).half().cuda() for _ in range(2))
    for b, (lo, hi) in enumerate(dark):
        for j in range(lo, hi):
            kp[int(tables[b, j // page]), :, j % page, 5] = -INF
    o = torch.full_like(q, 777.0)
    n = paged.paged_workspace_bytes(len(lens), H, G, D) if ws else 0
    w = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda") if n else None
    paged.paged_attention(q, kp, vp, o, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), window_size=window,
                          scale=D**-0.5, workspace=w)
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        at, row = tables[b].long().repeat_interleave(page)[:n], torch.arange(n, device="cuda") % page
        gone = torch.zeros(n, dtype=torch.bool, device="cuda")
        gone[dark[b][0]:dark[b][1]] = True
        hidden = torch.zeros(H // G, n, dtype=torch.bool)
        if window:
            hidden[:, :max(0, n - window)] = True
        for g in range(G):
            hs = slice(g * (H // G), (g + 1) * (H // G))
            check_rows(o[b, hs], q[b, hs], kp[at, g, row], vp[at, g, row], hidden, gone, D**-0.5, f"sequence {b} head {g}")
