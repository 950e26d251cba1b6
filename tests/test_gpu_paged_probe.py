"""The one launch over pages that waits for the device: the first that splits its keys over the flat tile list asks for the XCC
ids behind the weighted work shares.  A call that has no use for them does not ask.  The plan lines on stderr tell; the
library asks once per process, so this runs in a child process of its own."""

import os
import subprocess
import sys
import textwrap

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = textwrap.dedent("""
    import sys
    import torch
    sys.path.insert(0, %r)
    from g4b_amd.kernels import paged
    B, H, G, D, page, M = 80, 8, 2, 128, 16, 40
    q = torch.randn(B, H, D, device="cuda").half()
    o = torch.empty_like(q)
    k, v = (torch.randn(B * M, G, page, D, device="cuda").half() for _ in range(2))
    tables = torch.arange(B * M, device="cuda", dtype=torch.int32).view(B, M)
    lens = torch.full((B,), 600, dtype=torch.int32, device="cuda")
    ws = torch.empty(paged.paged_workspace_bytes(B, H, G, D), dtype=torch.uint8, device="cuda")
    for what, kw in (("unsplit", {}), ("window", dict(window_size=100, workspace=ws)), ("split", dict(workspace=ws))):
        print("call", what, file=sys.stderr, flush=True)
        paged.paged_attention(q, k, v, o, tables, lens, **kw)
    torch.cuda.synchronize()
    print("ok", flush=True)
""") % ROOT


def test_only_a_launch_over_the_flat_tile_list_asks(gpu_device):
    env = {k: v for k, v in os.environ.items() if k != "G4B_ATTN_XCD_SHARES"}
    res = subprocess.run([sys.executable, "-c", CHILD], env=dict(env, G4B_ATTN_PRINT_PLAN="1"), capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "ok" in res.stdout, res.stdout + res.stderr
    calls = res.stderr.split("call ")
    asked = {c.split()[0]: "XCC ids of workgroups" in c for c in calls[1:]}
    assert asked == {"unsplit": False, "window": False, "split": True}, res.stderr
