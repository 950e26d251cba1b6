"""Launches of more workgroups than one dimension of a grid holds (2^32 threads): the plain kernels and the append take every
size that the documentation allows."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_packed_rows_of_the_plain_kernel(gpu_device):
    """16 777 312 (token, head) rows of one-token prompts: every result is the token's own value row."""
    from g4b_amd.kernels import packed

    H, D = 32, 8
    T = (1 << 24) // H + 3
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, v = (torch.randn(T, H, D, generator=gen, device="cuda").half() for _ in range(2))
    o = torch.full_like(v, 777.0)
    packed.packed_attention(q, q, v, o, torch.arange(T + 1, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(o, v)


def test_sequences_of_the_plain_kernel(gpu_device):
    """65535 sequences of 257 kv heads, one position each on one of three pages."""
    from g4b_amd.kernels import paged

    B, G, D, page = 65535, 257, 8, 16
    gen = torch.Generator(device="cuda").manual_seed(1)
    kp, vp = (torch.randn(3, G, page, D, generator=gen, device="cuda").half() for _ in range(2))
    tables = (torch.arange(B, device="cuda", dtype=torch.int32) % 3)[:, None].contiguous()
    q = torch.randn(B, G, D, generator=gen, device="cuda").half()
    o = torch.full_like(q, 777.0)
    paged.paged_attention(q, kp, vp, o, tables, torch.ones(B, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(o, vp[tables[:, 0].long(), :, 0])


def test_rows_of_the_append(gpu_device):
    """2^24 + 5 rows of a workgroup each (they overlap in memory, eight elements from one to the next): all but the last three
    of the first sequence's stand in front of position 0 and are dropped, the second sequence's 40 all go in."""
    from g4b_amd.kernels import paged

    G, D, page, T, last = 32, 64, 16, (1 << 24) + 5, 40
    gen = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(T * 8 + D, generator=gen, device="cuda").half().as_strided((T, G, D), (8, 0, 1)) for _ in range(2))
    kp, vp = (torch.full((6, G, page, D), 777.0, device="cuda").half() for _ in range(2))
    tables = torch.tensor([[4, 1, 0], [2, 5, 3]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, T - last, T], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([3 - (T - last), 0], dtype=torch.int32, device="cuda")
    paged.add_kv_to_pages(k, v, kp, vp, tables, offsets, 1e-6, cu_seqlens=cu)
    torch.cuda.synchronize()
    for pool, x in ((kp, k), (vp, v)):
        want = torch.full_like(pool, 777.0)
        want[4, :, :3] = x[T - last - 3:T - last].transpose(0, 1)
        for i in range(last):
            want[tables[1, i // page].long(), :, i % page] = x[T - last + i]
        assert torch.equal(pool, want)
