"""Launches whose grids would hold 2^32 threads or more are refused on the host, before the first of their kernels runs."""

import pytest

from test_paged_refusals import UNSUPPORTED, K, packed_block, paged_block, refused  # noqa: F401  (K is a fixture)


def strides(*s):
    import ctypes

    return (ctypes.c_int64 * len(s))(*s)


@pytest.mark.parametrize("D", [128, 256, 512])
def test_too_many_query_tiles_are_refused(K, D):  # noqa: F811
    """A query tile per one-token prompt and kv head: 2^25 of them, with T * H as well below 2^31."""
    n = 1 << 20
    refused("g4b_packed_attn", packed_block(), UNSUPPORTED, T=n, N=n, H=32, G=32, D=D, q_stride=strides(32 * D, D, 1),
            k_stride=strides(32 * D, D, 1), v_stride=strides(32 * D, D, 1), o_stride=strides(32 * D, D, 1))


@pytest.mark.parametrize("D,workspace,page_size", [(128, False, 16), (128, True, 16), (256, False, 16), (256, True, 16), (512, True, 16),
                                                   (128, True, 48), (256, True, 1008), (512, True, 1008)])
def test_too_many_pairs_are_refused(K, D, workspace, page_size):  # noqa: F811
    """65535 sequences of 257 kv heads, more than 2^24 pairs: fewer tiles than 2^31, more threads than 2^32, in the one-kernel
    variant and, where the pages hold more keys than that takes, in the kernel that joins the splits."""
    from g4b_amd.kernels import paged

    B, G = 65535, 257
    change = dict(B=B, H=G, G=G, D=D, page_size=page_size, max_pages=2, q_stride=strides(G * D, D, 1), o_stride=strides(G * D, D, 1),
                  k_page_stride=G * page_size * D, v_page_stride=G * page_size * D)
    if workspace:
        change.update(workspace=1 << 20, workspace_bytes=paged.paged_workspace_bytes(B, G, G, D))
    refused("g4b_paged_attn", paged_block(), UNSUPPORTED, **change)
