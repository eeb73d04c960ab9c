"""The public workspace sizes: what the wrappers take by themselves, and enough to hand in."""
from __future__ import annotations

import ctypes

import pytest
import torch

from triattention_b200 import _native, ops

GEOMETRIES = [(2, 2, 4, 128, 16, 50, 8), (1, 8, 4, 64, 5, 9, 3), (40, 3, 7, 256, 16, 700, 12), (3, 1, 64, 64, 1, 100, 30)]


def layout(B, H, g, D, bs, nb, width):
    return _native.PagedLayout(1, B, H, g, D, bs, nb, width, bs * H * D, H * D, D, 0, 0)


@pytest.mark.parametrize("geometry", GEOMETRIES)
def test_public_sizes_are_the_librarys(geometry):
    B, H, g, D, bs, nb, width = geometry
    lay = layout(*geometry)
    lib = _native.load()
    for mq, listed in ((1, 0), (7, 0), (64, 0), (1, 2), (8, 5)):
        n = ops.attend_workspace_bytes(lay, mq, listed)
        assert n == lib.triattn_attend_workspace_bytes(ctypes.byref(lay), mq, listed) > 0
        assert n == ops._attend_bytes(B, H, g, D, bs, nb, width, bs * H * D, H * D, D, mq, listed)
    assert ops.attend_workspace_bytes(lay, 65) == 0
    need = B * H * width * 4
    assert need <= ops.select_blocks_workspace_bytes(lay) < need + 256


@pytest.mark.gpu
@pytest.mark.parametrize("g,n,D,bs", [(4, 1, 128, 16), (4, 3, 64, 16), (4, 40, 128, 16), (8, 30, 64, 16), (4, 12, 64, 5)])
def test_buffers_of_exactly_these_sizes(g, n, D, bs):
    """Workspaces of the stated size, inside larger buffers whose other bytes are left alone; one byte less is refused."""
    from test_gpu_attention import DEV, Batch
    gen = torch.Generator().manual_seed(2300 + n)
    bt = Batch([900, 300], [n, max(1, n - 1)], 2, g, D, bs, gen, tree=n > 1).dev()
    args = (bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, n)
    want = ops.attend_paged(*args, tree_mask=bt.d_words, kv_axis=0)
    lay = layout(2, 2, g, D, bs, bt.nb, bt.width)
    size = ops.attend_workspace_bytes(lay, n)
    big = torch.full((size + 512,), 171, dtype=torch.uint8, device=DEV)
    out, lse = ops.attend_paged(*args, tree_mask=bt.d_words, kv_axis=0, workspace=big[256 : 256 + size])
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert (big[:256] == 171).all() and (big[256 + size :] == 171).all()
    with pytest.raises(_native.NativeLibraryError):
        ops.attend_paged(*args, tree_mask=bt.d_words, kv_axis=0, workspace=big[256 : 255 + size])
    bounds = torch.randn((bt.nb, 2, 2, D), generator=gen).sort(2).values.to(torch.bfloat16).to(DEV)
    sel = 1 + max(2, (n + bs - 2) // bs + 1) + 3
    pick = lambda **kw: ops.select_blocks(bt.d_q, bounds, bt.d_lens, bt.d_start, bt.d_table, n, bs, sel, **kw)  # noqa: E731
    size = ops.select_blocks_workspace_bytes(lay)
    big = torch.full((size + 512,), 171, dtype=torch.uint8, device=DEV)
    assert torch.equal(pick(workspace=big[256 : 256 + size]), pick())
    assert (big[:256] == 171).all() and (big[256 + size :] == 171).all()
    with pytest.raises(_native.NativeLibraryError):
        pick(workspace=big[256 : 255 + size])
