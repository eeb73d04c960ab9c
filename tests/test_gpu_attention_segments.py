"""Several segments in one CTA's run, batches whose rows are checked one by one, values near the end of the range: the
attention kernels where the tests of single requests cannot go wrong.  Tolerances are those of test_gpu_attention.py."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import attention as oa
from test_gpu_attention import DEV, Batch, split

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,g,big,small", [(64, 4, 40, 1), (128, 4, 64, 1), (64, 8, 20, 3), (128, 3, 50, 12)])
def test_infinite_drafts_in_consecutive_segments(D, g, big, small):
    """As many KV heads as SMs, so that one CTA has all segments of a head: requests of more than 128 rows (both groups of
    the tensor-core kernel) alternate with requests of few rows and few tokens, and every request's last draft holds infinities
    and NaN.  Its own rows get them, whatever the next segment holds; all other rows are as without."""
    from triattention_b200 import ops
    H, bs = 148, 16
    lens, counts = [300, 20, 170, 90, 140, 30], [big, small] * 3
    gen = torch.Generator().manual_seed(2000 + D + big)
    bt = Batch(lens, counts, H, g, D, bs, gen)
    # a star: a draft sees the context and itself, the first one's row besides that every second draft but the last
    bt.words = []
    for c in counts:
        bt.words += [(1 << i) | (0x5555555555555555 & ((1 << (c - 1)) - 1) if i == 0 else 0) for i in range(c)]
    run = lambda: ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, big, tree_mask=bt.d_words, kv_axis=0)  # noqa: E731
    bt.dev()
    want, wlse = run()
    assert torch.isfinite(want.float()).all() and torch.isfinite(wlse).all()
    _, v = split(bt.cache[0], 0)
    last = []
    for b in range(len(lens)):
        blk, off = oa.token_slots(bt.table[b].tolist(), bs, lens[b])
        v[blk[-1], off[-1], :, 3] = float("inf")
        v[blk[-1], off[-1], :, D - 2] = float("-inf")
        v[blk[-1], off[-1], :, D // 2] = float("nan")
        last.append(bt.start[b + 1] - 1)
    bt.dev()
    for _ in range(3):
        out, lse = run()
        assert torch.equal(lse, wlse)
        others = [i for i in range(bt.start[-1]) if i not in last]
        assert torch.equal(out[others], want[others])
        assert (out[last][:, :, 3] == float("inf")).all() and (out[last][:, :, D - 2] == float("-inf")).all()
        assert torch.isnan(out[last][:, :, D // 2].float()).all()
        rest = [d for d in range(D) if d not in (3, D // 2, D - 2)]
        assert torch.equal(out[last][:, :, rest], want[last][:, :, rest])
