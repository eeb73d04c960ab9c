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


@pytest.mark.parametrize("B,H,g,n,D", [(40, 3, 2, 1, 64), (700, 1, 2, 1, 64), (400, 1, 2, 5, 64), (3, 40, 2, 1, 128), (2, 160, 2, 2, 64),
                                       (33, 2, 2, 9, 128), (45, 2, 4, 20, 64), (600, 1, 4, 40, 64), (300, 1, 2, 12, 256), (2, 150, 4, 6, 128)])
def test_every_row_of_large_batches(B, H, g, n, D):
    """Batches that are planned in one pass or several, head counts around and above the number of SMs: every row that a request
    owns is written and right, request by request, and the rows of nobody keep what they held.  out and lse start as NaN,
    so that a row that is not written, or joined from parts that are not there, cannot pass."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(2200 + B + H)
    lens = torch.randint(n, 60, (B,), generator=gen).tolist() if n < 60 else [n] * B
    lens[B // 2] = 500
    counts = [0 if b % 7 == 3 else int(torch.randint(1, n + 1, (1,), generator=gen)) for b in range(B)]
    bt = Batch(lens, counts, H, g, D, 16, gen, tree=n > 1).dev()
    N, extra = bt.start[-1], 5
    q = torch.cat([bt.d_q, torch.full((extra, H * g, D), float("nan"), dtype=torch.bfloat16, device=DEV)])
    words = None if bt.d_words is None else torch.cat([bt.d_words, torch.full((extra,), -1, dtype=torch.int64, device=DEV)])
    out = torch.full((N + extra, H * g, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    lse = torch.full((N + extra, H * g), float("nan"), device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.attend_paged(q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, n, tree_mask=words, kv_axis=0, out=out, lse=lse, status=status)
    assert int(status) == 0
    out, lse = out.cpu(), lse.cpu()
    assert torch.isnan(out[N:].float()).all() and torch.isnan(lse[N:]).all()
    assert torch.isfinite(out[:N].float()).all() and torch.isfinite(lse[:N]).all()
    split_p = n * g <= 8
    for b in range(B):
        c, T = counts[b], lens[b]
        if c == 0:
            continue
        k, v = (x.double() for x in bt.tokens(b))
        see = oa.visible(T, c, None if bt.words is None else bt.words[bt.rows(b)])
        r = bt.q[bt.rows(b)].double().view(c, H, g, D)
        s = torch.einsum("nhgd,thd->nhgt", r, k) / D ** 0.5
        L = (torch.einsum("nhgd,thd->nhgt", r.abs(), k.abs()) / D ** 0.5).amax(-1)
        s = s.masked_fill(~see[:, None, None, :], float("-inf"))
        p = torch.softmax(s, -1)
        o, a = (torch.einsum("nhgt,thd->nhgd", p, x) for x in (v, v.abs()))
        ds = (D + 4) * 2.0 ** -23 * L
        z = torch.logsumexp(s, -1)
        lse_tol = ds + 2.0 ** -21 + T * 2.0 ** -24 + 2.0 ** -22 * z.abs()
        assert ((lse[bt.rows(b)].double().view(c, H, g) - z).abs() <= lse_tol).all(), b
        p_rel = 2 * ds + 2.0 ** -21 + T * 2.0 ** -24
        tol = 2.0 ** -8 * o.abs() + (p_rel[..., None] + (2.0 ** -16 if split_p else 2.0 ** -8)) * a + 1e-30
        assert ((out[bt.rows(b)].double().view(c, H, g, D) - o).abs() <= tol).all(), b
