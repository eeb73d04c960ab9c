"""Values up to 2^127: a row's output is a mean of the values it sees, so it is finite where they are, whatever kernel serves
the call and wherever its reference lies.  Tolerances are those of test_gpu_attention.py (check_rows)."""
from __future__ import annotations

import pytest
import torch

from oracle import attention as oa
from test_gpu_attention import VARIANTS, Batch, check_rows, split

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,exponent", [("level", 126), ("steps", 126), ("steps", 100), ("steps", 70)])
@pytest.mark.parametrize("D,bs,g,n", VARIANTS)
def test_large_values_stay_finite(D, bs, g, n, shape, exponent):
    """Values of one sign and of size 2^exponent to 2^(exponent + 1).  "level": equal weights but for some noise, so that the sum
    of the values alone is far beyond fp32.  "steps": logits of 0 and of 38 (2^55) in turn, 128 tokens each."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(2100 + D + bs + n + exponent)
    T = 700
    bt = Batch([T], [n], 1, g, D, bs, gen, tree=n > 1)
    blk, off = oa.token_slots(bt.table[0].tolist(), bs, T)
    k, v = split(bt.cache[0], 0)
    bt.q[:] = 0
    bt.q[:, :, 0] = 16.0
    bt.q[:, :, 1:9] = (torch.randn((n, g, 8), generator=gen) * 0.3).to(torch.bfloat16)
    x = torch.where((torch.arange(T) // 128) % 2 == 1, 38.0, 0.0) if shape == "steps" else torch.zeros(T)
    k[blk, off, 0, 0] = (x / 16).to(torch.bfloat16)
    v[blk, off, 0] = ((1 + torch.rand((T, D), generator=gen, dtype=torch.float64) * 0.98) * 2.0 ** exponent).to(torch.bfloat16)
    bt.dev()
    out, lse = ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, n, tree_mask=bt.d_words, kv_axis=0, scale=1.0)
    assert torch.isfinite(out.float()).all()
    check_rows(bt, out, lse, n, 1.0)


@pytest.mark.parametrize("D,bs,g,n", VARIANTS)
def test_small_weights_count(D, bs, g, n):
    """Level logits but for three older tokens of 2^-100 of the others' weight: a value of 2^120 there adds 2^20 to its channel over 1400 tokens,
    and an infinite one makes its channel infinite."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(2400 + D + bs + n)
    T = 1400
    bt = Batch([T], [n], 1, g, D, bs, gen, tree=n > 1)
    blk, off = oa.token_slots(bt.table[0].tolist(), bs, T)
    k, v = split(bt.cache[0], 0)
    bt.q[:] = 0
    bt.q[:, :, 0] = 16.0
    k[blk, off, 0, 0] = 0
    for t, x in ((5, 2.0 ** 120), (700, 2.0 ** 110), (1001, -(2.0 ** 119))):
        k[blk[t], off[t], 0, 0] = -69.315 / 16
        v[blk[t], off[t], 0, t % 16] = x
    run = lambda: ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, n, tree_mask=bt.d_words, kv_axis=0, scale=1.0)  # noqa: E731
    bt.dev()
    out, lse = run()
    assert (out[:, :, 5] > 2.0 ** 8).all()
    check_rows(bt, out, lse, n, 1.0)
    v[blk[700], off[700], 0, 700 % 16] = float("inf")
    bt.dev()
    got, _ = run()
    assert (got[:, :, 700 % 16] == float("inf")).all()
    others = [d for d in range(D) if d != 700 % 16]
    assert torch.equal(got[:, :, others], out[:, :, others])
