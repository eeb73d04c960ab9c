"""Attention over the paged cache, weight sums, eviction, block bounds and block choice against the 64-bit oracle.

Tolerances.  K, V and Q are bf16 and their products exact in fp32; a logit is a sum of D products accumulated in fp32, each
step off by at most 2^-23 of the running magnitude (tensor cores truncate), so |ds| <= D 2^-23 L with L = max_t scale sum_d |q_d k_td|, and two
more roundings of the base-2 exponent: ds := (D + 4) 2^-23 L.  A probability is then off by a factor exp(2 ds) (numerator and
denominator) and the exponential's 2^-21; fp32 sums over T tokens add T 2^-24 at most (64-token tiles, then
parts: T is an upper bound).  Rounding p to bf16 for the product with V (only above 8 rows per KV head) adds 2^-8 of sum p |v|,
two bf16 parts 2^-16.  The output's own rounding is 2^-8 of its value (half a step of bf16).
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import attention as oa

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make_cache(nb, bs, H, D, gen, axis=0, hnd=False, layers=1):
    inner = (H, bs, D) if hnd else (bs, H, D)
    outer = (2, nb) if axis == 0 else (nb, 2)
    big = torch.randn((layers, *outer, *inner), generator=gen).to(torch.bfloat16)
    return big.transpose(3, 4) if hnd else big


def split(cache, axis):
    return (cache[0], cache[1]) if axis == 0 else (cache[:, 0], cache[:, 1])


def to_dev(cache):
    """Device copy that keeps the strides."""
    out = torch.empty_strided(cache.shape, cache.stride(), dtype=cache.dtype, device=DEV)
    return out.copy_(cache)


class Batch:
    """Lengths, query counts, block tables and queries of a batch of requests, on the host and on the device."""

    def __init__(self, lens, counts, H, g, D, bs, gen, axis=0, hnd=False, layers=1, tree=False, extra=3):
        self.lens, self.counts, self.H, self.g, self.D, self.bs, self.axis = lens, counts, H, g, D, bs, axis
        B = len(lens)
        width = max(1, max((t + bs - 1) // bs for t in lens))
        nb = B * width + extra
        self.nb, self.width = nb, width
        self.table = torch.randperm(nb, generator=gen)[: B * width].view(B, width).to(torch.int32)
        self.cache = make_cache(nb, bs, H, D, gen, axis, hnd, layers)
        self.start = [0]
        for c in counts:
            self.start.append(self.start[-1] + c)
        self.q = (torch.randn((self.start[-1], H * g, D), generator=gen) * 1.5).to(torch.bfloat16)
        self.words = None
        if tree:
            self.words = []
            for c in counts:
                mine = []
                for i in range(c):
                    parent = int(torch.randint(-1, i, (1,), generator=gen)) if i else -1
                    mine.append((mine[parent] if parent >= 0 else 0) | (1 << i))
                self.words += mine

    def dev(self):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        self.d_cache = to_dev(self.cache)
        self.d_table, self.d_lens, self.d_start = self.table.to(DEV), i32(self.lens), i32(self.start)
        self.d_q = self.q.to(DEV)
        self.d_words = None
        if self.words is not None:
            self.d_words = torch.tensor([w - (1 << 64) if w >> 63 else w for w in self.words], dtype=torch.int64, device=DEV)
        return self

    def tokens(self, b, layer=0):
        k, v = split(self.cache[layer], self.axis)
        blk, off = oa.token_slots(self.table[b].tolist(), self.bs, self.lens[b])
        return k[blk, off], v[blk, off]

    def rows(self, b):
        return slice(self.start[b], self.start[b + 1])

    def expect(self, b, scale, chosen=None):
        k, v = self.tokens(b)
        n = self.counts[b]
        see = oa.visible(self.lens[b], n, None if self.words is None else self.words[self.rows(b)])
        if chosen is not None:
            see = see.expand(self.H, *see.shape).clone()
            for h in range(self.H):
                some = torch.zeros((self.lens[b] + self.bs - 1) // self.bs, dtype=torch.bool)
                some[[int(x) for x in chosen[b, h] if x >= 0]] = True
                see[h] &= some.repeat_interleave(self.bs)[: self.lens[b]]
        return oa.attend_request(self.q[self.rows(b)], k, v, see, scale)


def check_rows(bt, out, lse, max_q, scale, chosen=None, extra_tokens=0):
    out, lse = out.cpu(), lse.cpu()
    split_p = max_q * bt.g <= 8
    wanted = []
    for b in range(len(bt.lens)):
        if bt.counts[b] == 0:
            wanted.append(None)
            continue
        e = bt.expect(b, scale, chosen)
        wanted.append(e)
        got, glse = out[bt.rows(b)].double(), lse[bt.rows(b)].double()
        ds = (bt.D + 4) * 2.0 ** -23 * e["logit"]
        p_rel = 2 * ds + 2.0 ** -21 + bt.lens[b] * 2.0 ** -24
        empty = torch.isinf(e["lse"])
        assert torch.equal(torch.isinf(glse) & (glse < 0), empty)
        lse_tol = ds + 2.0 ** -21 + bt.lens[b] * 2.0 ** -24 + 2.0 ** -22 * e["lse"].abs().nan_to_num(0, 0, 0)
        assert ((glse - e["lse"]).abs()[~empty] <= lse_tol[~empty]).all()
        tol = 2.0 ** -8 * e["out"].abs() + (p_rel[..., None] + (2.0 ** -16 if split_p else 2.0 ** -8)) * e["spread"] + 1e-30
        assert ((got - e["out"]).abs() <= tol).all(), float(((got - e["out"]).abs() / tol).max())
        assert (got[empty] == 0).all()
    return wanted


CASES = [
    # lens, counts, H, g, D, bs, axis, hnd, tree
    ([1], [1], 1, 1, 64, 16, 0, False, False),                       # the first token of a sequence
    ([17], [1], 2, 4, 128, 16, 0, False, False),
    ([300, 64, 65, 1], [1, 1, 1, 1], 2, 4, 128, 16, 1, False, False),
    ([129, 40], [1, 1], 1, 8, 64, 8, 0, True, False),
    ([200, 77], [1, 1], 2, 3, 128, 5, 0, False, False),              # blocks of five tokens
    ([90], [1], 2, 16, 64, 32, 0, False, False),                     # 16 rows
    ([150, 33], [1, 1], 1, 64, 64, 16, 0, False, False),             # 64 heads to one KV head
    ([130, 9, 700], [7, 5, 3], 2, 4, 128, 16, 0, False, True),
    ([64, 64], [64, 64], 1, 1, 128, 16, 0, False, True),             # no context, every bit of the word
    ([513, 100], [64, 26], 1, 4, 64, 16, 1, False, True),            # 256 rows
    ([257], [33], 2, 8, 128, 64, 0, False, False),                   # a chain, 264 rows
    ([70, 0, 12], [2, 0, 12], 1, 2, 256, 16, 0, False, True),        # a request without query tokens
    ([500, 130], [9, 4], 1, 4, 256, 16, 0, False, False),
    ([40, 41], [1, 1], 2, 2, 128, 1, 0, False, False),               # token-granular pool
    ([2000] * 3, [1] * 3, 1, 4, 64, 16, 0, False, False),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_attend_against_oracle(case):
    from triattention_b200 import ops
    lens, counts, H, g, D, bs, axis, hnd, tree = CASES[case]
    gen = torch.Generator().manual_seed(100 + case)
    bt = Batch(lens, counts, H, g, D, bs, gen, axis, hnd, tree=tree).dev()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    mq = max(counts)
    out, lse = ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, mq, tree_mask=bt.d_words,
                                kv_axis=axis, status=status)
    assert int(status) == 0
    check_rows(bt, out, lse, mq, 1 / math.sqrt(D))


def test_attend_many_parts_and_repeatability():
    """One long request over all SMs: parts joined in a fixed order, twice the same bits."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(7)
    for counts, g in (([1], 4), ([6], 4)):
        bt = Batch([12345], counts, 1, g, 128, 16, gen, tree=counts[0] > 1).dev()
        run = lambda: ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, counts[0],  # noqa: E731
                                       tree_mask=bt.d_words, kv_axis=0, scale=0.05)
        out, lse = run()
        check_rows(bt, out, lse, counts[0], 0.05)
        again = run()
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_masked_places_do_not_leak():
    """NaN and infinities in slots behind the sequence, in free blocks, and in K / V of drafts a row does not see."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(11)
    for g, n in ((2, 4), (4, 8), (4, 20)):
        bt = Batch([61, 30], [n, 3], 2, g, 128, 16, gen, tree=True)
        # token n-1 of request 0 is seen by itself only
        for i in range(n - 1):
            assert not (bt.words[i] >> (n - 1)) & 1
        used = {int(x) for b in range(2) for x in bt.table[b, : (bt.lens[b] + 15) // 16]}
        for blk in range(bt.nb):
            if blk not in used:
                bt.cache[0][0][blk] = float("nan")
                bt.cache[0][1][blk] = float("inf")
        for b in range(2):
            last, off = int(bt.table[b, (bt.lens[b] - 1) // 16]), bt.lens[b] % 16
            if off:
                bt.cache[0][0][last, off:] = float("nan")
                bt.cache[0][1][last, off:] = float("-inf")
        good = bt.cache.clone()
        k, v = split(bt.cache[0], 0)
        blk, off = oa.token_slots(bt.table[0].tolist(), 16, 61)
        k[blk[-1], off[-1]] = float("nan")
        v[blk[-1], off[-1], :, :5] = float("inf")
        v[blk[-1], off[-1], :, 5:9] = float("nan")
        bad = bt.dev()
        out, lse = ops.attend_paged(bad.d_q, bad.d_cache[0], bad.d_table, bad.d_lens, bad.d_start, n, tree_mask=bad.d_words,
                                    kv_axis=0)
        bt.cache = good
        bt.dev()
        ref, rlse = ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, n, tree_mask=bt.d_words,
                                     kv_axis=0)
        keep = [i for i in range(bt.start[-1]) if i != n - 1]
        assert torch.equal(out[keep], ref[keep]) and torch.equal(lse[keep], rlse[keep])
        assert torch.isnan(out[n - 1].float()).all() and torch.isnan(lse[n - 1]).all()  # the row that sees the NaN key
        check_rows(bt, ref, rlse, n, 1 / math.sqrt(128))


def test_infinite_value_reaches_only_the_rows_that_see_it():
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(12)
    for g, n in ((2, 4), (4, 20)):
        bt = Batch([61], [n], 2, g, 128, 16, gen, tree=True)
        ref = bt.dev()
        want, _ = ops.attend_paged(ref.d_q, ref.d_cache[0], ref.d_table, ref.d_lens, ref.d_start, n, tree_mask=ref.d_words, kv_axis=0)
        k, v = split(bt.cache[0], 0)
        blk, off = oa.token_slots(bt.table[0].tolist(), 16, 61)
        v[blk[-1], off[-1], :, 3] = float("inf")
        v[blk[-1], off[-1], :, 64] = float("-inf")
        bt.dev()
        out, lse = ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, n, tree_mask=bt.d_words, kv_axis=0)
        assert torch.equal(out[: n - 1], want[: n - 1])
        assert (out[n - 1, :, 3] == float("inf")).all() and (out[n - 1, :, 64] == float("-inf")).all()
        others = [d for d in range(128) if d not in (3, 64)]
        assert torch.equal(out[n - 1][:, others], want[n - 1][:, others])
        assert torch.isfinite(lse).all()


def test_rows_that_see_nothing_and_rows_of_nobody():
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(13)
    bt = Batch([5, 20], [5, 2], 2, 2, 64, 16, gen, tree=True)
    bt.words = [0, 0b00010, 0, 0b11111, 0b10000, 0, 0b11]
    bt.dev()
    N = bt.start[-1]
    q = torch.cat([bt.d_q, torch.full((3, 4, 64), float("nan"), dtype=torch.bfloat16, device=DEV)])
    words = torch.cat([bt.d_words, torch.full((3,), -1, dtype=torch.int64, device=DEV)])
    out = torch.full((N + 3, 4, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((N + 3, 4), 7.0, device=DEV)
    ops.attend_paged(q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, 5, tree_mask=words, kv_axis=0, out=out, lse=lse)
    check_rows(bt, out[:N], lse[:N], 5, 1 / 8)
    assert (out[N:] == 7).all() and (lse[N:] == 7).all()
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()


def test_strided_query_output_and_cache():
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(14)
    H, g, D = 2, 2, 64
    bt = Batch([75, 18], [3, 1], H, g, D, 16, gen, tree=True).dev()
    # q, k, v in one row of a projection's output; the cache inside a wider pool
    packed = torch.zeros((4, H * g + 2 * H, D), dtype=torch.bfloat16, device=DEV)
    packed[:, : H * g] = bt.d_q
    wide = torch.zeros((2, bt.nb, 16, H + 3, D + 8), dtype=torch.bfloat16, device=DEV)
    wide[:, :, :, 1 : H + 1, :D] = bt.d_cache[0]
    out = torch.zeros((4, H * g, D + 16), dtype=torch.bfloat16, device=DEV)[:, :, 8 : D + 8]
    _, lse = ops.attend_paged(packed[:, : H * g], wide[:, :, :, 1 : H + 1, :D], bt.d_table, bt.d_lens, bt.d_start, 3,
                              tree_mask=bt.d_words, kv_axis=0, out=out)
    check_rows(bt, out, lse, 3, 1 / 8)


def test_bad_metadata_is_reported_and_skipped():
    from triattention_b200 import _native, ops
    gen = torch.Generator().manual_seed(15)
    bt = Batch([40, 33, 21], [1, 1, 1], 2, 2, 64, 16, gen).dev()

    def run(lens, start, table, mq=1, n=3, **kw):
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = torch.full((3, 4, 64), 7.0, dtype=torch.bfloat16, device=DEV)
        lse = torch.full((3, 4), 7.0, device=DEV)
        ops.attend_paged(bt.d_q, bt.d_cache[0], table, lens, start, mq, kv_axis=0, out=out, lse=lse, status=status, **kw)
        return out, lse, int(status)

    good = run(bt.d_lens, bt.d_start, bt.d_table)
    assert good[2] == 0
    # longer than the table row; fewer tokens than queries; a query range outside q: skipped, the others unharmed
    for lens, start in (([40, 4000, 21], [0, 1, 2, 3]), ([40, 0, 21], [0, 1, 2, 3]), ([40, -5, 21], [0, 1, 2, 3]),
                        ([40, 33, 21], [0, 1, 2, 9]), ([40, 33, 21], [0, 1, 2, -3])):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        out, lse, st = run(i32(lens), i32(start), bt.d_table)
        assert st == _native.DEV_BAD_LENGTH
        skipped = 1 if start == [0, 1, 2, 3] else 2
        for r in range(3):
            if r == skipped:
                assert (out[r] == 7).all() and (lse[r] == 7).all()
            else:
                assert torch.equal(out[r], good[0][r])
    # blocks outside the cache: their tokens are not seen
    for bad in (-1, bt.nb, 2 ** 31 - 1):
        table = bt.d_table.clone()
        table[0, 0] = bad
        out, lse, st = run(bt.d_lens, bt.d_start, table)
        assert st == _native.DEV_BAD_BLOCK_ID
        k, v = bt.tokens(0)
        e = oa.attend_request(bt.q[:1], k[16:], v[16:], torch.ones((1, 24), dtype=torch.bool), 1 / 8)
        assert (lse[0].cpu().double() - e["lse"]).abs().max() < 1e-4
        assert torch.equal(out[1:], good[0][1:])
    # a listed block behind the request's end
    blocks = torch.tensor([[[0, 1, 2], [0, 1, 77]], [[2, 1, 0]] * 2, [[0, 1, -1]] * 2], dtype=torch.int32, device=DEV)
    out, lse, st = run(bt.d_lens, bt.d_start, bt.d_table, block_list=blocks)
    assert st == _native.DEV_BAD_KEEP_INDEX
    assert torch.equal(out[2], good[0][2]) and torch.equal(out[0, :2], good[0][0, :2])


SUMS = [([50, 200], [1, 1], 2, 4, 128, 16, False, False, False), ([33, 90], [5, 12], 1, 4, 64, 16, False, True, False),
        ([300], [32], 2, 4, 128, 16, True, False, True), ([140], [64], 1, 3, 64, 8, False, True, True),
        ([70, 9], [3, 1], 1, 64, 256, 16, False, True, False), ([1], [1], 1, 1, 64, 16, False, False, False)]


@pytest.mark.parametrize("case", range(len(SUMS)))
def test_weight_sums(case):
    from triattention_b200 import ops
    lens, counts, H, g, D, bs, hnd, tree, reset = SUMS[case]
    gen = torch.Generator().manual_seed(200 + case)
    bt = Batch(lens, counts, H, g, D, bs, gen, 0, hnd, tree=tree).dev()
    before = torch.rand((bt.nb, H, bs), generator=gen)
    for b in range(len(lens)):  # whatever an earlier owner left in the query tokens' slots
        blk, off = oa.token_slots(bt.table[b].tolist(), bs, lens[b])
        before[blk[-counts[b]:], :, off[-counts[b]:]] = float("nan")
    sums = before.to(DEV)
    out, lse = ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, max(counts), tree_mask=bt.d_words,
                                kv_axis=0, weight_sums=sums, reset_weight_sums=reset)
    wanted = check_rows(bt, out, lse, max(counts), 1 / math.sqrt(D))
    got, touched = sums.cpu(), torch.zeros((bt.nb, bs), dtype=torch.bool)
    for b, e in enumerate(wanted):
        blk, off = oa.token_slots(bt.table[b].tolist(), bs, lens[b])
        touched[blk, off] = True
        old = before[blk, :, off].T.double()
        if reset:
            old = torch.zeros_like(old)
        old[:, lens[b] - counts[b]:] = 0
        new = got[blk, :, off].T.double()
        rel = (2 * (D + 4) * 2.0 ** -23 * e["logit"]).max() + 2.0 ** -20 + lens[b] * 2.0 ** -24 + (counts[b] * g) * 2.0 ** -24
        tol = rel * e["weight"] + 2.0 ** -23 * (old + e["weight"]) + 1e-30
        assert ((new - old - e["weight"]).abs() <= tol).all()
        if not reset:
            assert abs(float((new - old).sum()) - counts[b] * H * g) < 1e-2
    assert torch.equal(got.permute(0, 2, 1)[~touched].nan_to_num(9.0), before.permute(0, 2, 1)[~touched].nan_to_num(9.0))
    again = before.to(DEV)
    ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, max(counts), tree_mask=bt.d_words, kv_axis=0,
                     weight_sums=again, reset_weight_sums=reset)
    assert torch.equal(again.cpu().nan_to_num(9.0), got.nan_to_num(9.0))


EVICT = [
    # lens, keep, window, prefill, H, D, bs, hnd, layers
    ([100], [40], 8, None, 2, 128, 16, False, 2),
    ([300, 64, 7], [100, 64, 10], 16, [3, 0, 0], 1, 64, 16, True, 3),
    ([2500, 1300], [1024, 1030], 128, None, 2, 64, 16, False, 1),       # more than one pass of a CTA's threads
    ([90], [0], 4, None, 1, 64, 8, False, 1),
    ([1], [1], 0, None, 1, 64, 16, False, 1),
    ([65], [64], 100, None, 2, 72, 5, False, 1),                        # the window covers everything: lowest indices stay
    ([50000], [3000 - 17], 64, [5], 1, 64, 16, False, 1),               # row beyond the keys kept in shared memory
]


@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict_against_oracle(case):
    from triattention_b200 import ops
    lens, keep, window, prefill, H, D, bs, hnd, L = EVICT[case]
    gen = torch.Generator().manual_seed(300 + case)
    bt = Batch(lens, [0] * len(lens), H, 1, D, bs, gen, 0, hnd, layers=L).dev()
    sums = torch.rand((L, bt.nb, H, bs), generator=gen).square_()
    sums = torch.where(sums < 0.3, (sums * 20).round() / 20, sums)     # many equal values around the border
    if case == 1:
        sums[0, :, 0, 3] = float("nan")
        sums[1, :, 0, 2] = -0.0
    d_sums = sums.to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    view = ops.PagedCacheView.from_layers(list(bt.d_cache.unbind(0)), kv_axis=0)
    layout = view.layout(len(lens), 1, bt.width)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    pitch = max(max(keep), 1) + 2
    got = ops.evict_paged(view, layout, d_sums, bt.d_table, bt.d_lens, i32(keep), pitch, window,
                          None if prefill is None else i32(prefill), status=status).cpu()
    assert int(status) == 0
    want_cache, want_sums = bt.cache.clone(), sums.clone()
    for l in range(L):
        for b, T in enumerate(lens):
            blk, off = oa.token_slots(bt.table[b].tolist(), bs, T)
            for h in range(H):
                k = oa.evict_keep(sums[l, blk, h, off], keep[b], window, prefill[b] if prefill else 0)
                assert torch.equal(got[l, b, h, : len(k)], k)
                assert (got[l, b, h, len(k):] == -1).all()
                src = k.long()
                want_cache[l][:, blk[: len(k)], off[: len(k)], h] = bt.cache[l][:, blk[src], off[src], h]
                want_sums[l, blk[: len(k)], h, off[: len(k)]] = sums[l, blk[src], h, off[src]]
    assert torch.equal(bt.d_cache.cpu().view(torch.int16), want_cache.view(torch.int16))
    assert torch.equal(d_sums.cpu().view(torch.int32), want_sums.view(torch.int32))


@pytest.mark.parametrize("D,bs,hnd,axis", [(64, 16, False, 0), (128, 16, True, 1), (256, 8, False, 0), (128, 5, False, 1), (64, 1, False, 0)])
def test_block_bounds_and_choice(D, bs, hnd, axis):
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(400 + D + bs)
    H, g, L = 2, 4, 2
    lens, counts = [1000, 37, 1, 16 * bs, 64], [1, 3, 1, 5, 0]
    bt = Batch(lens, counts, H, g, D, bs, gen, axis, hnd, layers=L).dev()
    kall = bt.cache[:, 0] if axis == 0 else bt.cache[:, :, 0]
    view = ops.PagedCacheView.from_layers(list(bt.d_cache.unbind(0)), kv_axis=axis)
    layout = view.layout(len(lens), g, bt.width)
    before = torch.full((L, bt.nb, H, 2, D), 3.0, dtype=torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    first = [0, 20, 0, lens[3] - 1, 64]
    bounds = before.to(DEV)
    ops.update_block_bounds(view, layout, bounds, bt.d_table, torch.tensor(first, dtype=torch.int32, device=DEV), bt.d_lens, status=status)
    want = before.clone()
    for l in range(L):
        for b, T in enumerate(lens):
            blk, off = oa.token_slots(bt.table[b].tolist(), bs, T)
            lo, hi = oa.block_bounds(kall[l][blk, off], bs)
            for x in range(first[b] // bs, (T + bs - 1) // bs):
                want[l, bt.table[b, x], :, 0], want[l, bt.table[b, x], :, 1] = lo[x], hi[x]
    assert torch.equal(bounds.cpu(), want)
    zero = torch.zeros(len(lens), dtype=torch.int32, device=DEV)
    ops.update_block_bounds(view, layout, bounds, bt.d_table, zero, bt.d_lens, status=status)
    sel = 1 + max(2, (5 + bs - 2) // bs + 1) + 6
    got = ops.select_blocks(bt.d_q, bounds[1], bt.d_lens, bt.d_start, bt.d_table, 5, bs, sel, sink_blocks=1, recent_blocks=2,
                            status=status)
    assert int(status) == 0
    host = got.cpu()
    for b, T in enumerate(lens):
        if counts[b] == 0:
            assert (host[b] == -1).all()
            continue
        blk, off = oa.token_slots(bt.table[b].tolist(), bs, T)
        lo, hi = oa.block_bounds(kall[1][blk, off], bs)
        sc = oa.block_scores(bt.q[bt.rows(b)], lo, hi)
        assert torch.equal(host[b], oa.select_blocks(sc, T, counts[b], bs, sel, 1, 2)), b
    # and the attention over the chosen blocks of that layer
    bt.cache = bt.cache[1:]
    out, lse = ops.attend_paged(bt.d_q, bt.d_cache[1], bt.d_table, bt.d_lens, bt.d_start, 5, block_list=got, kv_axis=axis, status=status)
    assert int(status) == 0
    check_rows(bt, out, lse, 5, 1 / math.sqrt(D), host)


def test_equal_scores_take_the_lowest_blocks():
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(500)
    bt = Batch([640], [1], 1, 2, 64, 16, gen).dev()
    bounds = torch.zeros((bt.nb, 1, 2, 64), dtype=torch.bfloat16, device=DEV)
    bounds[:, :, 0] = -0.0          # zeros of both signs are equal scores
    bounds[int(bt.table[0, 30])] = 1.0
    bounds[int(bt.table[0, 20]), :, 1] = float("inf")
    q = bt.d_q.abs()
    got = ops.select_blocks(q, bounds, bt.d_lens, bt.d_start, bt.d_table, 1, 16, 8, sink_blocks=0, recent_blocks=2)
    assert got[0, 0].tolist() == [0, 1, 2, 3, 20, 30, 38, 39]


def test_offsets_beyond_32_bits():
    """A layer of more than 4 G elements: tokens of its last blocks are read and written where they are."""
    from triattention_b200 import ops
    H, D, bs = 8, 128, 16
    nb = (1 << 32) // (bs * H * D) + 40                       # elements per K half: just above 2^32
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB")
    cache = torch.zeros((2, nb, bs, H, D), dtype=torch.bfloat16, device=DEV)
    gen = torch.Generator().manual_seed(600)
    small = Batch([100], [1], H, 2, D, bs, gen).dev()
    table = torch.tensor([[nb - 1 - 3 * i for i in range(7)]], dtype=torch.int32, device=DEV)
    cache[:, table[0].long()] = small.d_cache[0][:, small.d_table[0].long()]
    out, lse = ops.attend_paged(small.d_q, cache, table, small.d_lens, small.d_start, 1)
    check_rows(small, out, lse, 1, 1 / math.sqrt(D))
    sums = torch.zeros((nb, H, bs), device=DEV)
    ops.attend_paged(small.d_q, cache, table, small.d_lens, small.d_start, 1, weight_sums=sums)
    assert abs(float(sums[table[0].long()].sum()) - 16) < 1e-3
    del cache, sums
    torch.cuda.empty_cache()


def test_two_streams_and_graph_replay():
    """Calls on two streams at once and a captured graph give what eager calls give."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(700)
    a, b = (Batch([3000, 500], [1, 1], 2, 4, 128, 16, gen).dev(), Batch([900, 2100], [8, 5], 2, 4, 128, 16, gen, tree=True).dev())
    run = lambda x, **kw: ops.attend_paged(x.d_q, x.d_cache[0], x.d_table, x.d_lens, x.d_start, max(x.counts),  # noqa: E731
                                           tree_mask=x.d_words, kv_axis=0, **kw)
    wa, wb = run(a), run(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            ga = run(a)
        with torch.cuda.stream(s2):
            gb = run(b)
        got.append((ga, gb))
    torch.cuda.synchronize()
    for ga, gb in got:
        assert torch.equal(ga[0], wa[0]) and torch.equal(gb[0], wb[0]) and torch.equal(gb[1], wb[1])
    sums = torch.zeros((a.nb, 2, 16), device=DEV)
    out, lse = torch.empty_like(wa[0]), torch.empty_like(wa[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(a, out=out, lse=lse, weight_sums=sums)
    eager = torch.zeros_like(sums)
    for step in range(3):
        a.d_lens -= 7          # the graph reads lengths from the device
        out.zero_()
        g.replay()
        want = run(a, weight_sums=eager)
        assert torch.equal(out, want[0]) and torch.equal(sums, eager)


# ------------------------------------------------------------------------------------------ every kernel variant
# (D, block size, rows): decode with split and plain probabilities, tree with one and two row tiles, the gathered general kernel
VARIANTS = [(64, 16, 4, 2), (128, 16, 4, 4), (128, 16, 7, 5), (64, 8, 3, 12), (128, 16, 9, 20), (64, 32, 4, 40),
            (256, 16, 4, 2), (256, 16, 2, 8), (256, 16, 8, 7), (128, 5, 4, 2), (128, 5, 2, 8), (64, 5, 4, 12), (64, 24, 8, 30)]


@pytest.mark.parametrize("D,bs,g,n", VARIANTS)
def test_hidden_drafts_do_not_leak_in_any_variant(D, bs, g, n):
    """The last draft is hidden from all other rows; its key is NaN, its value holds infinities and NaN."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(800 + D + bs + n)
    T = 140
    bt = Batch([T], [n], 2, g, D, bs, gen, tree=True)
    for i in range(n - 1):
        assert not (bt.words[i] >> (n - 1)) & 1
    run = lambda: ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, n, tree_mask=bt.d_words, kv_axis=0)  # noqa: E731
    bt.dev()
    want, wlse = run()
    check_rows(bt, want, wlse, n, 1 / math.sqrt(D))
    blk, off = oa.token_slots(bt.table[0].tolist(), bs, T)
    k, v = split(bt.cache[0], 0)
    clean = bt.cache.clone()
    v[blk[-1], off[-1], :, 3] = float("inf")
    v[blk[-1], off[-1], :, D - 1] = float("-inf")
    bt.dev()
    out, lse = run()
    assert torch.equal(out[: n - 1], want[: n - 1]) and torch.equal(lse, wlse)
    assert (out[n - 1, :, 3] == float("inf")).all() and (out[n - 1, :, D - 1] == float("-inf")).all()
    rest = [d for d in range(D) if d not in (3, D - 1)]
    assert torch.equal(out[n - 1][:, rest], want[n - 1][:, rest])
    k[blk[-1], off[-1]] = float("nan")
    v[blk[-1], off[-1], :, :5] = float("nan")
    bt.dev()
    out, lse = run()
    assert torch.equal(out[: n - 1], want[: n - 1]) and torch.equal(lse[: n - 1], wlse[: n - 1])
    assert torch.isnan(out[n - 1].float()).all() and torch.isnan(lse[n - 1]).all()
    bt.cache = clean


@pytest.mark.parametrize("g,n,D", [(4, 1, 128), (4, 4, 64), (8, 6, 128), (4, 40, 128), (4, 64, 64), (2, 3, 256)])
def test_logits_that_grow_by_orders_of_magnitude(g, n, D):
    """Keys whose logits climb from -300 to 300 along the sequence: the running reference is raised again and again (2^64 steps
    included), and the first tiles vanish; then the same falling, and all equal."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(900 + n)
    T = 700
    for shape in ("climb", "fall", "jump"):
        bt = Batch([T], [n], 1, g, D, 16, gen, tree=n > 1)
        bt.q[:] = 0
        bt.q[:, :, 0] = 16.0                       # logits are 16 k_0 scale
        bt.q[:, :, 1:9] = torch.randn((n, g, 8), generator=gen).to(torch.bfloat16)
        blk, off = oa.token_slots(bt.table[0].tolist(), 16, T)
        x = torch.linspace(-300, 300, T) if shape == "climb" else torch.linspace(300, -300, T)
        if shape == "jump":
            x = torch.where(torch.arange(T) == 400, 500.0, -200.0)
        bt.cache[0][0][blk, off, 0, 0] = (x / 16).to(torch.bfloat16)
        bt.dev()
        out, lse = ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, n, tree_mask=bt.d_words, kv_axis=0, scale=1.0)
        check_rows(bt, out, lse, n, 1.0)


def test_caches_that_no_tensor_map_describes():
    """Block strides that are no multiple of the head stride: the gathered kernels serve, weight sums included."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(1000)
    for n in (1, 6, 30):
        bt = Batch([75, 50], [n, max(1, n - 2)], 2, 4, 64, 16, gen, tree=n > 1).dev()
        flat = torch.zeros(2 * bt.nb * (16 * 2 * 64 + 8), dtype=torch.bfloat16, device=DEV)
        odd = flat.as_strided((2, bt.nb, 16, 2, 64), (bt.nb * (16 * 2 * 64 + 8), 16 * 2 * 64 + 8, 128, 64, 1))
        odd.copy_(bt.d_cache[0])
        sums, want = (torch.zeros((bt.nb, 2, 16), device=DEV) for _ in range(2))
        args = (bt.d_table, bt.d_lens, bt.d_start, n)
        out, lse = ops.attend_paged(bt.d_q, odd, *args, tree_mask=bt.d_words, kv_axis=0, weight_sums=sums)
        check_rows(bt, out, lse, n, 1 / 8)
        ops.attend_paged(bt.d_q, bt.d_cache[0], *args, tree_mask=bt.d_words, kv_axis=0, weight_sums=want)
        assert torch.allclose(sums, want, rtol=1e-4, atol=1e-7)


@pytest.mark.parametrize("B,H,n", [(40, 3, 1), (700, 1, 1), (400, 1, 5), (3, 40, 1), (2, 160, 2), (33, 2, 9)])
def test_many_requests_and_many_heads(B, H, n):
    """Batches that are planned in several passes, head counts that do not divide the device."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(1100 + B)
    lens = torch.randint(n, 60, (B,), generator=gen).tolist()
    lens[B // 2] = 500
    counts = [0 if b % 7 == 3 else n for b in range(B)]
    bt = Batch(lens, counts, H, 2, 64, 16, gen, tree=n > 1).dev()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    sums = torch.zeros((bt.nb, H, 16), device=DEV)
    out, lse = ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, n, tree_mask=bt.d_words, kv_axis=0,
                                weight_sums=sums, status=status)
    assert int(status) == 0
    # all requests at once, dense over padded lengths in 64 bits (the oracle's loops would take minutes)
    T = max(lens)
    pos = torch.arange(T)
    blk = bt.table.long()[:, : (T + 15) // 16].repeat_interleave(16, 1)[:, :T]
    k, v = (x[blk, pos % 16].double() for x in split(bt.cache[0], 0))           # [B, T, H, D]
    worst, total = 0.0, 0.0
    for b in range(B):
        c = counts[b]
        if c == 0:
            continue
        see = oa.visible(lens[b], c, None if bt.words is None else bt.words[bt.rows(b)])
        q = bt.q[bt.rows(b)].double().view(c, H, 2, 64)
        s = torch.einsum("nhgd,thd->nhgt", q, k[b, : lens[b]]) / 8
        s = s.masked_fill(~see[:, None, None, :], -math.inf)
        p = torch.softmax(s, -1)
        o = torch.einsum("nhgt,thd->nhgd", p, v[b, : lens[b]]).reshape(c, H * 2, 64)
        a = torch.einsum("nhgt,thd->nhgd", p, v[b, : lens[b]].abs()).reshape(c, H * 2, 64)
        err = (out[bt.rows(b)].cpu().double() - o).abs() - 2.0 ** -8 * o.abs() - 2.0 ** -7.9 * a
        worst = max(worst, float(err.max()))
        assert torch.allclose(lse[bt.rows(b)].cpu().double(), torch.logsumexp(s, -1).reshape(c, H * 2), atol=1e-4)
        total += c * H * 2
    assert worst <= 0 and abs(float(sums.double().sum()) - total) < 1e-3 * total


def test_weight_sums_of_many_rows_go_in_passes():
    """512 rows to a KV head: two passes over the keys."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(1200)
    bt = Batch([200, 90], [64, 20], 1, 8, 128, 16, gen, tree=True).dev()
    sums = torch.full((bt.nb, 1, 16), 0.25, device=DEV)
    ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, 64, tree_mask=bt.d_words, kv_axis=0, weight_sums=sums)
    for b in range(2):
        e = bt.expect(b, 1 / math.sqrt(128))
        blk, off = oa.token_slots(bt.table[b].tolist(), 16, bt.lens[b])
        got = sums.cpu()[blk, 0, off].double()
        got[: bt.lens[b] - bt.counts[b]] -= 0.25
        rel = (2 * 132 * 2.0 ** -23 * e["logit"]).max() + 2.0 ** -20 + 512 * 2.0 ** -24
        assert ((got - e["weight"][0]).abs() <= rel * e["weight"][0] + 2.0 ** -22 * (0.25 + e["weight"][0])).all()


def test_eviction_with_counts_beyond_the_keep_rows():
    from triattention_b200 import _native, ops
    gen = torch.Generator().manual_seed(1300)
    bt = Batch([90, 30], [0, 0], 2, 1, 64, 16, gen).dev()
    view = ops.PagedCacheView.from_layers([bt.d_cache[0]], kv_axis=0)
    sums = torch.rand((1, bt.nb, 2, 16), generator=gen).to(DEV)
    a, b = sums.clone(), sums.clone()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    other = bt.d_cache.clone()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    keep = ops.evict_paged(view, view.layout(2, 1, bt.width), a, bt.d_table, bt.d_lens, i32([80, 20]), 33, 4, status=status)
    assert int(status) == _native.DEV_BAD_LENGTH
    view2 = ops.PagedCacheView.from_layers([other[0]], kv_axis=0)
    want = ops.evict_paged(view2, view2.layout(2, 1, bt.width), b, bt.d_table, bt.d_lens, i32([33, 20]), 33, 4)
    assert torch.equal(keep, want) and torch.equal(a, b) and torch.equal(bt.d_cache, other)


def test_wait_timeout_in_the_attention_kernels_reports_status_and_returns():
    """The test-only library build (waits of about a millisecond, barriers that expect 16 bytes more than ever arrive): the
    attention kernels set TRIATTN_DEV_WAIT_TIMEOUT, drain and return, and the GPU stays usable."""
    import os
    import subprocess
    import sys
    import textwrap
    from pathlib import Path

    from triattention_b200 import _native, build
    repo = Path(__file__).resolve().parent.parent
    lib = build.build_library(short_wait=True)
    code = textwrap.dedent("""
        import sys, torch
        sys.path.insert(0, %r)
        from triattention_b200 import ops
        bits = []
        for n, g, D in ((1, 4, 128), (1, 16, 64), (8, 4, 128), (40, 4, 64)):
            T, H = 900, 2
            cache = torch.randn((2, 60, 16, H, D), device="cuda").bfloat16()
            q = torch.randn((2 * n, H * g, D), device="cuda").bfloat16()
            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
            table = torch.arange(57, dtype=torch.int32, device="cuda").repeat(2, 1)
            status, sums = i32([0]), torch.zeros((60, H, 16), device="cuda")
            ops.attend_paged(q, cache, table, i32([T, T - 100]), i32([0, n, 2 * n]), n, weight_sums=sums, status=status)
            torch.cuda.synchronize()
            bits.append(int(status))
        print("STATUS", *bits, torch.arange(10, device="cuda").sum().item())
    """) % str(repo)
    out = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, TRIATTN_B200_LIB=str(lib)), capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    line = [x for x in out.stdout.splitlines() if x.startswith("STATUS")][-1].split()
    assert all(int(b) & _native.DEV_WAIT_TIMEOUT for b in line[1:5]) and int(line[5]) == 45, line


def test_strides_of_axes_with_one_entry_do_not_matter():
    """One KV head or one block: whatever the stride of that axis says, the same result."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(1400)
    bt = Batch([130], [1], 1, 4, 64, 16, gen).dev()
    want, wl = ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, 1, kv_axis=0)
    check_rows(bt, want, wl, 1, 1 / 8)
    st = list(bt.d_cache[0].stride())
    for s in (8, 72, 1 << 20):
        odd = bt.d_cache[0].as_strided(bt.d_cache[0].shape, st[:3] + [s] + st[4:])
        out, lse = ops.attend_paged(bt.d_q, odd, bt.d_table, bt.d_lens, bt.d_start, 1, kv_axis=0)
        assert torch.equal(out, want) and torch.equal(lse, wl)
    one = torch.randn((2, 1, 16, 2, 64), generator=gen).to(torch.bfloat16).to(DEV)
    q = torch.randn((1, 8, 64), generator=gen).to(torch.bfloat16).to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    outs = []
    for s in (16 * 128, 8, 24, 1 << 21):
        c = one.as_strided(one.shape, (one.stride(0), s, *one.stride()[2:]))
        outs.append(ops.attend_paged(q, c, i32([[0]]), i32([11]), i32([0, 1]), 1, kv_axis=0)[0])
    assert all(torch.equal(o, outs[0]) for o in outs[1:])


def test_choice_among_more_blocks_than_shared_memory_holds():
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(1500)
    T, n = 40000, 2
    bt = Batch([T, 33000], [n, 1], 1, 2, 64, 1, gen).dev()            # a block is a token
    bounds = torch.zeros((bt.nb, 1, 2, 64), dtype=torch.bfloat16, device=DEV)
    view = ops.PagedCacheView.from_layers([bt.d_cache[0]], kv_axis=0)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    ops.update_block_bounds(view, view.layout(2, 2, bt.width), bounds[None], bt.d_table, zero, bt.d_lens)
    got = ops.select_blocks(bt.d_q, bounds, bt.d_lens, bt.d_start, bt.d_table, n, 1, 700, sink_blocks=3, recent_blocks=20).cpu()
    for b in range(2):
        k, _ = bt.tokens(b)
        lo, hi = oa.block_bounds(k, 1)
        want = oa.select_blocks(oa.block_scores(bt.q[bt.rows(b)], lo, hi), bt.lens[b], bt.counts[b], 1, 700, 3, 20)
        assert torch.equal(got[b], want)


def test_eviction_refused_before_anything_moves():
    """A pool too large for the compaction is refused by the entry point before the selection has moved the sums."""
    import ctypes

    from triattention_b200 import _native
    lib = _native.load()
    lay = _native.PagedLayout(1, 1, 8, 1, 128, 16, 3_000_000, 8, 16 * 8 * 128, 8 * 128, 128, 0, 0)
    sums = torch.ones(64, device=DEV)
    p = sums.data_ptr()
    assert lib.triattn_evict_paged(ctypes.byref(lay), p, p, p, p, p, p, None, 1, p, 4, None, None) == 2
    torch.cuda.synchronize()
    assert (sums == 1).all()


def test_output_on_top_of_the_queries_is_refused():
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(1600)
    bt = Batch([20], [1], 1, 2, 64, 16, gen).dev()
    with pytest.raises(ValueError):
        ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, 1, kv_axis=0, out=bt.d_q)


@pytest.mark.parametrize("g,n,D,bs", [(3, 1, 128, 16), (4, 1, 64, 16), (5, 7, 128, 16), (4, 40, 64, 16), (3, 2, 128, 5), (5, 3, 256, 16)])
def test_keys_of_minus_infinite_logit_weigh_nothing(g, n, D, bs):
    """An infinite key channel against queries that are all negative there: the logit is -inf, the token weighs 0 and no
    other token is disturbed, in the output or in the sums."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(1700 + n)
    bt = Batch([150], [n], 2, g, D, bs, gen, tree=n > 1)
    bt.q[:, :, 0] = -bt.q[:, :, 0].abs() - 0.5
    blk, off = oa.token_slots(bt.table[0].tolist(), bs, 150)
    k, _ = split(bt.cache[0], 0)
    k[blk[37], off[37], :, 0] = float("inf")
    bt.dev()
    sums = torch.zeros((bt.nb, 2, bs), device=DEV)
    out, lse = ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, n, tree_mask=bt.d_words, kv_axis=0, weight_sums=sums)
    finite = bt.cache.clone()
    kk, vv = split(finite[0], 0)
    tk, tv = kk[blk, off].clone(), vv[blk, off]
    tk[37, :, 0] = 0
    see = oa.visible(150, n, bt.words)
    see[:, 37] = False
    e = oa.attend_request(bt.q, tk, tv, see, 1 / math.sqrt(D))
    assert torch.allclose(lse.cpu().double(), e["lse"], atol=1e-4)
    assert ((out.cpu().double() - e["out"]).abs() <= 2.0 ** -8 * e["out"].abs() + 2.0 ** -7.9 * e["spread"]).all()
    got = sums.cpu()[blk, :, off].T.double()
    assert (got[:, 37] == 0).all() and torch.allclose(got, e["weight"], rtol=1e-3, atol=1e-7)


def test_what_is_always_kept_ranks_above_infinities():
    """More infinite sums, or bounds, in front than there are places: the window's tokens and the recent blocks stay."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(1800)
    bt = Batch([640], [1], 1, 2, 64, 16, gen).dev()
    bounds = torch.full((bt.nb, 1, 2, 64), float("inf"), dtype=torch.bfloat16, device=DEV)
    got = ops.select_blocks(bt.d_q.abs(), bounds, bt.d_lens, bt.d_start, bt.d_table, 1, 16, 6, sink_blocks=1, recent_blocks=2)
    assert got[0, 0].tolist() == [0, 1, 2, 3, 38, 39]
    bounds.fill_(2.0 ** 127)                         # finite bounds whose sum is beyond 32 bits
    got = ops.select_blocks(bt.d_q.abs(), bounds, bt.d_lens, bt.d_start, bt.d_table, 1, 16, 6, sink_blocks=1, recent_blocks=2)
    assert got[0, 0].tolist() == [0, 1, 2, 3, 38, 39]
    view = ops.PagedCacheView.from_layers(list(bt.d_cache.unbind(0)), kv_axis=0)
    sums = torch.full((1, bt.nb, 1, 16), float("inf"), device=DEV)
    one = lambda v: torch.tensor([v], dtype=torch.int32, device=DEV)  # noqa: E731
    keep = ops.evict_paged(view, view.layout(1, 1, bt.width), sums, bt.d_table, bt.d_lens, one(20), 20, 8, one(3))
    assert keep[0, 0, 0].tolist() == list(range(12)) + list(range(632, 640))


@pytest.mark.parametrize("D,bs,g,n", VARIANTS)
def test_infinite_values_everyone_sees(D, bs, g, n):
    """An infinite value of an older token: its channel is infinite for every row, the others are as without it."""
    from triattention_b200 import ops
    gen = torch.Generator().manual_seed(1900 + D + n)
    bt = Batch([170], [n], 2, g, D, bs, gen, tree=n > 1).dev()
    run = lambda: ops.attend_paged(bt.d_q, bt.d_cache[0], bt.d_table, bt.d_lens, bt.d_start, n, tree_mask=bt.d_words, kv_axis=0)  # noqa: E731
    want, wlse = run()
    k, v = split(bt.cache[0], 0)
    blk, off = oa.token_slots(bt.table[0].tolist(), bs, 170)
    v[blk[33], off[33], :, 3] = float("inf")
    v[blk[90], off[90], :, D - 7] = float("-inf")
    bt.dev()
    out, lse = run()
    assert (out[:, :, 3] == float("inf")).all() and (out[:, :, D - 7] == float("-inf")).all()
    others = [d for d in range(D) if d not in (3, D - 7)]
    assert torch.equal(out[:, :, others], want[:, :, others]) and torch.equal(lse, wlse)
