"""The attention operators together, as a serving step uses them: prompt end with sums, drafted trees, accepted tokens moved
up, eviction, bounds, block-sparse decode.  A plain 64-bit model of every request's tokens runs beside the cache; tolerances
are those of test_gpu_attention.py (check_rows)."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import attention as oa
from test_gpu_attention import DEV, Batch, check_rows, split

pytestmark = pytest.mark.gpu

L, H, G, D, BS = 2, 2, 4, 128, 16


class Serving:
    """Host-side model: per request and layer the K / V / sums of every KV head, and the block ids."""

    def __init__(self, lens, gen, spare):
        self.gen = gen
        self.lens = list(lens)
        width = max((t + BS - 1) // BS for t in lens) + spare
        self.nb, self.width = len(lens) * width + 2, width
        ids = torch.randperm(self.nb, generator=gen).tolist()
        self.ids = [ids[i * width : (i + 1) * width] for i in range(len(lens))]
        self.cache = torch.randn((L, 2, self.nb, BS, H, D), generator=gen).to(torch.bfloat16).to(DEV)
        self.sums = torch.full((L, self.nb, H, BS), float("nan"), device=DEV)
        self.bounds = torch.zeros((L, self.nb, H, 2, D), dtype=torch.bfloat16, device=DEV)

    def i32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    def table(self):
        return self.i32([ids + [0] * (self.width - len(ids)) for ids in self.ids])

    def batch(self, layer, counts, q, words):
        """A Batch (test_gpu_attention) over this layer's present cache, for the oracle."""
        bt = Batch.__new__(Batch)
        bt.lens, bt.counts, bt.H, bt.g, bt.D, bt.bs, bt.axis = list(self.lens), counts, H, G, D, BS, 0
        bt.nb, bt.width, bt.table = self.nb, self.width, self.table().cpu()
        bt.cache = self.cache[layer : layer + 1].cpu()
        bt.start = [0]
        for c in counts:
            bt.start.append(bt.start[-1] + c)
        bt.q, bt.words = q, words
        return bt

    def append(self, counts):
        """The slots of the next tokens get new keys and values in every layer."""
        for b, c in enumerate(counts):
            for t in range(self.lens[b], self.lens[b] + c):
                self.cache[:, :, self.ids[b][t // BS], t % BS] = torch.randn((L, 2, H, D), generator=self.gen).to(torch.bfloat16).to(DEV)
            self.lens[b] += c

    def read_sums(self, layer, b):
        blk, off = oa.token_slots(self.ids[b], BS, self.lens[b])
        return self.sums[layer].cpu()[blk, :, off].T.double()   # [H, T]


def test_serving_steps_with_eviction_and_sparse_decode():
    from triattention_b200 import engine, ops
    gen = torch.Generator().manual_seed(42)
    s = Serving([200, 333], gen, spare=5)
    scale = 1 / math.sqrt(D)
    model = [[None, None] for _ in range(L)]   # sums per layer and request

    def attend(counts, words, reset=False, blocks=None, observe=True):
        n = sum(counts)
        start = s.i32([0] + torch.tensor(counts).cumsum(0).tolist())
        dw = None if words is None else torch.tensor(words, dtype=torch.int64, device=DEV)
        for l in range(L):
            q = (torch.randn((n, H * G, D), generator=gen) * 1.5).to(torch.bfloat16)
            lst = None
            if blocks is not None:
                lst = ops.select_blocks(q.to(DEV), s.bounds[l], s.i32(s.lens), start, s.table(), max(counts), BS, blocks)
            out, lse = ops.attend_paged(q.to(DEV), s.cache[l], s.table(), s.i32(s.lens), start, max(counts), tree_mask=dw,
                                        block_list=lst, weight_sums=s.sums[l] if observe else None, reset_weight_sums=reset, kv_axis=0)
            bt = s.batch(l, counts, q, words)
            if lst is not None:
                for b in range(len(counts)):  # the choice itself
                    k, _ = bt.tokens(b)
                    sc = oa.block_scores(q[bt.rows(b)], *oa.block_bounds(k, BS))
                    assert torch.equal(lst[b].cpu(), oa.select_blocks(sc, s.lens[b], counts[b], BS, blocks, 1, 2))
            for b, e in enumerate(check_rows(bt, out, lse, max(counts), scale, None if lst is None else lst.cpu())):
                if not observe:
                    continue
                old = torch.zeros_like(e["weight"])
                if not reset:
                    old[:, : model[l][b].shape[1]] = model[l][b]
                    old[:, s.lens[b] - counts[b] :] = 0
                model[l][b] = old + e["weight"]
                assert torch.allclose(s.read_sums(l, b), model[l][b], rtol=1e-3, atol=1e-6)

    # the end of the prompts: the last 16 tokens look back and start the sums
    attend([16, 16], None, reset=True)
    # two steps of drafted trees; afterwards the accepted path's tokens move up behind the context
    for accepted in ([0, 2], [0, 1, 3]):
        counts = [5, 4]
        s.append(counts)
        words = [0b00001, 0b00011, 0b00101, 0b01011, 0b10001, 0b0001, 0b0011, 0b0101, 0b1011]
        attend(counts, words)
        view = ops.PagedCacheView.from_layers(list(s.cache.unbind(0)), kv_axis=0)
        lay = view.layout(2, G, s.width)
        keep, after = [], []
        for b, c in enumerate(counts):
            ctx = s.lens[b] - c
            keep.append(list(range(ctx)) + [ctx + i for i in accepted])
            after.append(len(keep[b]))
        pitch = max(after)
        d_keep = s.i32([k + [-1] * (pitch - len(k)) for k in keep])
        ops.compact_paged(view, lay, s.table(), s.i32(s.lens), d_keep, (0, pitch, 0), s.i32(after))
        for b in range(2):  # the host keeps the sums of the accepted tokens with them
            blk, off = oa.token_slots(s.ids[b], BS, s.lens[b])
            src = torch.tensor(keep[b])
            moved = s.sums[:, blk[src], :, off[src]].clone()
            s.sums[:, blk[: after[b]], :, off[: after[b]]] = moved
            for l in range(L):
                model[l][b] = model[l][b][:, src]
            s.lens[b] = after[b]
    # eviction: every layer and head keeps its own tokens
    before = s.cache.clone()
    old_lens, old_ids = list(s.lens), [list(i) for i in s.ids]
    evictor = engine.AttentionEvictor(window=16)
    view = ops.PagedCacheView.from_layers(list(s.cache.unbind(0)), kv_axis=0)
    sums_then = [[s.read_sums(l, b) for b in range(2)] for l in range(L)]
    res = evictor.evict(view, s.sums, s.ids, s.lens, [100, 150], prefill_lens=[4, 0])
    assert res.device_status == 0 and res.keep_counts == [100, 150]
    assert [len(k) for k in res.kept_block_ids] == [7, 10]
    assert [k + r for k, r in zip(res.kept_block_ids, res.removed_block_ids)] == old_ids
    for l in range(L):
        for b in range(2):
            blk, off = oa.token_slots(old_ids[b], BS, old_lens[b])
            new = torch.empty((H, res.keep_counts[b]), dtype=torch.float64)
            for h in range(H):
                k = oa.evict_keep(sums_then[l][b][h].float(), res.keep_counts[b], 16, [4, 0][b]).long()
                assert torch.equal(res.keep[l, b, h, : len(k)].cpu().long(), k)
                for kv in range(2):
                    assert torch.equal(s.cache[l, kv][blk[: len(k)], off[: len(k)], h].view(torch.int16),
                                       before[l, kv][blk[k], off[k], h].view(torch.int16))
                new[h] = model[l][b][h, k]
            model[l][b] = new
    s.lens = list(res.keep_counts)
    # (the freed blocks stay in the row as spare ones, as after a reallocation)
    # what was evicted is gone: a decode step over the smaller caches, sums continued
    s.append([1, 1])
    attend([1, 1], None)
    # bounds of the compacted caches, then block-sparse steps that keep them up to date
    ops.update_block_bounds(view, view.layout(2, G, s.width), s.bounds, s.table(), s.i32([0, 0]), s.i32(s.lens))
    for _ in range(3):
        s.append([1, 1])
        ops.update_block_bounds(view, view.layout(2, G, s.width), s.bounds, s.table(), s.i32([n - 1 for n in s.lens]), s.i32(s.lens))
        attend([1, 1], None, blocks=4, observe=False)


def test_evictor_arguments_and_repeated_use():
    from triattention_b200 import engine, ops
    gen = torch.Generator().manual_seed(43)
    s = Serving([40, 70, 20], gen, spare=0)
    s.sums = torch.rand((L, s.nb, H, BS), generator=gen).to(DEV)
    view = ops.PagedCacheView.from_layers(list(s.cache.unbind(0)), kv_axis=0)
    ev = engine.AttentionEvictor(window=4)
    with pytest.raises(ValueError):
        ev.evict(view, s.sums, s.ids, [40, 70], [10, 10, 10])
    with pytest.raises(ValueError):
        ev.evict(view, s.sums, [], [], [])
    with pytest.raises(IndexError):
        ev.evict(view, s.sums, s.ids, [40, 700, 20], [10, 10, 10])
    res = ev.evict(view, s.sums, s.ids, [40, 70, 20], [10, 33, 50])
    assert res.keep_counts == [10, 33, 20] and res.keep.shape == (L, 3, H, 33)
    assert (res.keep[:, 2, :, :20].cpu() == torch.arange(20)).all() and (res.keep[:, 0, :, 10:] == -1).all()
    first = s.sums.clone()
    again = ev.evict(view, s.sums, s.ids, [10, 33, 20], [10, 33, 20])     # nothing left to evict
    assert torch.equal(s.sums, first) and again.keep_counts == [10, 33, 20]
