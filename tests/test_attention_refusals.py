"""What the attention operators refuse, checked without a GPU: the C entry points answer before they launch anything, the
Python wrappers before they call them."""
from __future__ import annotations

import ctypes

import pytest
import torch

from triattention_b200 import _native, ops

OK, BAD, SHAPE, ALIGN, SMALL = 0, 1, 2, 3, 4
P = 1 << 20  # an aligned address nobody reads


def layout(**kw):
    base = dict(num_layers=1, num_reqs=2, num_kv_heads=2, group_size=4, head_dim=128, block_size=16, num_blocks=50,
                max_blocks_per_req=8, block_stride=16 * 2 * 128, token_stride=2 * 128, head_stride=128)
    return _native.PagedLayout(**{**base, **kw})


def attend(lay=None, **kw):
    lib = _native.load()
    a = dict(k=P, v=P, table=P, lens=P, start=P, q=P, qts=1024, qhs=128, N=2, mq=1, scale=0.1, tree=None, lst=None, S=0,
             sums=None, reset=0, out=P, ots=1024, ohs=128, lse=P, ws=P, wsb=1 << 40)
    a.update(kw)
    return lib.triattn_attend_paged(ctypes.byref(lay or layout()), *a.values(), None, None)


def test_attend_entry_point_refuses():
    for name in ("k", "v", "table", "lens", "start", "q", "out", "lse", "ws"):
        assert attend(**{name: None}) == BAD, name
    assert attend(mq=0) == BAD and attend(mq=65) == SHAPE
    assert attend(scale=0.0) == BAD and attend(scale=-1.0) == BAD
    assert attend(scale=float("nan")) == BAD and attend(scale=float("inf")) == BAD
    assert attend(N=-1) == BAD
    assert attend(lst=P, S=0) == BAD
    for name in ("k", "v", "q", "out", "ws"):
        assert attend(**{name: P + 2}) == ALIGN, name
    for name in ("qts", "qhs", "ots", "ohs"):
        assert attend(**{name: 132}) == ALIGN, name
    for d in (72, 96, 512):
        assert attend(layout(head_dim=d)) == SHAPE
    assert attend(layout(group_size=65)) == SHAPE
    assert attend(layout(max_blocks_per_req=1 << 27)) == SHAPE     # token positions beyond 32 bits
    assert attend(layout(token_stride=4)) == ALIGN
    assert attend(wsb=16) == SMALL
    assert attend(N=0, q=None, out=None) == OK                      # nothing to do, nothing launched


def test_workspace_sizes():
    lib = _native.load()
    ws = lambda lay, mq=1, s=0: lib.triattn_attend_workspace_bytes(ctypes.byref(lay), mq, s)  # noqa: E731
    assert ws(layout()) > 0
    assert ws(layout(head_dim=80)) == 0 and ws(layout(), 65) == 0 and ws(layout(num_reqs=0)) == 0
    # bounded by the device, not by the lengths
    assert ws(layout(max_blocks_per_req=1 << 20), 64) <= 2 * 148 * 2 * 256 * (128 + 2) * 4 + 1024
    assert attend(wsb=ws(layout()) - 1) == SMALL
    sel = lib.triattn_select_blocks_workspace_bytes(ctypes.byref(layout()))
    assert sel == 2 * 2 * 8 * 4 + (256 - 128)


def test_eviction_bounds_and_choice_refuse():
    lib = _native.load()
    ref = ctypes.byref(layout())
    ev = lambda k=P, v=P, s=P, t=P, n=P, c=P, win=4, keep=P, pitch=8, lay=None: lib.triattn_evict_paged(  # noqa: E731
        ctypes.byref(lay) if lay else ref, k, v, s, t, n, c, None, win, keep, pitch, None, None)
    for name in ("k", "v", "s", "t", "n", "c", "keep"):
        assert ev(**{name: None}) == BAD, name
    assert ev(win=-1) == BAD and ev(pitch=0) == BAD and ev(lay=layout(max_blocks_per_req=1 << 27)) == SHAPE
    bd = lambda k=P, t=P, f=P, n=P, b=P, lay=None: lib.triattn_update_block_bounds(  # noqa: E731
        ctypes.byref(lay) if lay else ref, k, t, f, n, b, None, None)
    for name in ("k", "t", "f", "n", "b"):
        assert bd(**{name: None}) == BAD, name
    assert bd(b=P + 8) == ALIGN and bd(lay=layout(head_dim=96)) == SHAPE
    se = lambda q=P, qts=1024, N=2, mq=1, st=P, b=P, t=P, n=P, sel=4, sink=1, rec=2, lst=P, ws=P, wsb=1 << 30: (  # noqa: E731
        lib.triattn_select_blocks(ref, q, qts, 128, N, mq, st, b, t, n, sel, sink, rec, lst, ws, wsb, None, None))
    for name in ("q", "st", "b", "t", "n", "lst", "ws"):
        assert se(**{name: None}) == BAD, name
    assert se(sel=0) == BAD and se(sink=-1) == BAD and se(rec=-1) == BAD
    assert se(sel=2, sink=1, rec=2) == BAD            # the recent blocks do not fit
    assert se(mq=40, sel=4, sink=1) == BAD            # nor do the blocks of the query's own tokens
    assert se(b=P + 2) == ALIGN and se(q=P + 2) == ALIGN and se(qts=100) == ALIGN and se(wsb=8) == SMALL


@pytest.fixture
def on_cpu(monkeypatch):
    """The wrappers' checks on CPU tensors (device index -1); nothing below gets as far as the library."""
    monkeypatch.setattr(ops, "_require_cuda", lambda *a: None)
    calls = []
    monkeypatch.setattr(ops._native, "check", lambda rc, what: calls.append(what))
    yield
    assert not calls


def inputs():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return dict(q=torch.zeros((3, 8, 64), dtype=torch.bfloat16), kv_cache=torch.zeros((2, 9, 16, 2, 64), dtype=torch.bfloat16),
                block_table=i32(2, 4), seq_lens=i32(2), query_start_loc=i32(3), max_query_len=2)


@pytest.mark.parametrize("name,value", [
    ("q", torch.zeros((3, 8, 64))), ("q", torch.zeros((3, 8, 32), dtype=torch.bfloat16)),
    ("q", torch.zeros((3, 7, 64), dtype=torch.bfloat16)), ("q", torch.zeros((3, 64, 8), dtype=torch.bfloat16).transpose(1, 2)),
    ("q", torch.zeros((24, 64), dtype=torch.bfloat16)),
    ("kv_cache", torch.zeros((2, 9, 16, 2, 64), dtype=torch.float16)), ("kv_cache", torch.zeros((3, 9, 16, 2, 64), dtype=torch.bfloat16)),
    ("kv_cache", torch.zeros((2, 2, 16, 2, 64), dtype=torch.bfloat16)), ("kv_cache", torch.zeros((9, 16, 2, 64), dtype=torch.bfloat16)),
    ("block_table", torch.zeros((2, 4), dtype=torch.int64)), ("block_table", torch.zeros((3, 4), dtype=torch.int32)),
    ("block_table", torch.zeros((2, 0), dtype=torch.int32)), ("block_table", torch.zeros((2, 8), dtype=torch.int32)[:, ::2]),
    ("block_table", torch.zeros(8, dtype=torch.int32)),
    ("seq_lens", torch.zeros(2)), ("seq_lens", torch.zeros(0, dtype=torch.int32)),
    ("query_start_loc", torch.zeros(2, dtype=torch.int32)),
    ("tree_mask", torch.zeros(2, dtype=torch.int64)), ("tree_mask", torch.zeros(3, dtype=torch.int32)),
    ("block_list", torch.zeros((2, 2, 0), dtype=torch.int32)), ("block_list", torch.zeros((2, 4), dtype=torch.int32)),
    ("block_list", torch.zeros((2, 1, 4), dtype=torch.int32)),
    ("weight_sums", torch.zeros((9, 2, 16), dtype=torch.float64)), ("weight_sums", torch.zeros((9, 16, 2))),
    ("out", torch.zeros((3, 8, 64))), ("out", torch.zeros((2, 8, 64), dtype=torch.bfloat16)), ("lse", torch.zeros((3, 4))),
    ("status", torch.zeros(1)), ("workspace", torch.zeros(64, dtype=torch.uint8)[::2]),
])
def test_attend_wrapper_refuses(on_cpu, monkeypatch, name, value):
    monkeypatch.setattr(ops, "_on_device", lambda index: ops._NO_GUARD)
    with pytest.raises(ValueError):
        ops.attend_paged(**{**inputs(), name: value})


def test_tensors_on_the_host_are_refused():
    with pytest.raises(_native.NativeLibraryError):
        ops.attend_paged(**inputs())
    with pytest.raises(_native.NativeLibraryError):
        ops.select_blocks(inputs()["q"], torch.zeros((9, 2, 2, 64), dtype=torch.bfloat16), inputs()["seq_lens"],
                          inputs()["query_start_loc"], inputs()["block_table"], 2, 16, 8)


def test_other_wrappers_refuse(on_cpu, monkeypatch):
    monkeypatch.setattr(ops, "_on_device", lambda index: ops._NO_GUARD)
    x = inputs()
    bounds = torch.zeros((9, 2, 2, 64), dtype=torch.bfloat16)
    sel = lambda **kw: ops.select_blocks(**{**dict(q=x["q"], bounds=bounds, seq_lens=x["seq_lens"], block_table=x["block_table"],  # noqa: E731
                                                   query_start_loc=x["query_start_loc"], max_query_len=2, block_size=16, num_selected=8), **kw})
    for kw in (dict(bounds=bounds.float()), dict(bounds=bounds[:, :, 0]), dict(num_selected=2), dict(block_size=0),
               dict(seq_lens=x["seq_lens"].long()), dict(block_list=torch.zeros((2, 2, 7), dtype=torch.int32))):
        with pytest.raises(ValueError):
            sel(**kw)
    cache = [x["kv_cache"], x["kv_cache"].clone()]
    view = ops.PagedCacheView._build(cache, 0)
    lay = view.layout(2, 1, 4)
    sums, one = torch.zeros((2, 9, 2, 16)), torch.zeros(2, dtype=torch.int32)
    ev = lambda **kw: ops.evict_paged(**{**dict(view=view, layout=lay, weight_sums=sums, block_table=x["block_table"],  # noqa: E731
                                                seq_lens=one, keep_counts=one, keep_pitch=4, window=2), **kw})
    for kw in (dict(weight_sums=sums[:1]), dict(weight_sums=sums.double()), dict(block_table=x["block_table"][:, :3]),
               dict(keep_counts=one[:1]), dict(prefill_lens=one.long()), dict(keep_out=torch.zeros((2, 2, 2, 5), dtype=torch.int32))):
        with pytest.raises(ValueError):
            ev(**kw)
    bd = lambda **kw: ops.update_block_bounds(**{**dict(view=view, layout=lay, bounds=torch.zeros((2, 9, 2, 2, 64), dtype=torch.bfloat16),  # noqa: E731
                                                        block_table=x["block_table"], first_tokens=one, seq_lens=one), **kw})
    for kw in (dict(bounds=bounds), dict(first_tokens=one.long()), dict(seq_lens=one[:1])):
        with pytest.raises(ValueError):
            bd(**kw)


def test_oracle_against_a_dense_softmax():
    """The 64-bit oracle itself: masks, log-sums and weights of a small request against torch's dense softmax."""
    from oracle import attention as oa
    gen = torch.Generator().manual_seed(1)
    n, T, H, g, D = 4, 11, 2, 3, 8
    q, k, v = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((n, H * g, D), (T, H, D), (T, H, D)))
    words = [0b0001, 0b0011, 0b0101, 0b1011]
    see = oa.visible(T, n, words)
    assert see[:, : T - n].all() and see[:, T - n:].long().tolist() == [[1, 0, 0, 0], [1, 1, 0, 0], [1, 0, 1, 0], [1, 1, 0, 1]]
    e = oa.attend_request(q, k, v, see, 0.3)
    s = torch.einsum("nhd,thd->nht", q, k.repeat_interleave(g, 1)) * 0.3
    p = torch.softmax(s.masked_fill(~see[:, None], float("-inf")), -1)
    assert torch.allclose(e["out"], torch.einsum("nht,thd->nhd", p, v.repeat_interleave(g, 1)))
    assert torch.allclose(e["weight"], p.view(n, H, g, T).sum((0, 2)))
    assert torch.allclose(e["lse"], torch.logsumexp(s.masked_fill(~see[:, None], float("-inf")), -1))
    empty = oa.attend_request(q[:1], k[:1], v[:1], torch.zeros((1, 1), dtype=torch.bool), 0.3)
    assert (empty["out"] == 0).all() and (empty["lse"] == -float("inf")).all()
    lo, hi = oa.block_bounds(k, 4)
    sc = oa.block_scores(q, lo, hi)
    best = torch.einsum("nhd,thd->nht", q, k.repeat_interleave(g, 1)).view(n, H, g, T)
    for b in range(3):  # an upper bound of every logit, summed over the rows
        assert (sc[:, b] + 1e-4 >= best[..., 4 * b : 4 * b + 4].amax(-1).sum((0, 2))).all()


@pytest.mark.parametrize("name", ["num_layers", "num_blocks", "block_size", "num_kv_heads", "head_dim", "block_stride", "token_stride", "head_stride"])
def test_a_layout_that_is_not_the_views_is_refused(on_cpu, monkeypatch, name):
    monkeypatch.setattr(ops, "_on_device", lambda index: ops._NO_GUARD)
    x = inputs()
    view = ops.PagedCacheView._build([x["kv_cache"], x["kv_cache"].clone()], 0)
    lay, one = view.layout(2, 1, 4), torch.zeros(2, dtype=torch.int32)
    setattr(lay, name, getattr(lay, name) * 2)
    with pytest.raises(ValueError, match=name):
        ops.evict_paged(view, lay, torch.zeros((2, 9, 2, 16)), x["block_table"], one, one, 4, 2)
    with pytest.raises(ValueError, match=name):
        ops.update_block_bounds(view, lay, torch.zeros((2, 9, 2, 2, 64), dtype=torch.bfloat16), x["block_table"], one, one)
