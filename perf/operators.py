"""Attention over the paged cache, eviction by attention weight, and block-sparse attention: cases and plain forms.

The operators (all read the paged bf16 cache that the compression step works on):

attend   attention of the query tokens of a decode step over the cache, from one token per request to a tree of up
         to 64 drafted tokens whose keys are already in the cache's last slots;
observe  the same, and the probability mass every cached token received is added to its running sum;
evict    per layer, request and KV head the tokens with the largest sums are kept (a recent window always), K, V and
         the sums are compacted in place;
bounds   per cache block and channel the smallest and largest key value, rebuilt for the blocks that changed;
sparse   the blocks with the largest upper bound of the attention logits are selected per request and KV head,
         and the attention reads those blocks only.

``own`` false: elementary torch operations in 32 bits (64 for the block scores, whose order decides).  ``own`` true:
the calls a user makes of ``triattention_b200.ops``.
"""
import math

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one interactive user, short conversation: nothing but latency
        {"name": "attend_one_short", "op": "attend", "B": 1, "T": 517, "T_min": 517, "n": 1, "Hkv": 8, "g": 4, "D": 128,
         "bs": 16, "hnd": False, "axis": 0, "tree": False},
        # a decode step of 64 requests that the compression holds at its budget of 2048 + 128 tokens
        {"name": "attend_budget_batch", "op": "attend", "B": 64, "T": 2176, "T_min": 2048, "n": 1, "Hkv": 8, "g": 4,
         "D": 128, "bs": 16, "hnd": False, "axis": 0, "tree": False},
        # speculative decoding, an uneven tree of 26 drafts, eight query heads to a KV head
        {"name": "attend_tree_mid", "op": "attend", "B": 4, "T": 8191, "T_min": 5003, "n": 26, "Hkv": 8, "g": 8,
         "D": 128, "bs": 16, "hnd": False, "axis": 1, "tree": True},
        # the widest tree over prompts of 32768 tokens
        {"name": "attend_tree_long", "op": "attend", "B": 8, "T": 32768, "T_min": 32768, "n": 64, "Hkv": 8, "g": 4,
         "D": 128, "bs": 16, "hnd": False, "axis": 0, "tree": True},
        # a decode step that keeps the sums up to date, head dimension 64, ragged lengths
        {"name": "observe_decode", "op": "observe", "B": 16, "T": 8190, "T_min": 1021, "n": 1, "Hkv": 8, "g": 8, "D": 64,
         "bs": 16, "hnd": False, "axis": 0, "tree": False, "reset": False},
        # the last 32 tokens of two fresh prompts look back over them and start the sums
        {"name": "observe_prompt_end", "op": "observe", "B": 2, "T": 16384, "T_min": 12289, "n": 32, "Hkv": 8, "g": 4,
         "D": 128, "bs": 16, "hnd": False, "axis": 0, "tree": False, "reset": True},
        # the steady trigger: 2176 -> 2048 tokens, four layers' worth
        {"name": "evict_steady", "op": "evict", "L": 4, "B": 8, "T": 2176, "T_min": 2176, "Hkv": 8, "D": 128, "bs": 16,
         "hnd": False, "axis": 0, "keep": 2048, "window": 128},
        # the first trigger of two long prompts: 32768 -> 2048 tokens
        {"name": "evict_long", "op": "evict", "L": 8, "B": 2, "T": 32768, "T_min": 30011, "Hkv": 8, "D": 128, "bs": 16,
         "hnd": False, "axis": 0, "keep": 2048, "window": 128},
        # after a prefill: the bounds of whole prompts
        {"name": "bounds_prompt", "op": "bounds", "L": 2, "B": 4, "T": 32768, "T_min": 20001, "Hkv": 8, "D": 128,
         "bs": 16, "hnd": False, "axis": 0, "step": 0},
        # after a decode step: the last block of every request and layer
        {"name": "bounds_step", "op": "bounds", "L": 36, "B": 32, "T": 2176, "T_min": 2048, "Hkv": 8, "D": 128,
         "bs": 16, "hnd": False, "axis": 0, "step": 1},
        # one long request, 128 of 2048 blocks read
        {"name": "sparse_one_long", "op": "sparse", "B": 1, "T": 32768, "T_min": 32768, "n": 1, "Hkv": 8, "g": 4,
         "D": 128, "bs": 16, "hnd": False, "axis": 0, "tree": False, "sel": 128, "sink": 1, "recent": 4},
        # a batch of long requests with short drafted trees
        {"name": "sparse_batch_tree", "op": "sparse", "B": 24, "T": 32760, "T_min": 9001, "n": 8, "Hkv": 8, "g": 4,
         "D": 128, "bs": 16, "hnd": False, "axis": 0, "tree": True, "sel": 128, "sink": 1, "recent": 4},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attend", "attend", "observe", "evict", "bounds", "sparse"])
    Hkv, D, bs = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128]), rng.choice([8, 16, 16, 32, 64])
    case = {"op": op, "Hkv": Hkv, "D": D, "bs": bs, "hnd": rng.random() < 0.3, "axis": rng.choice([0, 1])}
    # total cached tokens x KV heads stay below the largest listed cases
    cap = 1_000_000 if op in ("attend", "sparse") else 500_000
    T = log_int(200, 32768)
    B = max(1, min(log_int(1, 64), cap // (T * Hkv)))
    case.update({"B": B, "T": T, "T_min": max(80, int(T * rng.uniform(0.3, 1.0)))})
    case["T_min"] = min(case["T_min"], T)
    if op in ("attend", "observe", "sparse"):
        n = rng.choice([1, 1, log_int(2, 64)])
        g = rng.choice([1, 2, 3, 4, 5, 8, 16])
        while n * g > 256:
            n = max(1, n // 2)
        case.update({"n": n, "g": g, "tree": n > 1 and rng.random() < 0.7})
        if op == "observe":
            case["reset"] = rng.random() < 0.3
        if op == "sparse":
            forced = 1 + 2 + (n + bs - 1) // bs + 1
            case.update({"sel": max(forced, log_int(8, 256)), "sink": 1, "recent": 2})
    else:
        case["L"] = max(1, min(rng.choice([1, 2, 4, 8]), cap // (B * T * Hkv)))
        if op == "evict":
            case["window"] = log_int(1, 128)
            case["keep"] = max(case["window"], int(case["T_min"] * rng.uniform(0.1, 1.0)))
        else:
            case["step"] = rng.choice([0, 1])
    return case


# ------------------------------------------------------------------------------------------------------------ inputs
def _lengths(case, cpu):
    return torch.randint(case["T_min"], case["T"] + 1, (case["B"],), generator=cpu)


def _counts(case):
    """Query tokens per request: the draft model stops early in some of the requests of a batch of trees."""
    n = case["n"]
    return [n - (b * 7) % (n // 4 + 1) if case["tree"] else n for b in range(case["B"])]


def _cache(case, layers, nb, gen):
    """[layers, 2, nb, bs, H, D] or, with the K/V axis behind the blocks, its permutation; bf16."""
    H, D, bs = case["Hkv"], case["D"], case["bs"]
    inner = (H, bs, D) if case["hnd"] else (bs, H, D)
    outer = (2, nb) if case["axis"] == 0 else (nb, 2)
    big = torch.empty((layers, *outer, *inner), dtype=torch.bfloat16, device=DEV)
    big.normal_(generator=gen)
    return big.transpose(3, 4) if case["hnd"] else big


def _trees(case, counts, cpu):
    """One 64-bit word per query token: bit j set where it sees drafted token j of its request."""
    words = []
    for c in counts:
        mine = []
        for i in range(c):
            parent = int(torch.randint(-1, i, (1,), generator=cpu)) if i else -1
            mine.append((mine[parent] if parent >= 0 else 0) | (1 << i))
        words += [w - (1 << 64) if w >= (1 << 63) else w for w in mine]
    return torch.tensor(words, dtype=torch.int64)


def prepare(case, seed):
    cpu = torch.Generator().manual_seed(int(seed))
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    op, B, bs, H, D = case["op"], case["B"], case["bs"], case["Hkv"], case["D"]
    lens = _lengths(case, cpu)
    width = (case["T"] + bs - 1) // bs
    nb = B * width + 7
    s = {"case": case}
    layers = case.get("L", 1)
    s["cache"] = _cache(case, layers, nb, gen)
    s["table"] = torch.randperm(nb, generator=cpu)[: B * width].view(B, width).to(torch.int32).to(DEV)
    s["lens"] = lens.to(torch.int32).to(DEV)
    if op in ("attend", "observe", "sparse"):
        counts = _counts(case)
        start = [0]
        for c in counts:
            start.append(start[-1] + c)
        s["start"] = torch.tensor(start, dtype=torch.int32).to(DEV)
        s["q"] = torch.randn((start[-1], H * case["g"], D), generator=gen, device=DEV).mul_(1.5).to(torch.bfloat16)
        s["tree"] = _trees(case, counts, cpu).to(DEV) if case["tree"] else None
    if op == "observe":
        s["sums"] = torch.rand((nb, H, bs), generator=gen, device=DEV).square_()
    if op == "evict":
        # a heavy tail, and many tokens that share the same small value
        w = torch.randn((layers, nb, H, bs), generator=gen, device=DEV).exp_()
        s["fresh"] = torch.where(w < 0.7, (w * 16).round() / 16, w)
        s["sums"] = s["fresh"].clone()
        s["keep"] = torch.minimum(lens, torch.tensor(case["keep"])).to(torch.int32).to(DEV)
    if op == "bounds":
        s["bounds"] = torch.zeros((layers, nb, H, 2, D), dtype=torch.bfloat16, device=DEV)
        s["first"] = (lens - 1 if case["step"] else torch.zeros_like(lens)).to(torch.int32).to(DEV)
    if op == "sparse":
        k = _split(s["cache"][0], case["axis"])[0]
        pos = torch.arange(width * bs, device=DEV)
        out = (pos.view(1, width, bs) >= s["lens"].view(B, 1, 1)).view(B, width, bs, 1, 1)
        kb = k[s["table"].long()]                                                   # [B, width, bs, H, D]
        lo = kb.masked_fill(out, float("inf")).amin(2)
        hi = kb.masked_fill(out, float("-inf")).amax(2)
        s["bounds"] = torch.zeros((nb, H, 2, D), dtype=torch.bfloat16, device=DEV)
        live = (pos[::bs].view(1, width) < s["lens"].view(B, 1)).view(B, width, 1, 1, 1)
        s["bounds"][s["table"].long()] = torch.where(live, torch.stack([lo, hi], 3), torch.zeros_like(lo).unsqueeze(3))
    return s


def _split(cache, axis):
    return (cache[0], cache[1]) if axis == 0 else (cache[:, 0], cache[:, 1])


# ------------------------------------------------------------------------------------------------------------- plain
def _padded_queries(s, H, g, D):
    """[B, n, H, g, D] fp32 (zeros behind a request's last token), the row of each and whether it exists."""
    start, n = s["start"].long(), s["case"]["n"]
    row = start[:-1, None] + torch.arange(n, device=DEV)
    there = row < start[1:, None]
    row = torch.where(there, row, 0)
    q = s["q"][row].float().masked_fill(~there[:, :, None, None], 0.0)
    return q.view(q.shape[0], n, H, g, D), row, there


def _plain_attend(s, blocks=None, sums=None):
    """Attention over all cached tokens, or over the listed blocks [B, H, S] of each KV head (-1: none)."""
    c = s["case"]
    H, g, D, bs, n, B = c["Hkv"], c["g"], c["D"], c["bs"], c["n"], c["B"]
    k, v = _split(s["cache"][0], c["axis"])
    table, lens = s["table"].long(), s["lens"].long()
    off = torch.arange(bs, device=DEV)
    if blocks is None:
        pos = torch.arange(table.shape[1] * bs, device=DEV).expand(B, 1, -1)
        phys = table.repeat_interleave(bs, 1)
        valid = pos < lens[:, None, None]
        kk = k[phys, pos[:, 0] % bs].transpose(1, 2)                                # [B, H, T, D]
        vv = v[phys, pos[:, 0] % bs].transpose(1, 2)
    else:
        listed_ = blocks >= 0
        b0 = blocks.clamp(min=0).long()
        pos = (b0[..., None] * bs + off).flatten(2)                                 # [B, H, S * bs]
        phys = table.gather(1, b0.flatten(1)).view_as(b0).repeat_interleave(bs, 2)
        valid = listed_.repeat_interleave(bs, 2) & (pos < lens[:, None, None])
        head = torch.arange(H, device=DEV).view(1, H, 1)
        kk, vv = k[phys, pos % bs, head], v[phys, pos % bs, head]
    kk, vv = kk.float(), vv.float()
    q, row, there = _padded_queries(s, H, g, D)
    count = (s["start"][1:] - s["start"][:-1]).long()
    draft = pos - (lens - count)[:, None, None]                                     # < 0: context
    word = s["tree"][row] if s["tree"] is not None else None
    if word is None:
        # a chain: query token i sees drafted tokens 0..i
        sees = draft[:, :, None, :] <= torch.arange(n, device=DEV)[:, None]
    else:
        sees = (draft[:, :, None, :] < 0) | (((word[:, None, :, None] >> draft.clamp(0, 63)[:, :, None, :]) & 1) != 0)
    sees = sees & valid[:, :, None, :] & there[:, None, :, None]                    # [B, 1 or H, n, T]
    qh = q.permute(0, 2, 1, 3, 4).reshape(B, H, n * g, D)
    x = qh @ kk.transpose(2, 3) * (1.0 / math.sqrt(D))                              # [B, H, n * g, T]
    x = x.view(B, H, n, g, -1).masked_fill(~sees[:, :, :, None, :], float("-inf"))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    inv = torch.where(total > 0, 1.0 / total, torch.zeros_like(total))
    vv = vv.masked_fill(~valid[..., None], 0.0)
    o = (p.view(B, H, n * g, -1) @ vv).view(B, H, n, g, D) * inv
    lse = (top + torch.log(total)).squeeze(-1)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, n, H * g, D).to(torch.bfloat16)
    lse = lse.permute(0, 2, 1, 3).reshape(B, n, H * g)
    flat = torch.nonzero(there.flatten()).flatten()
    o, lse = o.flatten(0, 1)[flat], lse.flatten(0, 1)[flat]
    if sums is None:
        return o, lse
    add = (p * inv).sum((2, 3))                                                     # [B, H, T]
    head = torch.arange(H, device=DEV).view(1, H, 1)
    old = sums[phys[:, None], head, pos % bs]
    fresh = draft >= 0 if not c["reset"] else torch.ones_like(draft, dtype=torch.bool)
    new = torch.where(fresh, torch.zeros_like(old), old) + add
    sums[phys[:, None], head, pos % bs] = torch.where(valid, new, old)
    return o, lse, sums


def _plain_evict(s):
    c = s["case"]
    L, B, H, bs, T = c["L"], c["B"], c["Hkv"], c["bs"], c["T"]
    cache, sums = s["cache"], s["sums"]
    table, lens, keep = s["table"].long(), s["lens"].long(), s["keep"].long()
    pitch = min(c["keep"], T)
    pos = torch.arange(T, device=DEV)
    phys, off = table[:, pos // bs], pos % bs
    layer, head = torch.arange(L, device=DEV).view(L, 1, 1, 1), torch.arange(H, device=DEV).view(1, 1, H, 1)
    x = sums[layer, phys.view(1, B, 1, T), head, off]                               # [L, B, H, T]
    x = x.masked_fill((pos >= lens[:, None] - c["window"]).view(1, B, 1, T), float("inf"))
    x = x.masked_fill((pos >= lens[:, None]).view(1, B, 1, T), float("-inf"))
    best = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :pitch]
    r = torch.arange(pitch, device=DEV)
    kept = r < keep.view(1, B, 1, 1)
    chosen = torch.sort(torch.where(kept, best, T), dim=-1).values
    dst = torch.minimum(r, lens.view(1, B, 1, 1) - 1).expand_as(chosen)
    src = torch.where(kept, chosen, dst)
    bi = torch.arange(B, device=DEV).view(1, B, 1, 1)
    ps, os_, pd, od = table[bi, src // bs], src % bs, table[bi, dst // bs], dst % bs
    for_kv = cache if c["axis"] == 0 else cache.transpose(1, 2)
    rows = for_kv[layer, :, ps, os_, head]
    for_kv[layer, :, pd, od, head] = rows
    sums[layer, pd, head, od] = sums[layer, ps, head, os_]
    return torch.where(kept, chosen, -1).to(torch.int32), cache, sums


def _plain_bounds(s):
    c = s["case"]
    L, B, bs = c["L"], c["B"], c["bs"]
    k = s["cache"][:, 0] if c["axis"] == 0 else s["cache"][:, :, 0]                 # [L, nb, bs, H, D]
    table, lens, first = s["table"].long(), s["lens"].long(), s["first"].long()
    width = 1 if c["step"] else table.shape[1]
    idx = (first // bs).view(B, 1) + torch.arange(width, device=DEV)
    live = idx * bs < lens.view(B, 1)
    phys = table.gather(1, idx.clamp(max=table.shape[1] - 1))
    pos = idx[..., None] * bs + torch.arange(bs, device=DEV)
    out = (pos >= lens.view(B, 1, 1)).view(1, B, width, bs, 1, 1)
    kb = k[:, phys]                                                                 # [L, B, width, bs, H, D]
    lo = kb.masked_fill(out, float("inf")).amin(3)
    hi = kb.masked_fill(out, float("-inf")).amax(3)
    new = torch.stack([lo, hi], 4)
    s["bounds"][:, phys] = torch.where(live.view(1, B, width, 1, 1, 1), new, s["bounds"][:, phys])
    return s["bounds"]


def _plain_select(s):
    c = s["case"]
    H, g, D, bs, B = c["Hkv"], c["g"], c["D"], c["bs"], c["B"]
    table, lens = s["table"].long(), s["lens"].long()
    q, _, _ = _padded_queries(s, H, g, D)
    q = q.double()
    up, down = q.clamp(min=0).sum((1, 3)), q.clamp(max=0).sum((1, 3))               # [B, H, D]
    bnd = s["bounds"][table].double()                                               # [B, width, H, 2, D]
    x = (bnd[:, :, :, 1] * up[:, None] + bnd[:, :, :, 0] * down[:, None]).sum(-1).float().transpose(1, 2)
    blk = torch.arange(table.shape[1], device=DEV)
    have = (lens + bs - 1) // bs
    count = (s["start"][1:] - s["start"][:-1]).long()
    from_ = torch.minimum(have - c["recent"], (lens - count) // bs)
    forced = (blk < c["sink"]) | (blk >= from_[:, None])
    x = x.masked_fill(forced[:, None], float("inf")).masked_fill((blk >= have[:, None])[:, None], float("-inf"))
    sel = c["sel"]
    best = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :sel]
    best = torch.nn.functional.pad(best, (0, sel - best.shape[-1]))
    there = torch.arange(sel, device=DEV) < have.view(B, 1, 1)
    none = table.shape[1]
    best = torch.sort(torch.where(there, best, none), dim=-1).values
    return torch.where(best < none, best, -1).to(torch.int32)


# --------------------------------------------------------------------------------------------------------------- run
def run(state):
    s = state
    c = s["case"]
    op = c["op"]
    if op == "evict":
        # attention has refilled the sums since the last eviction: every pass evicts as much as the first
        s["sums"].copy_(s["fresh"])
    if not own:
        if op == "attend":
            return _plain_attend(s)
        if op == "observe":
            return _plain_attend(s, sums=s["sums"])
        if op == "evict":
            return _plain_evict(s)
        if op == "bounds":
            return _plain_bounds(s)
        blocks = _plain_select(s)
        return (blocks, *_plain_attend(s, blocks))
    from triattention_b200 import ops
    if op in ("attend", "observe", "sparse"):
        kv = s["cache"][0]
        if op == "attend":
            return ops.attend_paged(s["q"], kv, s["table"], s["lens"], s["start"], c["n"], tree_mask=s["tree"],
                                    kv_axis=c["axis"])
        if op == "observe":
            out, lse = ops.attend_paged(s["q"], kv, s["table"], s["lens"], s["start"], c["n"], tree_mask=s["tree"],
                                        weight_sums=s["sums"], reset_weight_sums=c["reset"], kv_axis=c["axis"])
            return out, lse, s["sums"]
        blocks = ops.select_blocks(s["q"], s["bounds"], s["lens"], s["start"], s["table"], c["n"], c["bs"], c["sel"],
                                   sink_blocks=c["sink"], recent_blocks=c["recent"])
        return (blocks, *ops.attend_paged(s["q"], kv, s["table"], s["lens"], s["start"], c["n"], tree_mask=s["tree"],
                                          block_list=blocks, kv_axis=c["axis"]))
    view = ops.PagedCacheView.from_layers(list(s["cache"].unbind(0)), kv_axis=c["axis"])
    layout = view.layout(c["B"], 1, s["table"].shape[1])
    if op == "evict":
        keep = ops.evict_paged(view, layout, s["sums"], s["table"], s["lens"], s["keep"], min(c["keep"], c["T"]), c["window"])
        return keep, s["cache"], s["sums"]
    ops.update_block_bounds(view, layout, s["bounds"], s["table"], s["first"], s["lens"])
    return s["bounds"]


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Lengths are drawn between T_min and T: their mean stands for them."""
    c = case
    op, B, H, D, bs = c["op"], c["B"], c["Hkv"], c["D"], c["bs"]
    T = (c["T"] + c["T_min"]) / 2
    row = D * 2
    if op in ("attend", "observe", "sparse"):
        queries = sum(_counts(c)) * H * c["g"]
        cost = {"bytes": queries * (2 * row + 4), "flops": 0.0}
        tokens = T
        if op == "sparse":
            tokens = min(T, c["sel"] * bs)
            cost["bytes"] += B * H * (T / bs * 2 * row + c["sel"] * 4)
            cost["flops"] += B * H * T / bs * 4 * D
        if op == "observe":
            cost["bytes"] += B * H * T * (4 if c["reset"] else 8)
        cost["bytes"] += B * H * tokens * 2 * row
        cost["flops"] += queries * tokens * 4 * D
        return cost
    L = c["L"]
    if op == "evict":
        # sums restored (read, write), read by the selection; kept rows of K, V and sums read and written
        moved = min(c["keep"], T)
        return {"bytes": L * B * H * (T * 12 + moved * (4 * row + 4 + 4)), "flops": L * B * H * T}
    blocks = 1 if c["step"] else T / bs
    tokens = min(T, bs / 2) if c["step"] else T
    return {"bytes": L * B * H * (tokens * row + blocks * 2 * row), "flops": L * B * H * tokens * 2 * D}


# ------------------------------------------------------------------------------------------------------------- exact
def _exact_one(q, k, v, see):
    """q [R, D], k/v [T, D], see [R, T] in 64 bits -> output, log of the sum, probabilities."""
    x = torch.einsum("rd,td->rt", q, k) / (k.shape[-1] ** 0.5)
    x = torch.where(see, x, torch.full_like(x, float("-inf")))
    lse = torch.logsumexp(x, -1)
    p = torch.softmax(x, -1).nan_to_num(0.0)
    return p @ v, lse, p


def _exact_choice(c, q, lo, hi, T):
    """Truth value per block: q [n, g, D] and bounds lo/hi [blocks, D] of one KV head in 64 bits."""
    bs = c["bs"]
    score = torch.zeros(lo.shape[0], dtype=torch.float64, device=DEV)
    for row in q.flatten(0, 1):
        score += torch.maximum(row * lo, row * hi).sum(-1)
    score = score.float()
    score[: c["sink"]] = float("inf")
    score[max(0, min(lo.shape[0] - c["recent"], (T - q.shape[0]) // bs)) :] = float("inf")
    some = torch.zeros(lo.shape[0], dtype=torch.bool, device=DEV)
    some[torch.argsort(score, descending=True, stable=True)[: c["sel"]]] = True
    return some


def exact(case, seed):
    c = case
    op = c["op"]
    if op in ("evict", "bounds"):
        return None  # moved and compared values, nothing is computed
    s = prepare(case, seed)
    H, g, D, bs = c["Hkv"], c["g"], c["D"], c["bs"]
    k, v = _split(s["cache"][0], c["axis"])
    start, lens = s["start"].tolist(), s["lens"].tolist()
    N = start[-1]
    out = torch.zeros((N, H * g, D), dtype=torch.float64, device=DEV)
    lse = torch.zeros((N, H * g), dtype=torch.float64, device=DEV)
    sums = s["sums"].double() if op == "observe" else None
    for b in range(c["B"]):
        T, n = lens[b], start[b + 1] - start[b]
        ctx = T - n
        see = torch.ones((n, T), dtype=torch.bool, device=DEV)
        for i in range(n):
            word = int(s["tree"][start[b] + i]) if s["tree"] is not None else (1 << (i + 1)) - 1
            see[i, ctx:] = torch.tensor([bool((word >> j) & 1) for j in range(n)], device=DEV)
        used = s["table"][b, : (T + bs - 1) // bs].long()
        for h in range(H):
            kk = k[used, :, h].reshape(-1, D)[:T].double()
            vv = v[used, :, h].reshape(-1, D)[:T].double()
            mine = see
            qq = s["q"][start[b] : start[b + 1], h * g : (h + 1) * g].double()
            if op == "sparse":
                bnd = s["bounds"][used, h].double()
                mine = see & _exact_choice(c, qq, bnd[:, 0], bnd[:, 1], T).repeat_interleave(bs)[:T]
            qq = qq.reshape(n * g, D)
            o, z, p = _exact_one(qq, kk, vv, mine.repeat_interleave(g, 0))
            out[start[b] : start[b + 1], h * g : (h + 1) * g] = o.view(n, g, D)
            lse[start[b] : start[b + 1], h * g : (h + 1) * g] = z.view(n, g)
            if sums is not None:
                at = torch.arange(T, device=DEV)
                old = sums[used[at // bs], h, at % bs]
                old = torch.zeros_like(old) if c["reset"] else torch.where(at >= ctx, torch.zeros_like(old), old)
                sums[used[at // bs], h, at % bs] = old + p.sum(0)
    if op == "attend":
        return out, lse
    if op == "observe":
        return out, lse, sums
    return None, out, lse
