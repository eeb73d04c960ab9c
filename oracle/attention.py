"""64-bit oracle of the operators that attend to the paged cache: attention, weight sums, eviction, block choice.

Plain restatements of the formulas for one request (one layer) at a time; inputs are the tensors the kernels get.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch


def token_slots(table_row: Sequence[int], block_size: int, num_tokens: int):
    """(block, offset) index tensors of tokens 0 .. num_tokens - 1."""
    pos = torch.arange(num_tokens)
    row = torch.as_tensor(list(table_row), dtype=torch.long)
    return row[pos // block_size], pos % block_size


def visible(num_tokens: int, num_queries: int, words: Optional[Sequence[int]]) -> torch.Tensor:
    """[n, T] truth values: context tokens always, own token j where bit j of the row's word is set (chain without words)."""
    ctx = num_tokens - num_queries
    see = torch.ones((num_queries, num_tokens), dtype=torch.bool)
    for i in range(num_queries):
        word = (1 << (i + 1)) - 1 if words is None else int(words[i])
        for j in range(num_queries):
            see[i, ctx + j] = bool((word >> j) & 1)
    return see


def attend_request(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, see: torch.Tensor, scale: float):
    """One request.  q [n, Hq, D], k / v [T, Hkv, D], see [n, T] or [Hkv, n, T].

    Returns a dict of float64 tensors: out [n, Hq, D], lse [n, Hq], weight [Hkv, T] (sum over the rows of each KV head),
    spread [n, Hq, D] = sum_t p_t |v_t| and logit [n, Hq] = max_t scale sum_d |q_d k_td| (error bounds build on these).
    """
    n, Hq, D = q.shape
    T, H, _ = k.shape
    g = Hq // H
    if see.dim() == 2:
        see = see.expand(H, n, T)
    out, spread = torch.zeros(n, Hq, D, dtype=torch.float64), torch.zeros(n, Hq, D, dtype=torch.float64)
    lse, logit = torch.full((n, Hq), -math.inf, dtype=torch.float64), torch.zeros(n, Hq, dtype=torch.float64)
    weight = torch.zeros(H, T, dtype=torch.float64)
    q, k, v = q.double(), k.double(), v.double()
    for h in range(H):
        for j in range(g):
            for i in range(n):
                t = torch.nonzero(see[h, i]).flatten()
                if t.numel() == 0:
                    continue
                row = q[i, h * g + j]
                s = scale * (k[t, h] @ row)
                z = torch.logsumexp(s, 0)
                p = torch.exp(s - z)
                lse[i, h * g + j] = z
                out[i, h * g + j] = p @ v[t, h]
                spread[i, h * g + j] = p @ v[t, h].abs()
                logit[i, h * g + j] = scale * (k[t, h].abs() @ row.abs()).max()
                weight[h, t] += p
    return {"out": out, "lse": lse, "weight": weight, "spread": spread, "logit": logit}


def evict_keep(weights: torch.Tensor, keep: int, window: int, prefill_len: int = 0) -> torch.Tensor:
    """Ascending indices of the ``keep`` largest of one row [T]; ties to the lowest index, guarded tokens first, NaN last."""
    x = weights.double().clone()
    x[torch.isnan(x)] = -math.inf
    T = x.numel()
    x[max(0, T - window):] = math.inf
    x[:prefill_len] = math.inf
    order = sorted(range(T), key=lambda t: (-float(x[t]), t))[: min(keep, T)]
    return torch.tensor(sorted(order), dtype=torch.int32)


def block_bounds(k: torch.Tensor, block_size: int):
    """(min, max) [blocks, Hkv, D] over the tokens of each block of k [T, Hkv, D]."""
    parts = k.split(block_size)
    return torch.stack([p.amin(0) for p in parts]), torch.stack([p.amax(0) for p in parts])


def block_scores(q: torch.Tensor, lo: torch.Tensor, hi: torch.Tensor) -> torch.Tensor:
    """[Hkv, blocks] fp32 (rounded once): sum over the rows of a KV head of the upper bound of q . k."""
    n, Hq, D = q.shape
    nb, H, _ = lo.shape
    g = Hq // H
    out = torch.zeros(H, nb, dtype=torch.float64)
    for h in range(H):
        for row in q[:, h * g : (h + 1) * g].reshape(-1, D).double():
            out[h] += torch.maximum(row * lo[:, h].double(), row * hi[:, h].double()).sum(-1)
    return out.float()


def select_blocks(scores: torch.Tensor, num_tokens: int, num_queries: int, block_size: int, num_selected: int,
                  sink: int, recent: int) -> torch.Tensor:
    """[Hkv, num_selected] int32 ascending, -1 behind the last block."""
    H, nb = scores.shape
    x = scores.double().clone()
    x[:, :sink] = math.inf
    x[:, max(0, min(nb - recent, (num_tokens - num_queries) // block_size)):] = math.inf
    out = torch.full((H, num_selected), -1, dtype=torch.int32)
    for h in range(H):
        order = sorted(sorted(range(nb), key=lambda b: (-float(x[h, b]), b))[: min(num_selected, nb)])
        out[h, : len(order)] = torch.tensor(order, dtype=torch.int32)
    return out
