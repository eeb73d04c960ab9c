"""Recipes that the integration guide spells out in code, run as they stand there."""
from __future__ import annotations

import re
import textwrap
from pathlib import Path

import torch

TEXT = (Path(__file__).resolve().parent.parent / "INTEGRATION.md").read_text()


def snippet(mark: str) -> str:
    """The one code block that holds ``mark``."""
    found = [m for m in re.findall(r"^ *```python\n(.*?)^ *```", TEXT, re.S | re.M) if mark in m]
    assert len(found) == 1, mark
    return textwrap.dedent(found[0])


def test_sums_of_accepted_drafts_move_with_their_tokens():
    """Three requests (one keeps all, one accepts a path across a block's end, one only its context): every kept token's sum is found in
    its new slot, and slots that no kept token moves to hold what they held."""
    gen = torch.Generator().manual_seed(3)
    L, H, bs, B, width = 2, 3, 4, 3, 5
    nb = B * width + 2
    block_table = torch.randperm(nb, generator=gen)[: B * width].view(B, width).to(torch.int32)
    sums = torch.rand((L, nb, H, bs), generator=gen)
    before = sums.clone()
    rows = [list(range(17)), list(range(10)) + [11, 14, 15], list(range(6))]
    pitch = max(len(r) for r in rows)
    keep = torch.tensor([r + [-1] * (pitch - len(r)) for r in rows], dtype=torch.int32)
    exec(snippet("the tokens that move"), {"torch": torch, "keep": keep, "block_table": block_table, "sums": sums, "block_size": bs})
    want = before.clone()
    for b, row in enumerate(rows):
        for new, old in enumerate(row):
            want[:, block_table[b, new // bs].long(), :, new % bs] = before[:, block_table[b, old // bs].long(), :, old % bs]
    assert torch.equal(sums, want) and not torch.equal(sums, before)
