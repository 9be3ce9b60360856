"""The permutation in one launch, a workgroup for each 1024 entries, at its borders:
against a stable sort, all outputs whole."""
from __future__ import annotations

import pytest
import torch

from moe_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _check(idx, E):
    T, K = idx.shape
    plan = ops.permute(idx, E)
    bins = torch.where((idx >= 0) & (idx < E), idx, E).flatten()
    order = torch.sort(bins, stable=True)[1]
    assert torch.equal(plan.row_src.long(), order)
    slot = torch.empty_like(order)
    slot[order] = torch.arange(T * K, device=DEV)
    assert torch.equal(plan.slot.long(), slot)
    counts = torch.bincount(bins, minlength=E + 1)[:E]
    assert torch.equal(plan.counts.long(), counts)
    first = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    assert torch.equal(plan.offsets.long(), first)
    for b, rows in enumerate((64, 128, 256)):
        tiles = (counts + rows - 1) // rows
        starts = torch.cat([tiles.new_zeros(1), tiles.cumsum(0)])
        assert torch.equal(plan.tile_starts[b].long(), starts), rows
    return plan


@pytest.mark.parametrize("E,K", [(1, 1), (5, 3), (128, 8), (1792, 8), (2160, 4)])
@pytest.mark.parametrize("S", [1, 63, 64, 65, 1023, 1024, 1025, 2049, 8191, 8193, 16384, 16385])
def test_borders(S, E, K):
    if S % K:
        K = 1
    g = torch.Generator(device=DEV).manual_seed(S + E)
    idx = torch.randint(-1, E + 1, (S // K, K), generator=g, device=DEV)
    _check(idx, E)


@pytest.mark.parametrize("S", [1, 1024, 5000, 16384])
@pytest.mark.parametrize("e", [-1, 0, 3, 6, 7])
def test_all_to_one(S, e):
    """One expert has every entry, the last one, or none has any (ids outside)."""
    _check(torch.full((S, 1), e, device=DEV), 7)


def test_calls_by_turns():
    """Calls of both forms and sizes after one another leave nothing to each other."""
    g = torch.Generator(device=DEV).manual_seed(3)
    for S in (16384, 40, 20000, 1025, 16384, 17, 8168):
        _check(torch.randint(0, 128, (S, 1), generator=g, device=DEV), 128)
    assert ops.permute(torch.empty(0, 8, device=DEV, dtype=torch.int64), 16).offsets.tolist() == [0] * 17
