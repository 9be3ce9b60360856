"""Which form of the permutation a call takes, and its outputs at that border."""
from __future__ import annotations

import pytest
import torch
from torch.profiler import ProfilerActivity, profile

from moe_amd import ops
from test_gpu_permute_chunks import _check

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _launches(idx, E, calls=1):
    """(name, us) of the kernels of ``calls`` calls."""
    ops.permute(idx, E)
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        for _ in range(calls):
            ops.permute(idx, E)
        torch.cuda.synchronize()
    return [(e.name, e.device_time) for e in p.events() if "_kernel" in e.name]


@pytest.mark.parametrize("E,one", [(2160, True), (2161, True), (2287, True), (2288, False)])
@pytest.mark.parametrize("S", [16, 1025, 16384])
def test_many_experts(S, E, one):
    """Up to 2287 experts' counters fit the LDS of the form of one launch."""
    g = torch.Generator(device=DEV).manual_seed(S + E)
    idx = torch.randint(-1, E + 1, (S, 1), generator=g, device=DEV)
    _check(idx, E)
    assert len(_launches(idx, E)) == (1 if one else 3)


def _skewed(S, E, share, g):
    """Ids of which ``share`` are one expert's and the rest anybody's."""
    idx = torch.randint(-1, E + 1, (S, 1), generator=g, device=DEV)
    return torch.where(torch.rand(S, 1, generator=g, device=DEV) < share, E // 2, idx)


@pytest.mark.parametrize("E", [1, 4, 31, 128, 2287])
@pytest.mark.parametrize("share", [0.2, 0.37, 0.4, 0.8, 1.0])
@pytest.mark.parametrize("S", [6144, 6145, 8192, 12345, 16383, 16384])
def test_skewed_routing(S, share, E):
    _check(_skewed(S, E, share, torch.Generator(device=DEV).manual_seed(S)), E)


@pytest.mark.parametrize("S", [6145, 9000, 16384])
def test_segments(S):
    """An expert that has all of the first entries and none of the others, all but the first
    ones, and ids outside [0, E) alike."""
    E = 40
    for e in (0, 39, -1):
        for n in (64, 1024, 5000):
            idx = torch.randint(0, E, (S, 1), device=DEV)
            idx[:n] = e
            _check(idx, E)
            _check(idx.flip(0).contiguous(), E)


def test_skew_costs_no_more_than_launches():
    """16384 entries to one expert: the kernel's time, the median of 15, within twice that
    of even routing (it was four times)."""
    def us(idx):
        t = sorted(d for _, d in _launches(idx, 128, 15))
        return t[len(t) // 2]
    even = torch.arange(16384, device=DEV)[:, None] % 128
    assert us(torch.full_like(even, 5)) < 2 * us(even)
