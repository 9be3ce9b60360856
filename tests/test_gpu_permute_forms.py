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
