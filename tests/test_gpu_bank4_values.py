"""The values of the layer on a bank in 4 bits where they are largest."""
from __future__ import annotations

import pytest
import torch

from moe_amd import few, ops

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


@pytest.mark.parametrize("T", [1, 2, 16])
def test_acts_beyond_bf16(T):
    """One feature's act above the largest bf16 value, finite in fp32 or not: its sums
    are its own, not NaN.  gate = 2^64, up = 2^64 (1 - 2^-10) or 2^65, all others 0."""
    H, I, E = 64, 64, 1
    w1 = torch.zeros(E, 2 * I, H, device=DEV)
    w1[0, 0, 0] = w1[0, I, 0] = 1.0
    w1[0, I, 1] = 1.0
    w2 = torch.full((E, H, I), 2.0 ** -6, device=DEV)
    w2[0, ::2] *= -1
    b1, b2 = ops.pack4(w1, dtype=BF), ops.pack4(w2, dtype=BF)
    idx, w = torch.zeros(T, 1, device=DEV, dtype=torch.int64), torch.ones(T, 1, device=DEV)
    sign = torch.where(torch.arange(H, device=DEV) % 2 == 0, -1.0, 1.0)
    x = torch.zeros(T, H, device=DEV, dtype=BF)
    x[:, 0], x[:, 1] = 2.0 ** 64, -2.0 ** 54
    out = few.experts_forward_few(x, idx, w, b1, b2).float()
    # 2^122 (1 - 2^-10), which is nearer to 2^122 than to the bf16 value below it
    assert torch.equal(out, (sign * 2.0 ** 122).expand(T, H))
    x[:, 1] = 2.0 ** 64
    for n in (T, 40):      # 40 tokens: the form that rounds act
        out = few.experts_forward_few(x[:1].expand(n, H), idx[:1].expand(n, 1), w[:1].expand(n, 1),
                                      b1, b2).float()
        assert torch.equal(out, (sign * torch.inf).expand(n, H)), n
