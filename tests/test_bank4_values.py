"""That the limit of bank4_values tells a layer on a bank in 4 bits from one that
rounds once more: the roundings are planted in the reference."""
from __future__ import annotations

import pytest
import torch

from bank4_values import LIMIT, distance, layer
from moe_amd.layer import moe_layer
from pack4_oracle import held
from test_pack4 import _packed

BF = torch.bfloat16


def _case(T=24, E=4, K=2, H=256, I=128):
    g = torch.Generator().manual_seed(T)
    w1 = held(torch.randn(E, 2 * I, H, generator=g) * 0.02)
    w2 = held(torch.randn(E, H, I, generator=g) * 0.02)
    x = torch.randn(T, H, generator=g).to(BF)
    idx = torch.rand(T, E, generator=g).argsort(1)[:, :K].contiguous()
    return x, idx, torch.rand(T, K, generator=g) + 0.1, w1, w2


@pytest.mark.parametrize("act_bf16", [False, True])
def test_the_form_itself_is_within(act_bf16):
    case = _case()
    ref = layer(*case, act_bf16)
    assert distance(ref.to(BF), ref) == 1.0
    # y in fp16 of its own power of two
    x, idx, w, w1, w2 = case
    assert distance((ref * (1 + 2.0 ** -11 / 3 ** 0.5 * torch.randn(ref.shape))).to(BF), ref) < 1.1


@pytest.mark.parametrize("name", ["gate_up", "silu", "act", "y", "w", "wy"])
@pytest.mark.parametrize("act_bf16", [False, True])
def test_another_rounding_is_not(act_bf16, name):
    if act_bf16 and name == "act":
        pytest.skip("this form makes that rounding")
    case = _case()
    ref = layer(*case, act_bf16)
    assert distance(layer(*case, act_bf16, planted=(name,)).to(BF), ref) > LIMIT
