"""Banks in 4 bits: what a call or a packing refuses, it refuses before it changes
or computes anything."""
from __future__ import annotations

import pytest
import torch

from moe_amd.layer import moe_layer
from test_pack4 import _packed

BF = torch.bfloat16


def test_neither_or_both_weights_are_packed():
    x, wr = torch.zeros(4, 64, dtype=BF), torch.zeros(3, 64, dtype=BF)
    for router in ("softmax", "sigmoid"):
        with pytest.raises(TypeError, match="both be in 4 bits"):
            moe_layer(x, wr, torch.zeros(3, 128, 64, dtype=BF), _packed(3, 64, 64), 2, router=router)
