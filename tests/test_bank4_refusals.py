"""Banks in 4 bits: what a call or a packing refuses, it refuses before it changes
or computes anything."""
from __future__ import annotations

import pytest
import torch
from torch import nn

from moe_amd import _lib, hf, ops
from moe_amd.experts import pack_bank
from moe_amd.layer import SparseMoeBlock, moe_layer
from test_pack4 import _pack_on_cpu, _packed

BF = torch.bfloat16


def test_neither_or_both_weights_are_packed():
    x, wr = torch.zeros(4, 64, dtype=BF), torch.zeros(3, 64, dtype=BF)
    for router in ("softmax", "sigmoid"):
        with pytest.raises(TypeError, match="both be in 4 bits"):
            moe_layer(x, wr, torch.zeros(3, 128, 64, dtype=BF), _packed(3, 64, 64), 2, router=router)


def _bank(shape1, shape2):
    """A bank of bf16 weights that take no memory."""
    bank = nn.Module()
    for name, shape in (("gate_up_proj", shape1), ("down_proj", shape2)):
        setattr(bank, name, nn.Parameter(torch.zeros(1, 1, 1, dtype=BF).expand(shape)))
    return bank


@pytest.mark.parametrize("spoil,error", [
    (lambda b: b.float(), NotImplementedError),
    (lambda b: setattr(b, "has_bias", True), NotImplementedError),
    (lambda b: setattr(b, "down_proj", nn.Parameter(torch.zeros(3, 64, 128, dtype=BF))), ValueError),
    (lambda b: setattr(b, "gate_up_proj", nn.Parameter(torch.zeros(3, 128, 96, dtype=BF))),
     ValueError),
])
def test_a_model_is_packed_whole_or_not_at_all(monkeypatch, spoil, error):
    _pack_on_cpu(monkeypatch)
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    model = nn.ModuleList(SparseMoeBlock(64, 3, 2, 64).bfloat16() for _ in range(3))
    spoil(model[1].experts)
    with pytest.raises(error, match="mi355x experts|pack_bank"):
        hf.pack_experts(model)
    for block in model:
        assert sorted(n for n, _ in block.experts.named_parameters()) == ["down_proj", "gate_up_proj"]
        assert not list(block.experts.buffers())
    model[1] = SparseMoeBlock(64, 3, 2, 64).bfloat16()
    assert hf.pack_experts(model) == 3
    assert not any(list(b.experts.parameters()) for b in model)


def test_a_bank_elsewhere_keeps_a_model_as_it_is(monkeypatch):
    model = nn.ModuleList(SparseMoeBlock(64, 3, 2, 64).bfloat16() for _ in range(2))
    with pytest.raises(RuntimeError, match="GPU only"):
        hf.pack_experts(model)
    assert all(len(list(b.experts.parameters())) == 2 for b in model)


@pytest.mark.parametrize("E,H,I", [(10240, 64, 64), (1, (1 << 22) + 64, 64), (1, 64, (1 << 22) + 64),
                                   (2, 1 << 16, 1 << 16)])
def test_banks_that_no_call_takes_are_not_packed(built_lib, monkeypatch, E, H, I):
    _pack_on_cpu(monkeypatch)
    assert _lib.load().moe_amd_experts4_workspace_size(1, E, 1, H, I) == 0
    bank = _bank((E, 2 * I, H), (E, H, I))
    with pytest.raises(NotImplementedError, match="pack_bank"):
        pack_bank(bank)
    assert bank.gate_up_proj.shape == (E, 2 * I, H)


def test_the_largest_banks_are(built_lib):
    for E, H, I in ((10239, 64, 64), (1, 1 << 22, 64), (1, 64, 1 << 22), (1, 1 << 16, (1 << 15) - 64)):
        assert _lib.load().moe_amd_experts4_workspace_size(1, E, 1, H, I) > 0
        ops.check_bank4_size("test", E, H, I)
