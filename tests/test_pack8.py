"""8-bit activations without a GPU: refusals, sizes, and the choice's way to
the experts."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from moe_amd import _lib, experts_forward, hf, library, ops
from moe_amd.layer import SparseMoeBlock, moe_layer


@pytest.mark.parametrize("args,status,text", [
    ((4096, 2, 4, 64, 4096, 4096, None), "MOE_ERR_DTYPE", "neither bf16 nor fp32"),
    ((4096, 1, -1, 64, 4096, 4096, None), "MOE_ERR_ARG", "rows=-1"),
    ((4096, 1, 4, 1 << 31, 4096, 4096, None), "MOE_ERR_UNSUPPORTED", "too large"),
    ((None, 1, 4, 64, 4096, 4096, None), "MOE_ERR_ARG", "null pointer"),
    ((4096, 1, 4, 64, 4096, None, None), "MOE_ERR_ARG", "null pointer"),
    ((4097, 1, 4, 64, 4096, 4096, None), "MOE_ERR_ALIGN", "not aligned"),
    ((4098, 0, 4, 64, 4096, 4096, None), "MOE_ERR_ALIGN", "not aligned"),
])
def test_pack8_refuses(built_lib, args, status, text):
    with pytest.raises(RuntimeError, match=f"{status}.*{text}"):
        _lib.call("moe_amd_pack8", *args)
    x, dtype, rows, cols, q, scale, st = args
    with pytest.raises(RuntimeError, match=f"{status}.*{text}"):
        _lib.call("moe_amd_unpack8", q, scale, rows, cols, x, dtype, st)


def test_nothing_to_pack_is_no_call(built_lib):
    _lib.call("moe_amd_pack8", None, 1, 0, 64, None, None, None)
    _lib.call("moe_amd_unpack8", None, None, 5, 0, None, 0, None)


def test_fused_entry_points_refuse(built_lib):
    gu = [4096, 4096, 2, 4096, 4096, 4096, 4, 8, 4, 128, 64, 1, 4096, 4096, 4096, None]
    for at, value, text in ((11, 0, "bf16 only"), (9, 100, "multiples of 64"), (12, None, "null"),
                            (13, None, "null"), (12, 4104, "not 16-byte aligned"),
                            (7, 9, "T\\*top_k")):
        bad = list(gu)
        bad[at] = value
        with pytest.raises(RuntimeError, match=f"gemm_gate_up_swiglu_pack8.*{text}"):
            _lib.call("moe_amd_gemm_gate_up_swiglu_pack8", *bad)
    down = [4096, 4096, 2, 4096, 4096, 4096, 4096, 4096, 4096, 0, 4, 8, 4, 128, 64, 1, 4096, 4096,
            4096, None]
    for at, value, text in ((15, 0, "bf16 only"), (14, 32, "multiples of 64"), (6, None, "null"),
                            (7, None, "null"), (7, 4098, "not 16-byte aligned"),
                            (9, 4, "weights_dtype")):
        bad = list(down)
        bad[at] = value
        with pytest.raises(RuntimeError, match=f"gemm_down_backward_dx_fused_pack8.*{text}"):
            _lib.call("moe_amd_gemm_down_backward_dx_fused_pack8", *bad)


def test_python_refusals():
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.pack8(torch.zeros(4, 64))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.unpack8(ops.Packed8(torch.zeros(4, 64, dtype=torch.int8),
                                torch.zeros(4, 1, dtype=torch.uint8), torch.float32))
    x, idx, w = torch.zeros(4, 64), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    w1, w2 = torch.zeros(3, 128, 64), torch.zeros(3, 64, 64)
    with pytest.raises(ValueError, match="saved_activations 'int4'"):
        experts_forward(x, idx, w, w1, w2, saved_activations="int4")
    with pytest.raises(NotImplementedError, match="bf16 layers"):
        experts_forward(x, idx, w, w1, w2, saved_activations="int8")
    with pytest.raises(NotImplementedError, match="bf16 layers"):
        moe_layer(x, torch.zeros(3, 64), w1, w2, 2, saved_activations="int8_all")
    with pytest.raises(ValueError, match="saved_activations"):
        hf.install(SimpleNamespace(), saved_activations="fp8")


def test_packed_bytes():
    # 65 bytes for 64 values where bf16 has 128
    assert ops.packed_gate_up_bytes(10, 64) == 10 * 2 * 64 * 65 // 64
    assert ops.packed_gate_up_bytes(0, 768) == 0


def test_the_choice_reaches_the_experts(monkeypatch):
    from moe_amd import experts
    seen = []
    monkeypatch.setattr(experts, "experts_forward", lambda *a: seen.append(a[5]) or a[0])
    block = SparseMoeBlock(64, 4, 2, 64)
    bank = block.experts
    args = (torch.zeros(3, 64), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2))
    experts.mi355x_experts_forward(bank, *args)
    bank.saved_activations = "int8"
    experts.mi355x_experts_forward(bank, *args)
    assert seen == ["exact", "int8"] and library.KEEPS == ("exact", "int8", "int8_all")
    assert block.saved_activations == "exact"


@pytest.mark.parametrize("keep", ["int8", "int8_all"])
def test_fp32_modules_that_keep_nothing_run(keep):
    """Only what a backward will read is packed, so a call that wants no gradient
    takes any dtype; one that wants one refuses fp32."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from moe_amd.experts import mi355x_experts_forward

    with FakeTensorMode():
        block = SparseMoeBlock(128, 8, 2, 64)
        block.saved_activations = block.experts.saved_activations = keep
        x = torch.empty(100, 128)
        routing = torch.empty(100, 2, dtype=torch.int64), torch.empty(100, 2)

        def run():
            assert block(x).shape == x.shape
            assert mi355x_experts_forward(block.experts, x, *routing).shape == x.shape

        with torch.no_grad():
            run()
        block.requires_grad_(False)
        run()
        for part in (block.gate, block.experts):     # the routing weights' gradient too
            part.requires_grad_(True)
            with pytest.raises(NotImplementedError, match="bf16 layers"):
                block(x)
            part.requires_grad_(False)
        with pytest.raises(NotImplementedError, match="bf16 layers"):
            mi355x_experts_forward(block.experts, x.requires_grad_(True), *routing)
        block.saved_activations = block.experts.saved_activations = "int4"
        with torch.no_grad(), pytest.raises(ValueError, match="int4"):
            block(x)
        with torch.no_grad(), pytest.raises(ValueError, match="int4"):
            mi355x_experts_forward(block.experts, x, *routing)
