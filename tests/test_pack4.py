"""Weights and banks in 4 bits without a GPU: refusals, sizes, and the layer's
choice of form."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from moe_amd import _lib, experts_forward, few, hf, ops
from moe_amd.experts import bank_weights, mi355x_experts_forward, pack_bank
from moe_amd.layer import SparseMoeBlock, moe_layer

BF = torch.bfloat16
A = 4096  # an aligned address that no refused call reads


@pytest.mark.parametrize("args,status,text", [
    ((A, 2, 1, 4, 64, A, A, None), "MOE_ERR_DTYPE", "neither bf16 nor fp32"),
    ((A, 1, -1, 4, 64, A, A, None), "MOE_ERR_ARG", "batch=-1"),
    ((A, 1, 1, -4, 64, A, A, None), "MOE_ERR_ARG", "n=-4"),
    ((A, 1, 1, 4, 1 << 31, A, A, None), "MOE_ERR_UNSUPPORTED", "too large"),
    ((A, 1, 1 << 30, 1 << 20, 1 << 20, A, A, None), "MOE_ERR_UNSUPPORTED", "too large"),
    ((None, 1, 1, 4, 64, A, A, None), "MOE_ERR_ARG", "null pointer"),
    ((A, 1, 1, 4, 64, None, A, None), "MOE_ERR_ARG", "null pointer"),
    ((A, 1, 1, 4, 64, A, None, None), "MOE_ERR_ARG", "null pointer"),
    ((A + 1, 1, 1, 4, 64, A, A, None), "MOE_ERR_ALIGN", "not aligned"),
    ((A + 2, 0, 1, 4, 64, A, A, None), "MOE_ERR_ALIGN", "not aligned"),
    ((A, 1, 1, 4, 64, A + 2, A, None), "MOE_ERR_ALIGN", "not aligned|not to 4"),
])
def test_pack4_refuses(built_lib, args, status, text):
    with pytest.raises(RuntimeError, match=f"{status}.*({text})"):
        _lib.call("moe_amd_pack4", *args)
    x, dtype, batch, n, k, q, scale, st = args
    with pytest.raises(RuntimeError, match=f"{status}.*({text})"):
        _lib.call("moe_amd_unpack4", q, scale, batch, n, k, x, dtype, st)


def test_nothing_to_do_is_no_call(built_lib):
    _lib.call("moe_amd_pack4", None, 1, 0, 4, 64, None, None, None)
    _lib.call("moe_amd_unpack4", None, None, 3, 4, 0, None, 0, None)
    _lib.call("moe_amd_gemm_gate_up_swiglu4", None, None, 2, A, A, A, A, 0, 0, 4, 64, 64, None, None)
    _lib.call("moe_amd_gemm_down4", None, A, A, A, A, 0, 4, 64, 64, None, None, None)
    _lib.call("moe_amd_combine16", None, None, None, None, None, 0, 0, 2, 4, 64, None, None)
    _lib.call("moe_amd_experts_few4", None, None, None, 0, None, None, None, None, 0, 2, 4, 64, 64,
              None, 0, None, None)
    _lib.call("moe_amd_experts4", None, None, None, 0, None, None, None, None, 0, 2, 4, 64, 64, None,
              0, None, None)


@pytest.mark.parametrize("at,value,status,text", [
    (0, None, "MOE_ERR_ARG", "null"), (0, A + 8, "MOE_ERR_ALIGN", "not 16-byte aligned"),
    (1, None, "MOE_ERR_ARG", "null"), (2, 3, "MOE_ERR_ARG", r"T\*top_k"),
    (4, None, "MOE_ERR_ARG", "null"), (5, None, "MOE_ERR_ARG", "null"),
    (5, A + 4, "MOE_ERR_ALIGN", "not 16-byte"), (6, None, "MOE_ERR_ARG", "null"),
    (6, A + 8, "MOE_ERR_ALIGN", "not 16-byte"), (8, -8, "MOE_ERR_ARG", "bad sizes"),
    (9, 0, "MOE_ERR_ARG", "bad sizes"), (10, 96, "MOE_ERR_ARG", "multiples of 64"),
    (11, 32, "MOE_ERR_ARG", "multiples of 64"), (12, None, "MOE_ERR_ARG", "null"),
])
def test_gate_up4_refuses(built_lib, at, value, status, text):
    args = [A, A, 2, A, A, A, A, 4, 8, 4, 128, 64, A, None]
    args[at] = value
    with pytest.raises(RuntimeError, match=f"{status}.*gemm_gate_up_swiglu4.*{text}"):
        _lib.call("moe_amd_gemm_gate_up_swiglu4", *args)


def test_gate_up4_limits(built_lib):
    for T, K, E, H, I, text in ((1 << 28, 2, 4, 64, 64, "2\\^29"), (1 << 20, 1, 4, 1024, 64, "T\\*H"),
                                (4, 2, 4, 1 << 16, 1 << 16, "exceed 2 GB"),
                                (4, 2, 4, 64, 1 << 23, "2\\^22"), (1, 2, 4, 1 << 23, 64, "2\\^22")):
        with pytest.raises(RuntimeError, match=f"MOE_ERR_UNSUPPORTED.*{text}"):
            _lib.call("moe_amd_gemm_gate_up_swiglu4", A, A, K, A, A, A, A, T, T * K, E, H, I, A, None)


@pytest.mark.parametrize("at,value,status,text", [
    (0, None, "MOE_ERR_ARG", "null"), (1, None, "MOE_ERR_ARG", "null"),
    (3, None, "MOE_ERR_ARG", "null"), (4, None, "MOE_ERR_ARG", "null"),
    (4, A + 4, "MOE_ERR_ALIGN", "not 16-byte"), (7, 100, "MOE_ERR_ARG", "multiples of 64"),
    (8, 100, "MOE_ERR_ARG", "multiples of 64"), (9, None, "MOE_ERR_ARG", "null"),
    (9, A + 2, "MOE_ERR_ALIGN", "not 16-byte"), (10, None, "MOE_ERR_ARG", "null"),
])
def test_down4_refuses(built_lib, at, value, status, text):
    args = [A, A, A, A, A, 8, 4, 128, 64, A, A, None]
    args[at] = value
    with pytest.raises(RuntimeError, match=f"{status}.*gemm_down4.*{text}"):
        _lib.call("moe_amd_gemm_down4", *args)


@pytest.mark.parametrize("at,value,status,text", [
    (0, None, "MOE_ERR_ARG", "null"), (1, None, "MOE_ERR_ARG", "null"),
    (0, A + 8, "MOE_ERR_ALIGN", "not 16-byte"), (4, None, "MOE_ERR_ARG", "null"),
    (5, 7, "MOE_ERR_DTYPE", "weights dtype"), (6, -1, "MOE_ERR_ARG", "T=-1"),
    (9, 96, "MOE_ERR_ARG", "H=96"), (9, 1 << 23, "MOE_ERR_UNSUPPORTED", r"2\^22"), (10, None, "MOE_ERR_ARG", "null"),
    (10, A + 8, "MOE_ERR_ALIGN", "not 16-byte"),
])
def test_combine16_refuses(built_lib, at, value, status, text):
    args = [A, A, A, A, A, 0, 4, 2, 4, 128, A, None]
    args[at] = value
    with pytest.raises(RuntimeError, match=f"{status}.*combine16.*{text}"):
        _lib.call("moe_amd_combine16", *args)


def _experts4_ws(T=4, E=8, K=2, H=128, I=64):
    return _lib.load().moe_amd_experts4_workspace_size(T, E, K, H, I)


def test_experts4_workspace(built_lib):
    # act, y and the sorted rows' indices at least
    assert _experts4_ws() >= 8 * (64 * 2 + 128 * 2 + 2 + 8)
    assert 0 < _experts4_ws() < _experts4_ws(T=64) < _experts4_ws(T=64, K=16)
    for bad in (dict(T=-1), dict(K=0), dict(E=0), dict(E=16385), dict(H=96), dict(I=32), dict(H=0),
                dict(T=1 << 28), dict(T=1 << 20, H=1024)):
        assert _experts4_ws(**bad) == 0, bad


@pytest.mark.parametrize("at,value,status,text", [
    (0, None, "MOE_ERR_ARG", "null"), (0, A + 8, "MOE_ERR_ALIGN", "not 16-byte"),
    (1, None, "MOE_ERR_ARG", "null"), (2, None, "MOE_ERR_ARG", "null"),
    (3, 7, "MOE_ERR_DTYPE", "weights dtype"), (4, None, "MOE_ERR_ARG", "null"),
    (4, A + 8, "MOE_ERR_ALIGN", "not 16-byte"), (5, A + 4, "MOE_ERR_ALIGN", "not 16-byte"),
    (6, None, "MOE_ERR_ARG", "null"), (6, A + 8, "MOE_ERR_ALIGN", "not 16-byte"),
    (7, A + 4, "MOE_ERR_ALIGN", "not 16-byte"), (8, -1, "MOE_ERR_ARG", "T=-1"),
    (8, 1 << 24, "MOE_ERR_UNSUPPORTED", r"T\*H"), (9, 0, "MOE_ERR_ARG", "K=0"),
    (10, 16385, "MOE_ERR_ARG", "E=16385"), (11, 96, "MOE_ERR_ARG", "multiples of 64"),
    (12, 32, "MOE_ERR_ARG", "multiples of 64"), (13, None, "MOE_ERR_WORKSPACE", "needs"),
    (13, A + 8, "MOE_ERR_ALIGN", "not 16-byte"), (14, 16, "MOE_ERR_WORKSPACE", "needs"),
    (15, None, "MOE_ERR_ARG", "null"), (15, A + 8, "MOE_ERR_ALIGN", "not 16-byte"),
])
def test_experts4_refuses(built_lib, at, value, status, text):
    args = [A, A, A, 0, A, A, A, A, 4, 2, 8, 128, 64, A, 1 << 20, A, None]
    args[at] = value
    with pytest.raises(RuntimeError, match=f"{status}.*experts4.*{text}"):
        _lib.call("moe_amd_experts4", *args)


def _ws(T=4, E=8, K=2, H=128, I=64):
    return _lib.load().moe_amd_few4_workspace_size(T, E, K, H, I)


def test_few4_workspace(built_lib):
    assert 0 < _ws() < _ws(T=64) < _ws(T=64, K=16)
    for bad in (dict(T=65), dict(T=-1), dict(K=17), dict(K=0), dict(E=0), dict(E=4097), dict(H=96),
                dict(I=32), dict(H=0), dict(H=1 << 17)):
        assert _ws(**bad) == 0, bad


@pytest.mark.parametrize("change,status,text", [
    (dict(T=65), "MOE_ERR_UNSUPPORTED", "64 tokens"), (dict(K=17), "MOE_ERR_UNSUPPORTED", "top-16"),
    (dict(E=5000), "MOE_ERR_UNSUPPORTED", "4096 experts"),
    (dict(H=100), "MOE_ERR_ARG", "multiples of 64"), (dict(wdtype=5), "MOE_ERR_DTYPE", "weights dtype"),
    (dict(x=None), "MOE_ERR_ARG", "null pointer"), (dict(s2=None), "MOE_ERR_ARG", "null pointer"),
    (dict(ws=100), "MOE_ERR_WORKSPACE", "needs"), (dict(x=A + 8), "MOE_ERR_ALIGN", "16-byte aligned"),
    (dict(s2=A + 4), "MOE_ERR_ALIGN", "16-byte aligned"),
])
def test_experts_few4_refuses(built_lib, change, status, text):
    a = dict(T=4, E=8, K=2, H=128, I=64, wdtype=0, x=A, s2=A, ws=1 << 30)
    a.update(change)
    with pytest.raises(RuntimeError, match=f"{status}.*{text}"):
        _lib.call("moe_amd_experts_few4", a["x"], A, A, a["wdtype"], A, A, A, a["s2"], a["T"], a["K"],
                  a["E"], a["H"], a["I"], A, a["ws"], A, None)


@pytest.mark.parametrize("change,status,text", [
    (dict(router=2), "MOE_ERR_ARG", "router 2"), (dict(K=9), "MOE_ERR_ARG", "K=9"),
    (dict(groups=3), "MOE_ERR_ARG", "bad grouping"), (dict(ws=None), "MOE_ERR_WORKSPACE", "workspace"),
    (dict(wr=None), "MOE_ERR_ARG", "null pointer"), (dict(q1=None), "MOE_ERR_ARG", "null pointer"),
])
def test_moe_layer_few4_refuses(built_lib, change, status, text):
    a = dict(T=4, E=8, K=4, H=128, I=64, router=1, groups=0, gtopk=0, ws=A, wr=A, q1=A)
    a.update(change)
    with pytest.raises(RuntimeError, match=f"{status}.*{text}"):
        _lib.call("moe_amd_moe_layer_few4", A, a["wr"], a["q1"], A, A, A, a["T"], a["K"], a["E"],
                  a["H"], a["I"], a["router"], None, 1, 0.0, a["groups"], a["gtopk"], a["ws"],
                  1 << 30, None, None, A, None)


def _packed(E, N, K, dtype=BF):
    q = torch.zeros(E, -(-N // 16), -(-K // 128), 1024, dtype=torch.uint8)
    return ops.Packed4(q, torch.zeros(*q.shape[:3], 64, dtype=torch.uint8), (E, N, K), dtype)


def test_python_refusals():
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.pack4(torch.zeros(16, 128))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.unpack4(_packed(2, 16, 128))
    x, idx, w = torch.zeros(4, 64, dtype=BF), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    b1, b2 = _packed(3, 128, 64), _packed(3, 64, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        experts_forward(x, idx, w, b1, b2)
    for fn in (experts_forward, few.experts_forward_few):
        with pytest.raises(TypeError, match="both be in 4 bits"):
            fn(x, idx, w, b1, torch.zeros(3, 64, 64, dtype=BF))
        with pytest.raises(TypeError, match="both be in 4 bits"):
            fn(x, idx, w, torch.zeros(3, 128, 64, dtype=BF), b2)
        with pytest.raises(ValueError, match="shape mismatch"):
            fn(x, idx, w, b1, _packed(3, 64, 128))
        with pytest.raises(ValueError, match="shape mismatch"):
            fn(torch.zeros(4, 128, dtype=BF), idx, w, b1, b2)
        with pytest.raises(ValueError, match="multiples of 64"):
            fn(torch.zeros(4, 32, dtype=BF), idx, w, _packed(3, 128, 32), _packed(3, 32, 64))
        with pytest.raises(NotImplementedError, match="bf16 layers"):
            fn(x, idx, w, _packed(3, 128, 64, torch.float32), _packed(3, 64, 64, torch.float32))
        broken = ops.Packed4(b1.q, b1.scale[:, :1], b1.shape, BF)
        with pytest.raises(ValueError, match="not a packed"):
            fn(x, idx, w, broken, b2)
        with pytest.raises(RuntimeError, match="forward only"):
            fn(x.clone().requires_grad_(), idx, w, b1, b2)
        with pytest.raises(RuntimeError, match="forward only"):
            fn(x, idx, w.clone().requires_grad_(), b1, b2)
    with pytest.raises(ValueError, match="both be .T, K."):
        experts_forward(x, idx, w[:, :1], b1, b2)
    with pytest.raises(ValueError, match="saved_activations"):
        experts_forward(x, idx, w, b1, b2, saved_activations="int4")
    wr = torch.zeros(3, 64, dtype=BF, requires_grad=True)
    with pytest.raises(RuntimeError, match="forward only"):
        moe_layer(x, wr, b1, b2, 2)
    with pytest.raises(RuntimeError, match="forward only"):
        few.moe_layer_few(x, wr, b1, b2, 2)
    with pytest.raises(TypeError, match="both be in 4 bits"):
        moe_layer(x, wr, b1, torch.zeros(3, 64, 64, dtype=BF), 2)
    with pytest.raises(NotImplementedError, match="bf16 layers"):
        pack_bank(SparseMoeBlock(64, 3, 2, 64).experts)
    with pytest.raises(ValueError, match="multiples of 64"):
        pack_bank(SparseMoeBlock(96, 3, 2, 64).bfloat16().experts)
    bank = SparseMoeBlock(64, 3, 2, 64).bfloat16().experts
    bank.is_transposed = True   # no call would take it
    with pytest.raises(NotImplementedError, match="transposed"):
        pack_bank(bank)
    assert bank.gate_up_proj.dtype == BF


def _pack_on_cpu(monkeypatch):
    monkeypatch.setattr(ops, "pack4", lambda w: _packed(*w.shape))


def test_the_packed_bank_reaches_the_kernels(monkeypatch):
    """After pack_experts, with and without a few tokens."""
    from moe_amd import experts, layer
    _pack_on_cpu(monkeypatch)
    block = SparseMoeBlock(64, 4, 2, 64).bfloat16().pack_experts()
    bank = block.experts
    w1, w2 = bank_weights(bank)
    assert w1.shape == (4, 128, 64) and w2.shape == (4, 64, 64) and w1.q is bank.gate_up_proj_q
    assert hf.expert_banks(block) == [bank] and hf.pack_experts(block) == 0
    assert pack_bank(bank) is bank
    seen = []
    monkeypatch.setattr(few, "experts_forward_few", lambda *a: seen.append(("few", a[3:])) or a[0])
    monkeypatch.setattr(experts, "experts_forward", lambda *a: seen.append(("all", a[3:])) or a[0])
    args = (torch.zeros(3, 64, dtype=BF), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2))
    mi355x_experts_forward(bank, *args)
    bank.few_tokens = 8
    mi355x_experts_forward(bank, *args)
    assert [k for k, _ in seen] == ["all", "few"]
    assert all(isinstance(w, ops.Packed4) for _, a in seen for w in a[:2])
    calls = []
    monkeypatch.setattr(layer, "moe_layer", lambda *a, **k: calls.append(a) or (a[0],) * 4)
    with torch.no_grad():
        block(args[0])
    assert isinstance(calls[0][2], ops.Packed4)


def test_fake_tensors():
    with FakeTensorMode(), torch.no_grad():
        x, idx, w = torch.empty(5, 64, dtype=BF), torch.empty(5, 2, dtype=torch.int64), torch.empty(5, 2)
        b1, b2 = _packed(3, 128, 64), _packed(3, 64, 64)
        assert experts_forward(x, idx, w, b1, b2).shape == x.shape
        assert few.experts_forward_few(x, idx, w, b1, b2).shape == x.shape
        wr = torch.empty(3, 64, dtype=BF)
        out, fw, fi = few.moe_layer_few(x, wr, b1, b2, 2, return_routing=True)
        assert out.shape == x.shape and fw.shape == fi.shape == (5, 2)
        q, s = torch.ops.moe_amd.pack4(torch.empty(2, 17, 130))
        assert q.shape == (2, 2, 2, 1024) and s.shape == (2, 2, 2, 64)
        assert torch.ops.moe_amd.unpack4(q, s, 17, 130, BF).shape == (2, 17, 130)
