"""The few-token layer without a GPU: refusals of its C entry points and of
the Python functions, the workspace size, and the form a block chooses."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from moe_amd import _lib, few, hf, ops
from moe_amd.layer import SparseMoeBlock


def _ws(T=4, E=8, K=2, H=128, I=64, dtype=1):
    return _lib.load().moe_amd_few_workspace_size(T, E, K, H, I, dtype)


def test_workspace_size_and_refused_shapes(built_lib):
    assert _ws() > 0
    assert _ws(T=64, K=16) > _ws(T=1, K=16)
    assert _ws(dtype=0) > _ws(dtype=1)
    for bad in (dict(T=65), dict(T=-1), dict(K=17), dict(K=0), dict(E=0), dict(E=4097),
                dict(H=96), dict(I=32), dict(H=0), dict(dtype=2), dict(H=1 << 17)):
        assert _ws(**bad) == 0, bad


@pytest.mark.parametrize("change,status,text", [
    (dict(T=65), "MOE_ERR_UNSUPPORTED", "64 tokens"),
    (dict(K=17), "MOE_ERR_UNSUPPORTED", "top-16"),
    (dict(E=5000), "MOE_ERR_UNSUPPORTED", "4096 experts"),
    (dict(H=100), "MOE_ERR_ARG", "multiples of 64"),
    (dict(dtype=3), "MOE_ERR_DTYPE", "neither bf16 nor fp32"),
    (dict(wdtype=5), "MOE_ERR_DTYPE", "weights dtype"),
    (dict(x=None), "MOE_ERR_ARG", "null pointer"),
    (dict(ws_bytes=100), "MOE_ERR_WORKSPACE", "needs"),
    (dict(x=8), "MOE_ERR_ALIGN", "16-byte aligned"),
])
def test_experts_few_refuses(built_lib, change, status, text):
    a = dict(T=4, E=8, K=2, H=128, I=64, dtype=1, wdtype=0, x=4096, ws_bytes=1 << 30)
    a.update(change)
    with pytest.raises(RuntimeError, match=f"{status}.*{text}"):
        _lib.call("moe_amd_experts_few", a["x"], 4096, 4096, a["wdtype"], 4096, 4096, a["T"],
                  a["K"], a["E"], a["H"], a["I"], a["dtype"], 4096, a["ws_bytes"], 4096, None)


@pytest.mark.parametrize("change,status,text", [
    (dict(router=2), "MOE_ERR_ARG", "router 2"),
    (dict(K=9), "MOE_ERR_ARG", "K=9"),
    (dict(groups=3), "MOE_ERR_ARG", "bad grouping"),
    (dict(router=0, groups=2), "MOE_ERR_ARG", "bad grouping"),
    (dict(groups=4, gtopk=1), "MOE_ERR_ARG", "bad grouping"),
    (dict(ws=None), "MOE_ERR_WORKSPACE", "workspace"),
])
def test_moe_layer_few_refuses(built_lib, change, status, text):
    a = dict(T=4, E=8, K=4, H=128, I=64, router=1, groups=0, gtopk=0, ws=4096)
    a.update(change)
    with pytest.raises(RuntimeError, match=f"{status}.*{text}"):
        _lib.call("moe_amd_moe_layer_few", 4096, 4096, 4096, 4096, a["T"], a["K"], a["E"], a["H"],
                  a["I"], 1, a["router"], None, 1, 0.0, a["groups"], a["gtopk"], a["ws"], 1 << 30,
                  None, None, 4096, None)


def test_no_tokens_is_no_call(built_lib):
    # nothing is read or launched: the pointers may be null
    _lib.call("moe_amd_experts_few", None, None, None, 0, None, None, 0, 2, 8, 128, 64, 1, None, 0,
              None, None)


def _inputs(T=4, E=8, K=2, H=128, I=64):
    return (torch.zeros(T, H), torch.zeros(T, K, dtype=torch.int64), torch.zeros(T, K),
            torch.zeros(E, 2 * I, H), torch.zeros(E, H, I))


def test_cpu_tensors_and_gradients_are_refused():
    x, idx, w, w1, w2 = _inputs()
    with pytest.raises(RuntimeError, match="GPU only"):
        few.experts_forward_few(x, idx, w, w1, w2)
    with pytest.raises(RuntimeError, match="GPU only"):
        few.moe_layer_few(x, torch.zeros(8, 128), w1, w2, 2)
    w1.requires_grad_(True)
    with pytest.raises(RuntimeError, match="forward only"):
        few.experts_forward_few(x, idx, w, w1, w2)
    with pytest.raises(RuntimeError, match="forward only"):
        few.moe_layer_few(x, torch.zeros(8, 128), w1, w2, 2)


def test_a_block_takes_the_few_token_form_only_without_gradients():
    x = torch.zeros(4, 8)
    p = torch.nn.Parameter(torch.zeros(3))

    def wanted(n, t=x, k=2, e=8):
        return few.wanted(n, k, e, t, p)

    with torch.no_grad():
        assert wanted(4) and wanted(1000) and wanted(4, k=16, e=4096)
        assert not wanted(0) and not wanted(3)
        assert not wanted(64, torch.zeros(0, 8)) and not wanted(1000, torch.zeros(65, 8))
        assert not wanted(4, k=17) and not wanted(4, e=4097)   # the other form's
    assert not wanted(4)
    assert few.wanted(4, 2, 8, x, p.detach())


def test_install_sets_the_banks(monkeypatch):
    block = SparseMoeBlock(64, 4, 2, 64)
    assert hf.expert_banks(block) == [block.experts]
    assert few.MAX_TOKENS == ops.FEW_MAX_TOKENS == 64


def test_a_block_of_mixed_dtypes_keeps_the_other_form(monkeypatch):
    """The sigmoid router takes a router weight of another dtype than the
    experts', the few-token layer does not."""
    from moe_amd import layer

    took = []
    monkeypatch.setattr(few, "moe_layer_few",
                        lambda x, *a, **k: took.append("few") or (x, None, None))
    monkeypatch.setattr(layer, "moe_layer",
                        lambda x, *a, **k: took.append("layer") or (x, None, None, None))
    block = SparseMoeBlock(64, 4, 2, 64, router="sigmoid").to(torch.bfloat16)
    block.few_tokens = 4
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with torch.no_grad():
        block(x)
        block(x.float())
        block.gate.float()
        block(x)
        block(x.float())
    assert took == ["few", "layer", "layer", "layer"]


def test_tensors_of_two_devices_are_refused():
    bf = torch.bfloat16
    with FakeTensorMode():
        def make(shape, dtype=bf, dev="cuda:0"):
            return torch.empty(shape, dtype=dtype, device=dev)

        good = dict(x=((4, 128), bf), idx=((4, 2), torch.int64), w=((4, 2), torch.float32),
                    w1=((8, 128, 128), bf), w2=((8, 128, 64), bf))
        for other in good:
            t = {n: make(*s, dev="cuda:1" if n == other else "cuda:0") for n, s in good.items()}
            with pytest.raises(ValueError, match="one device"):
                ops.experts_few.__wrapped__(t["x"], t["idx"], t["w"], t["w1"], t["w2"])
        good = dict(x=((4, 128), bf), wr=((8, 128), bf), w1=((8, 128, 128), bf),
                    w2=((8, 128, 64), bf), off=((8,), torch.float32))
        for other in good:
            t = {n: make(*s, dev="cuda:1" if n == other else "cuda:0") for n, s in good.items()}
            with pytest.raises(ValueError, match="one device"):
                ops.moe_layer_few.__wrapped__(t["x"], t["wr"], t["w1"], t["w2"], 2,
                                              logit_offset=t["off"])


@pytest.mark.parametrize("few_tokens,grad", [(0, False), (0, True), (8, True)])
def test_a_number_of_tokens_that_depends_on_data(few_tokens, grad):
    """Without the few-token form, and where a gradient is wanted, the layers
    trace whatever the number of tokens turns out to be."""
    from torch.fx.experimental.symbolic_shapes import ShapeEnv

    from moe_amd.experts import mi355x_experts_forward

    env = ShapeEnv()
    with FakeTensorMode(shape_env=env):
        block = SparseMoeBlock(128, 8, 2, 64).requires_grad_(grad)
        block.few_tokens = block.experts.few_tokens = few_tokens
        n = env.create_unbacked_symint()
        x = torch.empty(n, 128)
        assert block(x).shape == (n, 128)
        out = mi355x_experts_forward(block.experts, x, torch.empty(n, 2, dtype=torch.int64),
                                     torch.empty(n, 2))
        assert out.shape == (n, 128)


@pytest.mark.parametrize("H,I", [(1 << 17, 64), (64, 1 << 17), ((1 << 16) + 64, 64)])
def test_a_layer_of_more_features_keeps_the_other_form(H, I):
    # the few-token entry points refuse its shape
    assert _ws(H=H, I=I) == 0 and _ws(H=1 << 16, I=1 << 16) > 0
    with FakeTensorMode(), torch.no_grad():
        block = SparseMoeBlock(H, 4, 2, I)
        p = (block.gate.weight, block.experts.gate_up_proj, block.experts.down_proj)
        x = torch.empty(2, H)
        assert not few.wanted(8, 2, 4, x, *p)
        assert not few.wanted(8, 2, 4, x, torch.empty(2, 2), *p[1:])
        small = SparseMoeBlock(1 << 16, 4, 2, 1 << 16)
        p = (small.gate.weight, small.experts.gate_up_proj, small.experts.down_proj)
        assert few.wanted(8, 2, 4, torch.empty(2, 1 << 16), *p)


def _blocks():
    return [SparseMoeBlock(128, 8, 2, 64, router=r).requires_grad_(False)
            for r in ("softmax", "sigmoid")]


@pytest.mark.parametrize("few_tokens", [0, 8])
def test_fake_tensors_pass_through_either_form(few_tokens):
    from moe_amd.experts import mi355x_experts_forward

    with FakeTensorMode():
        for block in _blocks():
            block.few_tokens = block.experts.few_tokens = few_tokens
            x = torch.empty(4, 128)
            assert block(x).shape == (4, 128) and block.topk_index.shape == (4, 2)
            assert (block.router_logits is None) == bool(few_tokens)
            idx, w = torch.empty(4, 2, dtype=torch.int64), torch.empty(4, 2)
            assert mi355x_experts_forward(block.experts, x, idx, w).shape == (4, 128)
    # fake tensors outside their mode
    assert few.experts_forward_few(x, idx, w, block.experts.gate_up_proj,
                                   block.experts.down_proj).shape == (4, 128)


def _traced(pre_dispatch, mode):
    from torch.fx.experimental.proxy_tensor import make_fx

    def fn(x, idx, w, wr, w1, w2):
        return few.experts_forward_few(few.moe_layer_few(x, wr, w1, w2, 2), idx, w, w1, w2)

    x, idx, w, w1, w2 = _inputs()
    gm = make_fx(fn, tracing_mode=mode, pre_dispatch=pre_dispatch)(
        x, idx, w, torch.zeros(8, 128), w1, w2)
    return {str(n.target).removesuffix(".default") for n in gm.graph.nodes
            if n.op == "call_function"}


@pytest.mark.parametrize("pre_dispatch", [False, True])
def test_a_trace_holds_the_ops(pre_dispatch):
    with torch.no_grad():
        assert {"moe_amd.experts_few", "moe_amd.moe_layer_few"} <= _traced(pre_dispatch, "fake")


def test_modes_tracers_and_transforms_see_the_ops():
    """Under each of them the call is the moe_amd:: op's, not the kernels' own."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, fn, types, args=(), kwargs=None):
            seen.append(str(fn))
            return torch.empty(4, 128) if "moe_amd" in str(fn) else fn(*args, **(kwargs or {}))

    x, idx, w, w1, w2 = _inputs()
    seen = []
    with torch.no_grad(), Mode():
        few.experts_forward_few(x, idx, w, w1, w2)
    assert seen == ["moe_amd.experts_few.default"]

    unseen = []

    def probe(t):
        unseen.append(few._unseen(t))
        return t + 1

    probe(x)
    with torch.inference_mode():
        probe(x)
    with torch.no_grad():
        probe(torch.nn.Parameter(x))
    assert unseen == [True, True, True] and few._unseen(x, None)
    unseen.clear()
    torch.func.vmap(probe)(x)
    torch.func.functionalize(probe)(x)
    torch.jit.trace(probe, x, check_trace=False)
    assert unseen == [False, False, False]
    # a tensor whose values the dispatcher would negate first
    assert not few._unseen(x._neg_view())


def test_install_sets_and_resets_the_banks():
    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.blocks = torch.nn.ModuleList(SparseMoeBlock(64, 4, 2, 64) for _ in range(2))
            self.other = torch.nn.Linear(4, 4)
            self.chosen = []

        def set_experts_implementation(self, name):
            self.chosen.append(name)

    def options():
        return {(b.few_tokens, b.saved_activations) for b in hf.expert_banks(model)}

    model = Model()
    banks = hf.expert_banks(model)
    assert banks == [b.experts for b in model.blocks]
    assert hf.install(model, few_tokens=16, saved_activations="int8") is model
    assert options() == {(16, "int8")} and not hasattr(model.other, "few_tokens")
    hf.install(model, few_tokens=8, saved_activations="int8_all", experts=False)   # experts' options
    assert options() == {(16, "int8")} and model.chosen == [hf.EXPERTS_KEY]
    hf.install(model)
    assert options() == {(0, "exact")} and model.chosen == [hf.EXPERTS_KEY] * 2
    with pytest.raises(ValueError, match="saved_activations"):
        hf.install(model, few_tokens=4, saved_activations="int4")
    assert options() == {(0, "exact")}
