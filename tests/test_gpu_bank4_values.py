"""The values of the layer on a bank in 4 bits, form by form, in the 2-norm
(bank4_values has the tolerance and its derivation), and where they are largest."""
from __future__ import annotations

import pytest
import torch

from bank4_values import LIMIT, distance, layer
from moe_amd import experts_forward, few, ops
from moe_amd.layer import moe_layer
from pack4_oracle import tiles

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


class Bank:
    """A packed weight, an expert of which indexing gives in 64 bits."""

    def __init__(self, w):
        self.packed = ops.pack4(w, dtype=BF)

    def __len__(self):
        return self.packed.shape[0]

    def __getitem__(self, e):
        p = self.packed
        return tiles(p.q[e], p.scale[e], p.shape[1:]).to(DEV)


def _banks(g, E, H, I):
    return (Bank(torch.randn(E, 2 * I, H, generator=g, device=DEV) * 0.02),
            Bank(torch.randn(E, H, I, generator=g, device=DEV) * 0.02))


def _inputs(g, T, H, E, K):
    x = torch.randn(T, H, generator=g, device=DEV, dtype=BF)
    idx = torch.rand(T, E, generator=g, device=DEV).argsort(1)[:, :K].contiguous()
    return x, idx, torch.rand(T, K, generator=g, device=DEV) + 0.1


def _small(T, K, I):
    """Whether act of a few tokens is not rounded."""
    return T * K <= 16 and T * K * I <= 12288


FEW = [  # T, H, E, K, I
    (1, 2048, 128, 8, 768), (2, 1024, 16, 8, 768), (1, 8192, 3, 3, 64), (1, 1024, 8, 8, 1600),
    (3, 2048, 128, 8, 768), (13, 1024, 128, 4, 768), (64, 2048, 128, 8, 768),
    (20, 4160, 6, 2, 1600), (64, 256, 8, 8, 64),
]


@pytest.mark.parametrize("T,H,E,K,I", FEW)
def test_few(T, H, E, K, I):
    g = _gen(T + I)
    b1, b2 = _banks(g, E, H, I)
    x, idx, w = _inputs(g, T, H, E, K)
    out = few.experts_forward_few(x, idx, w, b1.packed, b2.packed)
    assert distance(out, layer(x, idx, w, b1, b2, not _small(T, K, I))) < LIMIT


ROUTERS = [
    ("softmax", {}), ("softmax", dict(offset=True)), ("softmax", dict(renormalize=False)),
    ("sigmoid", {}), ("sigmoid", dict(scaling_factor=2.5)),
    ("sigmoid", dict(num_groups=8, group_topk=4, scaling_factor=1.5)),
    ("sigmoid", dict(num_groups=16, group_topk=2, renormalize=False)),
]


def _layer_case(router, kw, T, E, H=512, I=128):
    g = _gen(T + E)
    b1, b2 = _banks(g, E, H, I)
    x, wr = (torch.randn(n, H, generator=g, device=DEV, dtype=BF) * s for n, s in ((T, 1), (E, 0.05)))
    kw, extra = dict(kw, router=router), torch.rand(E, generator=g, device=DEV)
    if kw.pop("offset", False):
        kw["logit_offset"] = extra
    if router == "sigmoid":
        kw["expert_bias"] = extra * 0.1
    return x, wr, b1, b2, kw


@pytest.mark.parametrize("router,kw", ROUTERS)
@pytest.mark.parametrize("T", [1, 2, 7, 64])
@pytest.mark.parametrize("E", [64, 512])
def test_routers_few(router, kw, T, E):
    """Offsets, biases, scaling and groups: the routing is the exact bank's, bit for
    bit, and the experts follow it."""
    K = 8
    x, wr, b1, b2, kw = _layer_case(router, kw, T, E)
    out, w, idx = few.moe_layer_few(x, wr, b1.packed, b2.packed, K, return_routing=True, **kw)
    _, w0, idx0 = few.moe_layer_few(x, wr, ops.unpack4(b1.packed), ops.unpack4(b2.packed), K,
                                    return_routing=True, **kw)
    assert torch.equal(idx, idx0) and torch.equal(w, w0)
    assert distance(out, layer(x, idx, w, b1, b2, not _small(T, K, 128))) < LIMIT


@pytest.mark.parametrize("router,kw", ROUTERS)
def test_routers(router, kw):
    x, wr, b1, b2, kw = _layer_case(router, kw, 150, 64)
    with torch.no_grad():
        out, probs, w, idx = moe_layer(x, wr, b1.packed, b2.packed, 8, **kw)
        _, probs0, w0, idx0 = moe_layer(x, wr, ops.unpack4(b1.packed), ops.unpack4(b2.packed), 8,
                                        **kw)
    assert torch.equal(idx, idx0) and torch.equal(w, w0) and torch.equal(probs, probs0)
    assert distance(out, layer(x, idx, w, b1, b2, True)) < LIMIT


PROMPT = [  # T, H, E, K, I
    (509, 1024, 128, 4, 768), (200, 1024, 3, 1, 832), (1021, 2048, 128, 8, 768),
    (1500, 512, 4, 4, 320), (2050, 576, 16, 8, 256), (70, 128, 1, 1, 64),
]


@pytest.mark.parametrize("T,H,E,K,I", PROMPT)
def test_prompt(T, H, E, K, I):
    g = _gen(T + I)
    b1, b2 = _banks(g, E, H, I)
    x, idx, w = _inputs(g, T, H, E, K)
    out = experts_forward(x, idx, w, b1.packed, b2.packed)
    assert distance(out, layer(x, idx, w, b1, b2, True)) < LIMIT


@pytest.mark.parametrize("ratio", [2.0 ** 4, 2.0 ** 10, 2.0 ** 12, 2.0 ** 20])
@pytest.mark.parametrize("T,E", [(40, 2), (300, 2), (300, 16)])
def test_columns_beside_a_large_one(T, E, ratio):
    """Output columns far larger than their neighbours: the others keep their exactness
    (down to 2^-28 of the largest, fp16 holds 2^-11 of a value)."""
    g = _gen(T)
    H, I, K = 256, 128, 2
    b1, _ = _banks(g, E, H, I)
    w2 = torch.randn(E, H, I, generator=g, device=DEV) * 0.02
    large = torch.tensor([5, 64, 127, 200], device=DEV)
    w2[:, large] *= ratio
    b2 = Bank(w2)
    x, idx, w = _inputs(g, T, H, E, K)
    ref = layer(x, idx, w, b1, b2, True)
    others = torch.ones(H, dtype=torch.bool, device=DEV)
    others[large] = False
    fns = [experts_forward] + [few.experts_forward_few] * (T <= 64)
    for fn in fns:
        out = fn(x, idx, w, b1.packed, b2.packed)
        assert distance(out[:, others], ref[:, others]) < LIMIT
        assert distance(out[:, large], ref[:, large]) < LIMIT


@pytest.mark.parametrize("T", [40, 300])
def test_a_column_that_is_not_finite(T):
    """Weights of one output column so large that its sums are infinite: its
    neighbours are what they are without them."""
    g = _gen(T)
    E, H, I, K = 2, 128, 64, 1
    b1 = Bank(torch.rand(E, 2 * I, H, generator=g, device=DEV) * 0.02)
    w2 = torch.randn(E, H, I, generator=g, device=DEV) * 0.02
    x, idx, w = _inputs(g, T, H, E, K)
    clean = ops.pack4(w2, dtype=BF)
    w2[:, 70] = 2.0 ** 127
    bad = ops.pack4(w2, dtype=BF)
    x = x.abs() * 8    # and all acts above 1
    others = torch.arange(H, device=DEV) != 70
    for fn in [experts_forward] + [few.experts_forward_few] * (T <= 64):
        got, ref = (fn(x, idx, w, b1.packed, b) for b in (bad, clean))
        assert torch.isfinite(ref).all() and torch.isinf(got[:, 70]).all()
        assert torch.equal(got[:, others], ref[:, others])


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


def test_the_most_experts():
    """What the workspace's size allows, the call takes: 10239 experts, and not one more."""
    g = _gen(3)
    E, H, I, T, K = 10239, 64, 64, 600, 2
    b1, b2 = _banks(g, E, H, I)
    x, w = torch.randn(T, H, generator=g, device=DEV, dtype=BF), torch.rand(T, K, device=DEV)
    idx = torch.randint(0, 40, (T, K), generator=g, device=DEV) * 257 % E
    idx[:, 1] = torch.where(idx[:, 1] == idx[:, 0], E - 1, idx[:, 1])
    out = experts_forward(x, idx, w, b1.packed, b2.packed)
    assert distance(out, layer(x, idx, w, b1, b2, True)) < LIMIT
    more = [ops.Packed4(p.q[:1].expand(E + 1, *p.q.shape[1:]), p.scale[:1].expand(E + 1, *p.scale.shape[1:]),
                        (E + 1, *p.shape[1:]), BF) for p in (b1.packed, b2.packed)]
    with pytest.raises(RuntimeError, match="E=10240"):
        experts_forward(x, idx, w, *more)
