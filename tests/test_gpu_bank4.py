"""The expert layer on banks in 4 bits against the formulas in 64 bits.

Tolerances.  The weights that a bank holds are exact bf16 values, so only the
layer rounds.  Let u = 2^-8, half a step of bf16 relative to a value, and v =
2^-24.  A sum of n fp32 products is off by at most n v sum|a b|, so gate and up are
off by dg = H v |W1| |x|; with |silu'| < 1.1 and |silu(g)| <= |g|, act before its
rounding by da = 1.1 dg |up| + |gate| du + dg du + 16 v |act| (the last term: the
hardware's exp2 and reciprocal, 1 ulp each, exp2's argument rounded once, which
its size |g| log2 e multiplies, where sigmoid's own slope is below 1/|g|; and the
products), and by u (|act| + da) more after it.  y is off by dy = |W2| da' + I v
|W2| (|act| + da'); grouped products hold it in 16-bit blocks of 64 columns, off by
2^-15 (max|y| + dy) of the block at most.  out is off by the weighted sum of that,
(K + 1) v |w y| more and its own rounding.  The bounds below are these sums,
evaluated in 64 bits.
"""
from __future__ import annotations

import pytest
import torch

from moe_amd import experts_forward, few, hf, library, ops  # noqa: F401
from moe_amd.layer import SparseMoeBlock, moe_layer
from pack4_oracle import tiles

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
U, V = 2.0 ** -8, 2.0 ** -24


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _bank(g, E, H, I):
    w1 = torch.randn(E, 2 * I, H, generator=g, device=DEV) * 0.02
    w2 = torch.randn(E, H, I, generator=g, device=DEV) * 0.02
    return ops.pack4(w1, dtype=BF), ops.pack4(w2, dtype=BF)


def _routing(g, T, E, K, skew=0.0):
    logits = torch.rand(T, E, generator=g, device=DEV)
    logits += skew * torch.linspace(1, 0, E, device=DEV) ** 4
    idx = logits.argsort(1, descending=True)[:, :K].contiguous()
    return idx, torch.rand(T, K, generator=g, device=DEV) + 0.1


def _oracle(x, idx, w, b1, b2, blocks=False):
    """(out, bound) in 64 bits, expert by expert; blocks: y in 16-bit blocks."""
    T, H = x.shape
    E, I, K = b1.shape[0], b2.shape[2], idx.shape[1]
    out = torch.zeros(T, H, device=DEV, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for e in torch.unique(idx).tolist():
        if not 0 <= e < E:
            continue
        t, k = torch.nonzero(idx == e, as_tuple=True)
        m1 = tiles(b1.q[e], b1.scale[e], b1.shape[1:]).to(DEV)
        m2 = tiles(b2.q[e], b2.scale[e], b2.shape[1:]).to(DEV)
        xt, wk = x[t].double(), w[t, k].double()[:, None]
        gu, dgu = xt @ m1.t(), H * V * (xt.abs() @ m1.abs().t())
        gt, up, dg, du = gu[:, :I], gu[:, I:], dgu[:, :I], dgu[:, I:]
        act = gt * torch.sigmoid(gt) * up
        da = 1.1 * dg * up.abs() + gt.abs() * du + dg * du + 16 * V * act.abs()
        da = da + U * (act.abs() + da)
        y = act @ m2.t()
        dy = da @ m2.abs().t() + I * V * ((act.abs() + da) @ m2.abs().t())
        if blocks:
            most = (y.abs() + dy).unflatten(1, (-1, 64)).amax(-1, keepdim=True)
            dy = dy + (most * 2.0 ** -15).expand(-1, -1, 64).flatten(1)
        out.index_add_(0, t, y * wk)
        tol.index_add_(0, t, wk.abs() * (dy + (K + 1) * V * y.abs()))
    return out, tol + U * (out.abs() + tol)


def _close(got, ref, tol):
    assert torch.isfinite(got).all()
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst by " \
        f"{float(((got.double() - ref).abs() / tol.clamp(min=1e-300)).max()):.2f} bounds"


def _x(g, T, H):
    return torch.randn(T, H, generator=g, device=DEV, dtype=BF)


FEW = [  # T, H, E, K, I
    (1, 64, 4, 2, 64), (1, 2048, 128, 8, 768), (2, 192, 16, 4, 192), (3, 128, 1, 1, 64),
    (5, 320, 7, 3, 448), (13, 1024, 128, 4, 768), (17, 64, 300, 16, 128), (37, 704, 40, 8, 576),
    (20, 4160, 6, 2, 1600), (1, 2112, 4, 2, 6208), (2, 64, 8, 8, 768), (1, 8256, 3, 3, 64),
    (64, 256, 8, 8, 64), (64, 1088, 512, 6, 320), (64, 2048, 128, 8, 768), (33, 128, 3, 2, 832),
]


@pytest.mark.parametrize("T,H,E,K,I", FEW)
def test_experts_few(T, H, E, K, I):
    g = _gen(T + H)
    b1, b2 = _bank(g, E, H, I)
    x, (idx, w) = _x(g, T, H), _routing(g, T, E, K)
    out = few.experts_forward_few(x, idx, w, b1, b2)
    _close(out, *_oracle(x, idx, w, b1, b2))
    assert torch.equal(out, few.experts_forward_few(x, idx, w, b1, b2))


@pytest.mark.parametrize("T,K", [(1, 4), (16, 4), (40, 8)])
def test_experts_few_padding_and_repeats(T, K):
    """Ids outside [0, E), tokens without any expert, one expert named twice and by
    everybody, bf16 weights."""
    g = _gen(7)
    E, H, I = 6, 192, 128
    b1, b2 = _bank(g, E, H, I)
    x = _x(g, T, H)
    idx = torch.randint(-1, E + 2, (T, K), generator=g, device=DEV)
    idx[-1] = E
    idx[0, :2] = 3
    w = (torch.rand(T, K, generator=g, device=DEV) - 0.5).to(BF)
    _close(few.experts_forward_few(x, idx, w, b1, b2), *_oracle(x, idx, w, b1, b2))
    _close(experts_forward(x, idx, w, b1, b2), *_oracle(x, idx, w, b1, b2, blocks=True))
    none = torch.full_like(idx, E)
    assert (few.experts_forward_few(x, none, w, b1, b2) == 0).all()
    assert (experts_forward(x, none, w, b1, b2) == 0).all()
    same = torch.full_like(idx, 5)
    _close(few.experts_forward_few(x, same, w, b1, b2), *_oracle(x, same, w, b1, b2))


@pytest.mark.parametrize("router", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,H,E,K,I", [(1, 256, 128, 8, 128), (2, 128, 64, 4, 192),
                                       (9, 192, 300, 6, 64), (64, 512, 32, 8, 320)])
def test_moe_layer_few(router, T, H, E, K, I):
    """The routing is that of the layer on an exact bank, bit for bit."""
    g = _gen(E)
    b1, b2 = _bank(g, E, H, I)
    x, wr = _x(g, T, H), torch.randn(E, H, generator=g, device=DEV, dtype=BF) * 0.05
    bias = torch.rand(E, generator=g, device=DEV) * 0.1 if router == "sigmoid" else None
    kw = dict(router=router, expert_bias=bias, return_routing=True)
    out, w, idx = few.moe_layer_few(x, wr, b1, b2, K, **kw)
    _, w0, idx0 = few.moe_layer_few(x, wr, ops.unpack4(b1), ops.unpack4(b2), K, **kw)
    assert torch.equal(idx, idx0) and torch.equal(w, w0)
    _close(out, *_oracle(x, idx, w, b1, b2))
    kw["return_routing"] = False
    assert torch.equal(out, few.moe_layer_few(x, wr, b1, b2, K, **kw))


PROMPT = [  # T, H, E, K, I, skew
    (1, 64, 4, 2, 64, 0.0), (3, 192, 128, 8, 192, 0.0), (65, 320, 16, 4, 448, 0.0),
    (200, 64, 3, 1, 832, 0.0), (509, 1024, 128, 4, 768, 0.0), (300, 128, 2, 2, 128, 0.0),
    (1021, 256, 16, 8, 320, 2.0), (777, 704, 8, 3, 576, 0.0), (1500, 192, 4, 4, 128, 0.0),
    (4096, 512, 24, 8, 256, 3.0), (2050, 2048, 128, 8, 768, 1.0), (127, 64, 1, 1, 64, 0.0),
    (64, 64, 1, 1, 64, 0.0), (20, 128, 80, 70, 64, 0.0),
    (900, 448, 4, 3, 320, 0.0), (700, 960, 6, 2, 192, 1.0), (333, 512, 2, 1, 576, 0.0),
]


@pytest.mark.parametrize("T,H,E,K,I,skew", PROMPT)
def test_experts_forward(T, H, E, K, I, skew):
    g = _gen(T + I)
    b1, b2 = _bank(g, E, H, I)
    x, (idx, w) = _x(g, T, H), _routing(g, T, E, K, skew)
    out = experts_forward(x, idx, w, b1, b2)
    _close(out, *_oracle(x, idx, w, b1, b2, blocks=True))
    assert torch.equal(out, experts_forward(x, idx, w, b1, b2))


@pytest.mark.parametrize("H", [192, 448])
@pytest.mark.parametrize("rows", [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300])
def test_rows_of_an_expert(rows, H):
    """Row counts around the tiles' heights; one expert without a row, one with all."""
    g = _gen(rows)
    E, I = 3, 192
    b1, b2 = _bank(g, E, H, I)
    for e in (0, 2):
        x, idx = _x(g, rows, H), torch.full((rows, 1), e, device=DEV)
        w = torch.ones(rows, 1, device=DEV)
        _close(experts_forward(x, idx, w, b1, b2), *_oracle(x, idx, w, b1, b2, blocks=True))


def test_row_heights_give_the_same_bits():
    """A row's results do not depend on how many others there are."""
    g = _gen(5)
    E, H, I = 2, 512, 192
    b1, b2 = _bank(g, E, H, I)
    x = _x(g, 1500, H)
    idx = torch.arange(1500, device=DEV)[:, None] % 2
    w = torch.rand(1500, 1, generator=g, device=DEV)
    all_ = experts_forward(x, idx, w, b1, b2)
    for n in (10, 140, 300):
        assert torch.equal(all_[:n], experts_forward(x[:n], idx[:n], w[:n], b1, b2)), n


def test_not_finite_values_stay_in_their_rows():
    g = _gen(6)
    E, H, I = 4, 128, 128
    b1, b2 = _bank(g, E, H, I)
    x, (idx, w) = _x(g, 200, H), _routing(g, 200, E, 2)
    ref = experts_forward(x, idx, w, b1, b2)
    bad = x.clone()
    bad[17, 5], bad[60, 9] = torch.nan, torch.inf
    got = experts_forward(bad, idx, w, b1, b2)
    rows = torch.ones(200, dtype=torch.bool, device=DEV)
    rows[[17, 60]] = False
    assert torch.equal(got[rows], ref[rows]) and torch.isnan(got[17]).all()
    assert not torch.isfinite(got[60]).any()
    few_ref = few.experts_forward_few(x[:40], idx[:40], w[:40], b1, b2)
    few_got = few.experts_forward_few(bad[:40], idx[:40], w[:40], b1, b2)
    assert torch.equal(few_got[rows[:40]], few_ref[rows[:40]]) and torch.isnan(few_got[17]).all()
    # a weight that is not finite: the tokens of its expert alone
    w1 = ops.unpack4(b1)
    w1[2, 3, 40] = torch.inf
    bank = ops.pack4(w1)
    hit = (idx == 2).any(1)
    got = experts_forward(x, idx, w, bank, b2)
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], ref[~hit])
    got = few.experts_forward_few(x[:40], idx[:40], w[:40], bank, b2)
    assert torch.isnan(got[hit[:40]]).all() and torch.equal(got[~hit[:40]], few_ref[~hit[:40]])


@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** 40])
def test_magnitudes_of_y(scale):
    """The 16-bit blocks have y's range: weights of down_proj far from 1."""
    g = _gen(8)
    E, H, I, T = 2, 128, 64, 150
    b1, _ = _bank(g, E, H, I)
    b2 = ops.pack4(torch.randn(E, H, I, generator=g, device=DEV) * scale, dtype=BF)
    x, (idx, w) = _x(g, T, H), _routing(g, T, E, 1)
    _close(experts_forward(x, idx, w, b1, b2), *_oracle(x, idx, w, b1, b2, blocks=True))


def test_inputs_of_any_stride_and_type():
    g = _gen(9)
    E, H, I, T, K = 5, 128, 64, 70, 3
    b1, b2 = _bank(g, E, H, I)
    wide = _x(g, T, 2 * H)
    x, (idx, w) = wide[:, ::2], _routing(g, T, E, K)
    for fn, n in ((experts_forward, T), (few.experts_forward_few, 40)):
        ref = fn(x[:n].contiguous(), idx[:n], w[:n], b1, b2)
        assert torch.equal(ref, fn(x[:n], idx[:n].int(), w.t().contiguous().t()[:n], b1, b2))
        f32 = fn(x[:n].float(), idx[:n], w[:n], b1, b2)
        assert f32.dtype == F32 and torch.equal(f32, ref.float())
        moved = ops.Packed4(b1.q.transpose(1, 2).contiguous().transpose(1, 2), b1.scale, b1.shape, BF)
        assert torch.equal(ref, fn(x[:n], idx[:n], w[:n], moved, b2))
    assert experts_forward(x[:0], idx[:0], w[:0], b1, b2).shape == (0, H)
    assert few.experts_forward_few(x[:0], idx[:0], w[:0], b1, b2).shape == (0, H)


@pytest.mark.parametrize("router", ["softmax", "sigmoid"])
@pytest.mark.parametrize("gating", ["torch", "hip", "hip_fused"])
def test_moe_layer(router, gating):
    g = _gen(10)
    T, H, E, K, I = 150, 256, 128, 8, 64
    b1, b2 = _bank(g, E, H, I)
    x, wr = _x(g, T, H), torch.randn(E, H, generator=g, device=DEV, dtype=BF) * 0.05
    with torch.no_grad():
        out, probs, w, idx = moe_layer(x, wr, b1, b2, K, router=router, gating=gating)
        _, probs0, w0, idx0 = moe_layer(x, wr, ops.unpack4(b1), ops.unpack4(b2), K, router=router,
                                        gating=gating)
    assert torch.equal(idx, idx0) and torch.equal(w, w0) and torch.equal(probs, probs0)
    _close(out, *_oracle(x, idx, w, b1, b2, blocks=True))


def test_block_serves_prompt_and_tokens():
    """A block put in 4 bits: a prompt, then single tokens, as it is served; its
    state goes through state_dict."""
    H, E, K, I = 256, 32, 4, 128
    block = SparseMoeBlock(H, E, K, I).to(DEV, BF)
    g = _gen(11)
    with torch.no_grad():
        for p in block.parameters():
            p.copy_(torch.randn(p.shape, generator=g, device=DEV) * 0.02)
    exact1, exact2 = block.experts.gate_up_proj.detach(), block.experts.down_proj.detach()
    b1, b2 = ops.pack4(exact1), ops.pack4(exact2)
    assert block.pack_experts() is block
    block.few_tokens = 64
    assert [n for n, _ in block.experts.named_parameters()] == []
    x = _x(g, 3 * 50, H).view(3, 50, H)
    with torch.no_grad():
        out = block(x)
        w, idx = block.router_logits.gather(1, block.topk_index), block.topk_index
        w = w / w.sum(-1, keepdim=True)
        _close(out.view(-1, H), *_oracle(x.view(-1, H), idx, w, b1, b2, blocks=True))
        for t in range(3):
            y = _x(g, 3, H).view(3, 1, H)
            got = block(y)
            assert block.router_logits is None and got.shape == y.shape
            ref, w, idx = few.moe_layer_few(y.view(-1, H), block.gate.weight, b1, b2, K,
                                            return_routing=True)
            assert torch.equal(got.view(-1, H), ref)
            _close(ref, *_oracle(y.view(-1, H), idx, w, b1, b2))
        other = SparseMoeBlock(H, E, K, I).to(DEV, BF).pack_experts()
        other.load_state_dict(block.state_dict())
        assert torch.equal(other(x), out)
    with pytest.raises(RuntimeError, match="forward only"):
        block(x)


def test_transformers_bank():
    from transformers import Qwen3MoeConfig
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeForCausalLM
    cfg = Qwen3MoeConfig(vocab_size=64, hidden_size=128, intermediate_size=128,
                         moe_intermediate_size=64, num_hidden_layers=2, num_attention_heads=2,
                         num_key_value_heads=1, head_dim=64, num_experts=16, num_experts_per_tok=4,
                         norm_topk_prob=True, max_position_embeddings=64)
    torch.manual_seed(0)
    model = Qwen3MoeForCausalLM(cfg).to(DEV, BF).eval()
    twin = Qwen3MoeForCausalLM(cfg).to(DEV, BF).eval()
    twin.load_state_dict(model.state_dict())
    with torch.no_grad():   # the twin holds what the packed banks hold
        for bank in hf.expert_banks(twin):
            for p in (bank.gate_up_proj, bank.down_proj):
                p.copy_(ops.unpack4(ops.pack4(p)))
    hf.install(twin)
    assert hf.pack_experts(model) == 2 and hf.pack_experts(model) == 0
    hf.install(model, few_tokens=64)
    assert all(bank.few_tokens == 64 for bank in hf.expert_banks(model))
    for shape in ((2, 40), (2, 3)):
        ids = torch.randint(0, 64, shape, device=DEV)
        with torch.no_grad():
            a, b = model(ids).logits.float(), twin(ids).logits.float()
        # the twin rounds gate, up, silu and y to bf16 besides act; a layer's output is
        # within 4 roundings of 2^-8 of its sums' magnitudes, two layers and a head follow
        assert float((a - b).norm() / b.norm()) < 2 * 4 * U
    with pytest.raises(RuntimeError, match="forward only"):
        model(ids.repeat(1, 30))


def test_graphs_streams_and_workspaces():
    """Two captured graphs, each with its workspace, replayed by turns and beside
    eager calls; another stream."""
    g = _gen(12)
    H, E, K, I = 256, 16, 4, 128
    b1, b2 = _bank(g, E, H, I)
    wr = torch.randn(E, H, generator=g, device=DEV, dtype=BF) * 0.05
    xs = [_x(g, 3, H), _x(g, 20, H)]

    def call(x):
        return few.moe_layer_few(x, wr, b1, b2, K)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(s):
        for x in xs:
            call(x)
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=s):
                outs.append(call(x))
    torch.cuda.synchronize()
    for k in range(4):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        for i in (0, 1) if k % 2 else (1, 0):
            graphs[i].replay()
        eager = [call(x) for x in xs]
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o, e), k
    with torch.cuda.stream(s):
        side = experts_forward(xs[1], *_routing(_gen(1), 20, E, K), b1, b2)
    torch.cuda.synchronize()
    assert torch.equal(side, experts_forward(xs[1], *_routing(_gen(1), 20, E, K), b1, b2))


def test_custom_ops():
    g = _gen(13)
    T, H, E, K, I = 12, 128, 8, 2, 64
    b1, b2 = _bank(g, E, H, I)
    x, (idx, w) = _x(g, T, H), _routing(g, T, E, K)
    bank = (b1.q, b1.scale, b2.q, b2.scale)
    wr = torch.randn(E, H, generator=g, device=DEV, dtype=BF)
    torch.library.opcheck(torch.ops.moe_amd.experts_fwd4.default, (x, idx, w, *bank))
    torch.library.opcheck(torch.ops.moe_amd.experts_few4.default, (x, idx, w, *bank))
    torch.library.opcheck(torch.ops.moe_amd.moe_layer_few4.default,
                          (x, wr, *bank, K, "softmax", True, None, None, None, None, None))
    ref = experts_forward(x, idx, w, b1, b2), few.experts_forward_few(x, idx, w, b1, b2)

    def both(x, idx, w):
        return experts_forward(x, idx, w, b1, b2), few.experts_forward_few(x, idx, w, b1, b2)

    got = torch.compile(both, fullgraph=True)(x, idx, w)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_the_products_one_by_one():
    """The entries that experts_forward consists of, and the op of its dispatcher."""
    g = _gen(11)
    T, H, E, K, I = 333, 192, 9, 3, 128
    b1, b2 = _bank(g, E, H, I)
    x = _x(g, T, H)
    idx = torch.randint(-1, E + 1, (T, K), generator=g, device=DEV)
    w = torch.rand(T, K, generator=g, device=DEV)
    out = experts_forward(x, idx, w, b1, b2)
    plan = ops.permute(idx, E)
    y, ys = ops.gemm_down4(ops.gemm_gate_up_swiglu4(x, plan, b1), plan, b2)
    assert torch.equal(out, ops.combine16(y, ys, plan, w))
    assert torch.equal(out, torch.ops.moe_amd.experts_fwd4(x, idx, w, b1.q, b1.scale, b2.q, b2.scale))
    # other strides and types of the same values
    wide = torch.randn(T, 2 * H, generator=g, device=DEV, dtype=BF)
    wide[:, ::2] = x
    assert torch.equal(out, experts_forward(wide[:, ::2], idx.to(torch.int32), w.t().contiguous().t(),
                                            b1, b2))


def test_banks_past_four_gigabytes():
    """The last experts of a bank whose codes take more than 2^32 bytes."""
    g = _gen(14)
    E, H, I, K = 2800, 2048, 768, 2

    def bank(n, k):
        q = torch.empty(E, n // 16, k // 128, 1024, device=DEV, dtype=torch.uint8)
        for part in q.split(200):
            part.random_(0, 256, generator=g)
        s = torch.randint(119, 122, (E, n // 16, k // 128, 64), generator=g, device=DEV)
        return ops.Packed4(q, s.to(torch.uint8), (E, n, k), BF)

    b1, b2 = bank(2 * I, H), bank(H, I)
    assert b1.q.numel() > 1 << 32
    idx = torch.tensor([[E - 1, 0], [E - 2, E - 1], [2733, 1400]], device=DEV).repeat(14, 1)
    x, w = _x(g, len(idx), H), torch.rand(len(idx), K, generator=g, device=DEV)
    _close(few.experts_forward_few(x, idx, w, b1, b2), *_oracle(x, idx, w, b1, b2))
    _close(few.experts_forward_few(x[:1], idx[:1], w[:1], b1, b2),
           *_oracle(x[:1], idx[:1], w[:1], b1, b2))
    _close(experts_forward(x, idx, w, b1, b2), *_oracle(x, idx, w, b1, b2, blocks=True))
    # a tile row and an expert's end of the bank through the packing too
    last = ops.Packed4(b1.q[E - 1:], b1.scale[E - 1:], (1, 2 * I, H), BF)
    whole = ops.unpack4(ops.Packed4(b1.q, b1.scale, b1.shape, BF))
    assert torch.equal(whole[E - 1:], ops.unpack4(last))


@pytest.mark.parametrize("T", [1, 3, 40])
def test_masked_places_hold_anything(T):
    """Ids far outside [0, E), NaN and infinite weights beside them, and hidden states that
    are not finite in a token without experts."""
    g = _gen(15)
    E, H, I, K = 9, 128, 192, 4
    b1, b2 = _bank(g, E, H, I)
    x = _x(g, T + 1, H)
    idx = torch.randint(0, E, (T + 1, K), generator=g, device=DEV)
    w = torch.rand(T + 1, K, generator=g, device=DEV)
    idx[:, 1], w[:, 1] = (1 << 33) + 2, torch.nan
    idx[0, 2], w[0, 2] = -(1 << 40), torch.inf
    idx[T], x[T] = E, torch.nan
    clean = torch.where((idx >= 0) & (idx < E), w, torch.zeros_like(w))
    for fn, blocks in ((experts_forward, True), (few.experts_forward_few, False)):
        out = fn(x, idx, w, b1, b2)
        assert (out[T] == 0).all()
        _close(out[:T], *_oracle(x[:T], idx[:T], clean[:T], b1, b2, blocks=blocks))
        one = fn(x[:1], idx[:1], w[:1], b1, b2)
        _close(one, *_oracle(x[:1], idx[:1], clean[:1], b1, b2, blocks=blocks))


def test_as_many_tokens_as_are_taken():
    """The most tokens of 2048 columns, y beyond 2^32 bytes: some of them give the bits
    that they give alone; one token more is refused."""
    g = _gen(16)
    T, H, E, K, I = (1 << 19) - 1, 2048, 4, 3, 64
    b1, b2 = _bank(g, E, H, I)
    x = _x(g, T, H)
    idx = torch.randint(-1, E, (T, K), generator=g, device=DEV)
    w = torch.rand(T, K, generator=g, device=DEV)
    out = experts_forward(x, idx, w, b1, b2)
    some = torch.cat([torch.arange(0, T, 4099, device=DEV), torch.arange(T - 70, T, device=DEV)])
    assert torch.equal(out[some], experts_forward(x[some], idx[some], w[some], b1, b2))
    _close(out[some[-70:]], *_oracle(x[some[-70:]], idx[some[-70:]], w[some[-70:]], b1, b2,
                                     blocks=True))
    del out, x
    with pytest.raises(RuntimeError, match="T.H too large"):
        experts_forward(torch.zeros(T + 1, H, device=DEV, dtype=BF), idx[:1].expand(T + 1, K),
                        w[:1].expand(T + 1, K), b1, b2)


def test_calls_that_overlap():
    """Prompts and tokens on the same bank from two streams at once."""
    g = _gen(17)
    H, E, K, I = 512, 32, 4, 256
    b1, b2 = _bank(g, E, H, I)
    sets = [(_x(g, T, H), *_routing(g, T, E, K)) for T in (2000, 1500)]
    ref = [(experts_forward(*s, b1, b2), few.experts_forward_few(*(t[:50] for t in s), b1, b2))
           for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append((experts_forward(*sets[i], b1, b2),
                               few.experts_forward_few(*(t[:50] for t in sets[i]), b1, b2)))
    torch.cuda.synchronize()
    for r, outs in zip(ref, got):
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, r))
