"""The few-token layer against the formulas in 64 bits.

Tolerances.  Let u be half a step of the layer's type relative to a value
(bf16 2^-8, fp32 2^-24) and v = 2^-24.  A sum of n fp32 products is off by at
most n v sum|a b|, so gate and up are off by dg = H v |W1| |x|; with |silu'| <
1.1 and |silu(g)| <= |g|, act before its rounding by da = 1.1 dg |up| + |gate|
du + dg du + 8 v |act| (the last term: exp, divide and products in fp32), and
by u (|act| + da) more after it.  y is off by |W2| (da + u (|act| + da)) + I v
|W2| (|act| + ...), out by the weighted sum of that, K v |w y| more and its own
rounding.  The bounds below are these sums, evaluated in 64 bits.
"""
from __future__ import annotations

import pytest
import torch

from moe_amd import _lib, few, hf, ops
from moe_amd.experts import experts_forward
from moe_amd.layer import SparseMoeBlock, moe_layer

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
V = 2.0 ** -24


def _half(dt):
    return torch.finfo(dt).eps / 2


def _weights(g, E, H, I, dt):
    w1 = (torch.randn(E, 2 * I, H, generator=g, device=DEV) * 0.02).to(dt)
    w2 = (torch.randn(E, H, I, generator=g, device=DEV) * 0.02).to(dt)
    return w1, w2


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _oracle(x, idx, w, w1, w2):
    """(out, bound) in 64 bits, entry by entry."""
    T, H = x.shape
    E, I = w1.shape[0], w2.shape[2]
    K = idx.shape[1]
    u = _half(x.dtype)
    out = torch.zeros(T, H, device=DEV, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for e in torch.unique(idx).tolist():
        if not 0 <= e < E:
            continue
        t, k = torch.nonzero(idx == e, as_tuple=True)
        m1, m2 = w1[e].double(), w2[e].double()
        xt, wk = x[t].double(), w[t, k].double()[:, None]
        gu, dgu = xt @ m1.t(), H * V * (xt.abs() @ m1.abs().t())
        gt, up, dg, du = gu[:, :I], gu[:, I:], dgu[:, :I], dgu[:, I:]
        act = gt * torch.sigmoid(gt) * up
        da = 1.1 * dg * up.abs() + gt.abs() * du + dg * du + 8 * V * act.abs()
        da = da + u * (act.abs() + da)
        y = act @ m2.t()
        dy = da @ m2.abs().t() + I * V * ((act.abs() + da) @ m2.abs().t())
        out.index_add_(0, t, y * wk)
        tol.index_add_(0, t, wk.abs() * (dy + (K + 1) * V * y.abs()))
    return out, tol + u * (out.abs() + tol)


def _close(got, ref, tol):
    assert torch.isfinite(got).all()
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst by " \
        f"{float(((got.double() - ref).abs() / tol.clamp(min=1e-300)).max()):.2f} bounds"


def _routing(g, T, E, K):
    idx = torch.rand(T, E, generator=g, device=DEV).argsort(1)[:, :K].contiguous()
    return idx, torch.rand(T, K, generator=g, device=DEV) + 0.1


SHAPES = [  # T, H, E, K, I
    (1, 64, 4, 2, 64),
    (1, 2048, 128, 8, 768),
    (2, 128, 1, 1, 64),
    (3, 1024, 16, 4, 768),
    (5, 192, 16, 4, 320),
    (16, 512, 8, 8, 128),       # 16 rows in every expert
    (17, 448, 8, 8, 192),       # 17
    (33, 1024, 128, 4, 768),
    (63, 320, 6, 3, 832),
    (64, 128, 1792, 8, 64),
    (64, 576, 4, 4, 64),        # 64 rows in every expert
    (64, 128, 40, 16, 1088),
    (64, 4096, 20, 16, 64),     # 1024 rows: the down kernel's largest LDS
    (3, 8192, 4, 2, 192),
    (2, 64, 3, 2, 4160),
]


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T,H,E,K,I", SHAPES)
def test_experts(T, H, E, K, I, dt):
    print(f"experts_few {T} {H} {E} {K} {I} {dt}", flush=True)
    g = _gen(T * 1000 + H)
    x = torch.randn(T, H, generator=g, device=DEV).to(dt)
    w1, w2 = _weights(g, E, H, I, dt)
    idx, w = _routing(g, T, E, K)
    ref, tol = _oracle(x, idx, w, w1, w2)
    got = few.experts_forward_few(x, idx, w, w1, w2)
    assert got.dtype == dt and got.shape == x.shape
    _close(got, ref, tol)
    assert torch.equal(got, few.experts_forward_few(x, idx, w, w1, w2))
    wb = w.bfloat16()
    ref, tol = _oracle(x, idx, wb, w1, w2)
    _close(few.experts_forward_few(x, idx, wb, w1, w2), ref, tol)


@pytest.mark.parametrize("seed", range(6))
def test_few_entries_in_any_arrangement(seed):
    """Up to 64 entries, whose list every workgroup makes for itself: random ids
    over few or many experts, padded and repeated."""
    print(f"experts_few arrangement {seed}", flush=True)
    g = _gen(100 + seed)
    T, K = ((2, 3), (8, 8), (7, 9), (16, 4), (64, 1), (3, 16))[seed]
    E, H, I = (2, 3, 200, 5, 4, 9)[seed], 128, 128
    x = torch.randn(T, H, generator=g, device=DEV).to(BF)
    w1, w2 = _weights(g, E, H, I, BF)
    idx = torch.randint(-1, E + 1, (T, K), generator=g, device=DEV)
    w = torch.rand(T, K, generator=g, device=DEV)
    _close(few.experts_forward_few(x, idx, w, w1, w2), *_oracle(x, idx, w, w1, w2))


@pytest.mark.parametrize("T", [21, 9])
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
def test_padding_contributes_nothing(dt, T):
    print("experts_few padding", flush=True)
    H, E, K, I = 256, 12, 4, 128
    g = _gen(5)
    x = torch.randn(T, H, generator=g, device=DEV).to(dt)
    w1, w2 = _weights(g, E, H, I, dt)
    idx, w = _routing(g, T, E, K)
    idx[3] = -1
    idx[4] = E
    idx[7, 1:] = (1 << 40) + 1     # beyond 32 bits; its low half is a real id
    idx[6, 2] = -(1 << 40) + 2
    last = T - 1
    idx[last] = E + 5
    # what padding names may hold anything
    w[idx.lt(0) | idx.ge(E)] = float("nan")
    x[3], x[4], x[last] = float("nan"), float("inf"), float("-inf")
    ref, tol = _oracle(torch.nan_to_num(x, 0.0, 0.0, 0.0), idx, torch.nan_to_num(w), w1, w2)
    got = few.experts_forward_few(x, idx, w, w1, w2)
    _close(got, ref, tol)
    assert (got[[3, 4, last]] == 0).all()
    # nothing but padding
    assert (few.experts_forward_few(x, torch.full_like(idx, E), w, w1, w2) == 0).all()


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("ids", [[5, -1, 7, 0], [-1, 5, 9, 7], [9, -1, 1 << 33, -3], [2, 2, 7, 2],
                                 [0, 1, 2, 3], [8, 8, 8, 7]])
def test_one_token_with_padding_and_repeats(ids, dt):
    print(f"experts_few one token {ids}", flush=True)
    H, E, I = 320, 8, 192
    g = _gen(15)
    x = torch.randn(1, H, generator=g, device=DEV).to(dt)
    w1, w2 = _weights(g, E, H, I, dt)
    idx = torch.tensor([ids], device=DEV)
    w = torch.rand(1, 4, generator=g, device=DEV)
    w[idx.lt(0) | idx.ge(E)] = float("nan")
    got = few.experts_forward_few(x, idx, w, w1, w2)
    _close(got, *_oracle(x, idx, torch.nan_to_num(w), w1, w2))
    # as one of several tokens: the same sums
    many = few.experts_forward_few(x.repeat(3, 1), idx.repeat(3, 1), w.repeat(3, 1), w1, w2)
    assert torch.equal(many, got.expand(3, H))


def test_a_value_that_is_not_finite_stays_with_its_token():
    print("experts_few not finite", flush=True)
    T, H, E, K, I = 19, 256, 2, 2, 64
    g = _gen(6)
    x = torch.randn(T, H, generator=g, device=DEV).to(BF)
    w1, w2 = _weights(g, E, H, I, BF)
    idx, w = _routing(g, T, E, K)
    clean = few.experts_forward_few(x, idx, w, w1, w2)
    x[0, 3], x[18, 255] = float("nan"), float("inf")
    got = few.experts_forward_few(x, idx, w, w1, w2)
    assert torch.equal(got[1:18], clean[1:18])
    assert got[0].isnan().all() and not got[18].isfinite().any()


@pytest.mark.parametrize("T,K", [(3, 2), (64, 16), (4, 16), (8, 8), (5, 13), (2, 16), (9, 7)])
def test_one_expert_named_many_times(T, K):
    print(f"experts_few same expert {T} {K}", flush=True)
    H, E, I = 128, 3, 64
    g = _gen(7)
    x = torch.randn(T, H, generator=g, device=DEV).to(BF)
    w1, w2 = _weights(g, E, H, I, BF)
    idx = torch.full((T, K), 2, device=DEV)
    w = torch.rand(T, K, generator=g, device=DEV)
    ref, tol = _oracle(x, idx, w, w1, w2)
    _close(few.experts_forward_few(x, idx, w, w1, w2), ref, tol)


def test_a_bank_beyond_32_bit_offsets():
    print("experts_few large bank", flush=True)
    T, H, E, K, I = 3, 2048, 1792, 2, 768
    g = _gen(8)
    w1 = torch.zeros(E, 2 * I, H, device=DEV, dtype=BF)   # 5.6e9 values
    w2 = torch.zeros(E, H, I, device=DEV, dtype=BF)
    for e in (0, E - 2, E - 1):
        w1[e] = (torch.randn(2 * I, H, generator=g, device=DEV) * 0.02).to(BF)
        w2[e] = (torch.randn(H, I, generator=g, device=DEV) * 0.02).to(BF)
    x = torch.randn(T, H, generator=g, device=DEV).to(BF)
    idx = torch.tensor([[E - 1, 0], [E - 2, E - 1], [0, E - 2]], device=DEV)
    w = torch.rand(T, K, generator=g, device=DEV)
    ref, tol = _oracle(x, idx, w, w1, w2)
    _close(few.experts_forward_few(x, idx, w, w1, w2), ref, tol)


def test_strided_and_other_dtypes():
    print("experts_few strides", flush=True)
    T, H, E, K, I = 6, 128, 8, 2, 64
    g = _gen(9)
    xx = torch.randn(T, 2 * H, generator=g, device=DEV).to(BF)
    w1, w2 = _weights(g, E, H, I, BF)
    idx, w = _routing(g, T, E, K)
    want = few.experts_forward_few(xx[:, :H].contiguous(), idx, w, w1, w2)
    assert torch.equal(few.experts_forward_few(xx[:, :H], idx, w, w1, w2), want)
    wide = torch.stack([idx, idx], -1)[..., 0]
    assert torch.equal(few.experts_forward_few(xx[:, :H], wide.int(), w.t().contiguous().t(), w1,
                                               w2), want)
    # fp32 hidden states over bf16 weights are cast, the result cast back
    got = few.experts_forward_few(xx[:, :H].float(), idx, w, w1, w2)
    assert got.dtype == F32 and torch.equal(got.to(BF), want)
    # some of a bank's experts: a view that starts inside it
    part = few.experts_forward_few(xx[:, :H], idx % 3, w, w1[2:5], w2[2:5])
    assert torch.equal(part, few.experts_forward_few(xx[:, :H], idx % 3 + 2, w, w1, w2))


def test_subnormal_fp32():
    """fp32 operands and sums below 2^-126 are kept, to the last of their bits:
    half a step of 2^-149 for each of the I products' sums and the K y's."""
    print("experts_few subnormal", flush=True)
    T, H, E, K, I = 3, 128, 4, 2, 64
    g = _gen(16)
    x = torch.randn(T, H, generator=g, device=DEV)
    w1, w2 = _weights(g, E, H, I, F32)
    w1 = w1 * 20
    w2 = (w2.double() * 2.0 ** -130).float()
    idx, w = _routing(g, T, E, K)
    ref, tol = _oracle(x, idx, w, w1, w2)
    got = few.experts_forward_few(x, idx, w, w1, w2)
    assert (ref.abs().max() < 2.0 ** -126) and (got != 0).any()
    assert ((got.double() - ref).abs() <= tol + (I + K + 1) * K * 2.0 ** -149).all()


def test_no_tokens():
    w1, w2 = _weights(_gen(1), 4, 128, 64, BF)
    x = torch.empty(0, 128, device=DEV, dtype=BF)
    idx, w = torch.empty(0, 2, device=DEV, dtype=torch.int64), torch.empty(0, 2, device=DEV)
    assert few.experts_forward_few(x, idx, w, w1, w2).shape == (0, 128)
    out, w, idx = few.moe_layer_few(x, torch.zeros(4, 128, device=DEV, dtype=BF), w1, w2, 2,
                                    return_routing=True)
    assert out.shape == (0, 128) and w.shape == idx.shape == (0, 2)


def test_writes_its_output_only():
    """Guards around the output and behind the workspace stay as they were."""
    print("experts_few guards", flush=True)
    T, H, E, K, I = 13, 192, 8, 4, 64
    g = _gen(10)
    x = torch.randn(T, H, generator=g, device=DEV).to(BF)
    w1, w2 = _weights(g, E, H, I, BF)
    idx, w = _routing(g, T, E, K)
    want = few.experts_forward_few(x, idx, w, w1, w2)
    n = _lib.load().moe_amd_few_workspace_size(T, E, K, H, I, 1)
    ws = torch.full((n + 4096,), 0x5A, device=DEV, dtype=torch.uint8)
    out = torch.full((T + 2, H), 7.0, device=DEV, dtype=BF)
    _lib.call("moe_amd_experts_few", x.data_ptr(), idx.data_ptr(), w.data_ptr(), 0, w1.data_ptr(),
              w2.data_ptr(), T, K, E, H, I, 1, ws.data_ptr(), n, out[1:].data_ptr(),
              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(out[1:T + 1], want)
    assert (out[0] == 7).all() and (out[T + 1] == 7).all() and (ws[n:] == 0x5A).all()


# ---------------------------------------------------------------- the layer

def _layer(g, T, H, E, I, dt, whole=False):
    x = torch.randn(T, H, generator=g, device=DEV)
    wr = torch.randn(E, H, generator=g, device=DEV)
    if whole:  # small whole numbers: every logit exact in any order, many of them equal
        x, wr = x.clamp(-2, 2).round(), (wr * 0.4).clamp(-1, 1).round()
    else:
        wr = wr * 0.02
    return (x.to(dt), wr.to(dt)) + _weights(g, E, H, I, dt)


def _select(rank, K):
    return torch.sort(rank, dim=-1, descending=True, stable=True)[1][:, :K]


def _softmax_ref(logits, K, renorm):
    p = torch.softmax(logits, -1)
    idx = _select(logits, K)
    w = p.gather(1, idx)
    return (w / w.sum(-1, keepdim=True) if renorm else w), idx


# exp, sums and divides in fp32: e^(l - m) is off by |l - m| v + 2 v, a sum of E terms by
# E v more, a quotient and the renormalisation by as much again
def _w_tol(w, E, spread):
    return w * (4 * E + 2 * spread + 32) * V + 1e-37


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T,H,E,K,I,renorm", [
    (1, 128, 128, 8, 64, True), (7, 64, 16, 16, 64, False), (64, 256, 64, 6, 64, True),
    (5, 64, 1792, 8, 64, True), (3, 64, 4096, 4, 64, False), (33, 128, 200, 1, 64, True),
    (1, 64, 1, 1, 64, True), (1, 64, 300, 16, 64, True), (1, 128, 256, 16, 64, False),
    (2, 64, 257, 5, 64, True), (2, 256, 128, 8, 128, True), (2, 64, 20, 16, 64, False), (19, 192, 16, 16, 128, True)])
def test_layer_softmax_on_exact_logits(T, H, E, K, I, renorm, dt):
    print(f"moe_layer_few softmax {T} {H} {E} {K} {dt}", flush=True)
    x, wr, w1, w2 = _layer(_gen(E + K), T, H, E, I, dt, whole=True)
    logits = (x.double() @ wr.double().t().contiguous()).to(dt).double()  # |logit| <= 512: exact
    w_ref, i_ref = _softmax_ref(logits, K, renorm)
    out, w, idx = few.moe_layer_few(x, wr, w1, w2, K, renormalize=renorm, return_routing=True)
    assert torch.equal(idx, i_ref)
    spread = float(logits.max() - logits.min())
    assert ((w.double() - w_ref).abs() <= _w_tol(w_ref, E, spread)).all()
    _close(out, *_oracle(x, idx, w, w1, w2))
    assert torch.equal(few.moe_layer_few(x, wr, w1, w2, K, renormalize=renorm), out)


@pytest.mark.parametrize("T,H,E,K,groups,gtopk,scale", [
    (1, 128, 64, 8, None, None, 2.5), (17, 128, 64, 8, 8, 4, None), (64, 64, 1792, 8, None, None, None),
    (9, 64, 96, 6, 3, 2, 1.5), (4, 64, 128, 16, 64, 16, None), (5, 64, 256, 4, 1, 1, None),
    (2, 64, 64, 8, 4, 2, None), (2, 64, 200, 16, None, None, None), (3, 64, 1024, 8, 8, 4, None), (1, 64, 512, 8, 64, 8, 2.0), (17, 64, 320, 6, 5, 3, None)])
def test_layer_sigmoid_on_exact_logits(T, H, E, K, groups, gtopk, scale):
    print(f"moe_layer_few sigmoid {T} {H} {E} {K} {groups}", flush=True)
    g = _gen(E * K)
    x, wr, w1, w2 = _layer(g, T, H, E, 64, BF, whole=True)
    x, wr = x.clamp(-1, 1), wr * 0.0625   # logits of multiples of 1/16
    bias = (torch.randint(-8, 8, (E,), generator=g, device=DEV) / 64).float()
    # the router kernel on the same fp32 logits: same arithmetic, same order
    logits = (x.float().double() @ wr.double().t().contiguous()).float()
    scores, w_ref, i_ref = ops.router_sigmoid_topk(logits, bias, K, True, scale, groups, gtopk,
                                                   torch.float32)
    out, w, idx = few.moe_layer_few(x, wr, w1, w2, K, router="sigmoid", expert_bias=bias,
                                    scaling_factor=scale, num_groups=groups, group_topk=gtopk,
                                    return_routing=True)
    assert torch.equal(idx, i_ref) and torch.equal(w, w_ref)
    if not groups:  # and the definition
        sel = _select((scores + bias).double(), K)
        assert torch.equal(idx, sel)
        s = torch.sigmoid(logits.double()).gather(1, sel)
        ref = s / (s.sum(-1, keepdim=True) + 1e-20) * (scale or 1.0)
        assert ((w.double() - ref).abs() <= ref * (2 * K + 32) * V).all()
    _close(out, *_oracle(x, idx, w, w1, w2))


@pytest.mark.parametrize("router", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
def test_layer_on_random_logits(router, dt):
    """Selections on rounded sums: no unselected expert beats a selected one by
    more than the logits' error (H v |x||W_r| of the sum, half a bf16 step on
    either side for the softmax router's bf16 logits)."""
    print(f"moe_layer_few random {router} {dt}", flush=True)
    T, H, E, K, I = 37, 1024, 128, 8, 128
    x, wr, w1, w2 = _layer(_gen(3), T, H, E, I, dt)
    out, w, idx = few.moe_layer_few(x, wr, w1, w2, K, router=router, return_routing=True)
    logits = x.double() @ wr.double().t().contiguous()
    err = H * V * (x.double().abs() @ wr.double().abs().t().contiguous())
    if router == "softmax" and dt == BF:
        err = err + _half(BF) * (logits.abs() + err)
    lo = (logits - err).scatter(1, idx, float("-inf")).amax(1)
    hi = (logits + err).gather(1, idx).amin(1)
    assert (lo <= hi).all()
    assert all(len(set(r)) == K for r in idx.tolist())
    _close(out, *_oracle(x, idx, w, w1, w2))


def test_layer_offsets_masks_and_nan():
    print("moe_layer_few masks", flush=True)
    T, H, E, K, I = 6, 64, 32, 4, 64
    x, wr, w1, w2 = _layer(_gen(12), T, H, E, I, BF, whole=True)
    off = torch.zeros(E, device=DEV)
    off[:20] = float("-inf")
    off[20:24] = torch.finfo(F32).min
    off[30] = 3.0
    logits = x.double() @ wr.double().t().contiguous() + off.double()
    w_ref, i_ref = _softmax_ref(logits, K, True)
    out, w, idx = few.moe_layer_few(x, wr, w1, w2, K, logit_offset=off, return_routing=True)
    assert torch.equal(idx, i_ref)
    assert ((w.double() - w_ref).abs() <= _w_tol(w_ref, E, 600)).all()
    _close(out, *_oracle(x, idx, w, w1, w2))
    # fewer open experts than K: the closed ones fill up in order, with weight zero
    off[:] = float("-inf")
    off[[7, 9]] = 0.0
    out, w, idx = few.moe_layer_few(x, wr, w1, w2, K, logit_offset=off, return_routing=True)
    assert (idx[:, 2:] == torch.tensor([0, 1], device=DEV)).all() and (w[:, 2:] == 0).all()
    _close(out, *_oracle(x, idx, w, w1, w2))
    # a token that is not finite has no routing, the others keep theirs
    x[2, 5] = float("nan")
    out2, w2_, idx2 = few.moe_layer_few(x, wr, w1, w2, K, logit_offset=off, return_routing=True)
    keep = [0, 1, 3, 4, 5]
    assert torch.equal(out2[keep], out[keep]) and out2[2].isnan().all()
    assert (idx2[2] == torch.arange(K, device=DEV)).all()


def test_layer_agrees_with_moe_layer():
    """Against the framework's own layer, whose gate, up and y are rounded to
    bf16 on the way: five roundings of half a step where this has two."""
    print("moe_layer_few vs moe_layer", flush=True)
    T, H, E, K, I = 48, 512, 64, 8, 256
    x, wr, w1, w2 = _layer(_gen(14), T, H, E, I, BF, whole=True)
    ref, _, w_ref, i_ref = moe_layer(x, wr, w1, w2, K, gating="hip")
    out, w, idx = few.moe_layer_few(x, wr, w1, w2, K, return_routing=True)
    assert torch.equal(idx, i_ref)
    d = (out.double() - ref.double()).norm() / ref.double().norm()
    assert d <= 7 * _half(BF)
    with torch.no_grad():
        a = experts_forward(x, i_ref, w_ref, w1, w2)
    b = few.experts_forward_few(x, i_ref, w_ref, w1, w2)
    assert (a.double() - b.double()).norm() / a.double().norm() <= 7 * _half(BF)


def test_block_and_bank_choose_by_tokens():
    print("SparseMoeBlock few_tokens", flush=True)
    H, E, K, I = 128, 8, 2, 64
    torch.manual_seed(0)
    blk = SparseMoeBlock(H, E, K, I).to(DEV, BF)
    with torch.no_grad():
        for p in blk.parameters():
            p.normal_(0, 0.1)
    h = torch.randn(2, 3, H, device=DEV, dtype=BF)
    with torch.no_grad():
        ref = blk(h)
        assert blk.router_logits is not None
        blk.few_tokens = 6
        got = blk(h)
        assert blk.router_logits is None and got.shape == h.shape
        want = few.moe_layer_few(h.reshape(-1, H), blk.gate.weight, blk.experts.gate_up_proj,
                                 blk.experts.down_proj, K)
        assert torch.equal(got.reshape(-1, H), want)
        big = blk(h.repeat(2, 1, 1))   # 12 tokens: the other form
        assert torch.equal(big[:2], ref) and blk.router_logits is not None
    out = blk(h)                       # a gradient is wanted: the other form
    out.sum().backward()
    assert blk.experts.down_proj.grad is not None and torch.equal(out.detach(), ref)
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        blk(h)
        assert blk.router_logits is not None
    blk.router = "sigmoid"
    with torch.no_grad():
        got = blk(h)
        want = few.moe_layer_few(h.reshape(-1, H), blk.gate.weight, blk.experts.gate_up_proj,
                                 blk.experts.down_proj, K, router="sigmoid",
                                 expert_bias=blk.expert_bias)
        assert torch.equal(got.reshape(-1, H), want)


def test_hf_model_decodes_through_the_few_token_experts(monkeypatch):
    print("hf few_tokens", flush=True)
    from transformers import Qwen3MoeConfig, Qwen3MoeForCausalLM
    cfg = Qwen3MoeConfig(vocab_size=64, hidden_size=128, intermediate_size=128,
                         moe_intermediate_size=64, num_hidden_layers=2, num_attention_heads=2,
                         num_key_value_heads=1, head_dim=64, num_experts=8,
                         num_experts_per_tok=2, norm_topk_prob=True, decoder_sparse_step=1,
                         max_position_embeddings=64)
    torch.manual_seed(0)
    m = Qwen3MoeForCausalLM(cfg).to(DEV, BF).eval()
    hf.install(m, few_tokens=16)
    calls = []
    real = few.experts_forward_few
    monkeypatch.setattr(few, "experts_forward_few", lambda *a: calls.append(len(a[0])) or real(*a))
    ids = torch.randint(0, 64, (2, 4), device=DEV)
    with torch.no_grad():
        got = m(ids).logits
        assert calls == [8, 8]
        hf.install(m)
        ref = m(ids).logits
    assert calls == [8, 8]
    assert (got.double() - ref.double()).norm() / ref.double().norm() < 0.02
    m(ids).logits.float().sum().backward()   # training keeps the other form
    assert calls == [8, 8]


# ------------------------------------------------------- streams and graphs

def test_two_streams_at_once():
    print("few: two streams", flush=True)
    T, H, E, K, I = 32, 512, 32, 4, 256
    sets = [_layer(_gen(20 + i), T, H, E, I, BF) for i in range(2)]
    want = [few.moe_layer_few(*s, K) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(few.moe_layer_few(*sets[i], K))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_graph_replays():
    print("few: graph", flush=True)
    T, H, E, K, I = 9, 256, 16, 4, 128
    x, wr, w1, w2 = _layer(_gen(30), T, H, E, I, BF)
    xs = x.clone()

    def step():
        a = few.moe_layer_few(xs, wr, w1, w2, K)
        out, w, idx = few.moe_layer_few(a, wr, w1, w2, K, router="sigmoid", return_routing=True)
        return out, few.experts_forward_few(out, idx, w, w1, w2)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        xs.copy_(torch.randn(T, H, generator=_gen(40 + i), device=DEV).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_compiled_and_custom_ops():
    print("few: custom ops", flush=True)
    T, H, E, K, I = 5, 128, 8, 2, 64
    x, wr, w1, w2 = _layer(_gen(50), T, H, E, I, BF)
    out, w, idx = few.moe_layer_few(x, wr, w1, w2, K, return_routing=True)
    utils = ("test_schema", "test_faketensor")
    torch.library.opcheck(torch.ops.moe_amd.experts_few.default, (x, idx, w, w1, w2),
                          test_utils=utils)
    args = (x, wr, w1, w2, K, "softmax", True, None, None, None, None, None)
    torch.library.opcheck(torch.ops.moe_amd.moe_layer_few.default, args, test_utils=utils)
    assert torch.equal(torch.ops.moe_amd.moe_layer_few(*args)[0], out)

    @torch.no_grad()
    def fn(x):
        a, w, idx = few.moe_layer_few(x, wr, w1, w2, K, return_routing=True)
        return few.moe_layer_few(a, wr, w1, w2, K), few.experts_forward_few(a, idx, w, w1, w2)

    for a, b in zip(torch.compile(fn, fullgraph=True, backend="aot_eager")(x), fn(x)):
        assert torch.equal(a, b)


def test_refusals_on_the_gpu():
    x, wr, w1, w2 = _layer(_gen(60), 4, 128, 8, 64, BF)
    idx = torch.zeros(4, 2, device=DEV, dtype=torch.int64)
    w = torch.ones(4, 2, device=DEV)
    with pytest.raises(RuntimeError, match="at most 64"):
        few.experts_forward_few(x.repeat(17, 1), idx.repeat(17, 1), w.repeat(17, 1), w1, w2)
    with pytest.raises(ValueError, match="shape mismatch"):
        few.experts_forward_few(x[:, :64], idx, w, w1, w2)
    with pytest.raises(ValueError, match="must both be"):
        few.experts_forward_few(x, idx[:3], w, w1, w2)
    with pytest.raises(TypeError, match="dtypes"):
        few.experts_forward_few(x, idx, w, w1, w2.float())
    with pytest.raises(TypeError, match="unsupported dtype"):
        few.experts_forward_few(x, idx, w, w1.half(), w2.half())
    with pytest.raises(TypeError, match="unsupported dtype"):
        few.experts_forward_few(x, idx, w.double(), w1, w2)
    with pytest.raises(ValueError, match="unknown router"):
        few.moe_layer_few(x, wr, w1, w2, 2, router="hash")
    with pytest.raises(ValueError, match="softmax router's"):
        few.moe_layer_few(x, wr, w1, w2, 2, expert_bias=torch.zeros(8, device=DEV))
    with pytest.raises(ValueError, match="router weight"):
        few.moe_layer_few(x, wr[:4], w1, w2, 2)
    with pytest.raises(ValueError, match="offset or bias"):
        few.moe_layer_few(x, wr, w1, w2, 2, logit_offset=torch.zeros(4, device=DEV))
    with pytest.raises(RuntimeError, match="K=9"):
        few.moe_layer_few(x, wr, w1, w2, 9)
    flat = torch.empty(4 * 128 + 4, device=DEV, dtype=BF)
    with pytest.raises(RuntimeError, match="MOE_ERR_ALIGN"):
        few.experts_forward_few(flat[4:].view(4, 128), idx, w, w1, w2)


def test_block_of_mixed_dtypes():
    """fp32 router weights over bf16 experts: the same with few_tokens as without."""
    print("SparseMoeBlock fp32 gate", flush=True)
    torch.manual_seed(1)
    blk = SparseMoeBlock(128, 8, 2, 64, router="sigmoid").to(DEV, BF)
    with torch.no_grad():
        for p in blk.parameters():
            p.normal_(0, 0.1)
        blk.gate.float()
        for dt in (BF, torch.float32):
            h = torch.randn(5, 128, device=DEV).to(dt)
            blk.few_tokens = 0
            ref = blk(h)
            blk.few_tokens = 8
            got = blk(h)
            assert got.dtype == dt and torch.equal(got, ref)


@pytest.mark.parametrize("how", ["make_fx", "make_fx_pre_dispatch", "jit_trace"])
def test_traces_repeat_on_other_inputs(how):
    from torch.fx.experimental.proxy_tensor import make_fx

    print(f"few: {how}", flush=True)
    T, H, E, K, I = 5, 128, 8, 2, 64
    x, wr, w1, w2 = _layer(_gen(70), T, H, E, I, BF)
    idx, w = _routing(_gen(71), T, E, K)

    def fn(x, idx, w):
        return few.experts_forward_few(few.moe_layer_few(x, wr, w1, w2, K), idx, w, w1, w2)

    with torch.no_grad():
        if how == "jit_trace":
            traced = torch.jit.trace(fn, (x, idx, w))
        else:
            traced = make_fx(fn, pre_dispatch=how != "make_fx")(x, idx, w)
        for seed in (72, 73):
            x = _layer(_gen(seed), T, H, E, I, BF)[0]
            idx, w = _routing(_gen(seed), T, E, K)
            assert torch.equal(traced(x, idx, w), fn(x, idx, w))


def test_a_negated_view():
    """Hidden states that torch holds as the negative of their memory."""
    print("few: negated view", flush=True)
    T, H, E, K, I = 5, 128, 8, 2, 64
    x, wr, w1, w2 = _layer(_gen(74), T, H, E, I, F32)
    idx, w = _routing(_gen(75), T, E, K)
    assert x._neg_view().is_neg() and x._neg_view().is_contiguous()
    assert torch.equal(few.experts_forward_few(x._neg_view(), idx, w, w1, w2),
                       few.experts_forward_few(-x, idx, w, w1, w2))
    assert torch.equal(few.moe_layer_few(x._neg_view(), wr, w1, w2, K),
                       few.moe_layer_few(-x, wr, w1, w2, K))


@pytest.mark.parametrize("router", ["softmax", "sigmoid"])
def test_a_router_weight_of_any_alignment(router):
    """As moe_layer's gating product takes it, a slice of a flat buffer say."""
    print(f"few: unaligned router weight {router}", flush=True)
    T, H, E, K, I = 5, 128, 8, 2, 64
    x, wr, w1, w2 = _layer(_gen(76), T, H, E, I, BF)
    flat = torch.empty(E * H + 3, device=DEV, dtype=BF)
    odd = flat[3:].view(E, H).copy_(wr)
    assert odd.is_contiguous() and odd.data_ptr() % 16
    for a, b in zip(few.moe_layer_few(x, odd, w1, w2, K, router=router, return_routing=True),
                    few.moe_layer_few(x, wr, w1, w2, K, router=router, return_routing=True)):
        assert torch.equal(a, b)
    assert moe_layer(x, odd, w1, w2, K, router=router)[0].shape == x.shape
