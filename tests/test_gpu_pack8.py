"""8-bit activations: pack8 / unpack8 against their definition (exact
arithmetic in fp64, so equality), the two GEMMs that keep gate_up in 8 bits
against the ones that keep it in bf16, and the layers' gradients
against the formulas in 64 bits and against differences."""
from __future__ import annotations

import pytest
import torch

from moe_amd import experts_forward, hf, ops
from moe_amd.layer import SparseMoeBlock, moe_layer

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
U, V = 2.0 ** -8, 2.0 ** -24   # half a step of bf16 and of fp32, relative


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _reference(x):
    """(q, exponent of s) in fp64: the smallest k >= -126 with max|v| <= 127 * 2^k."""
    v = x.double()
    n = v.shape[-1]
    b = torch.nn.functional.pad(v, (0, -n % 64)).unflatten(-1, (-1, 64))
    a = b.abs().amax(-1)
    k = torch.full_like(a, -126)
    for e in range(-126, 123):   # 127 * 2^k is exact in fp64
        k = torch.where(a > 127 * 2.0 ** e, e + 1, k)
    q = torch.round(b / torch.exp2(k)[..., None])
    return q.flatten(-2)[..., :n], k


def _restored(x):
    q, k = _reference(x)
    return q * torch.exp2(k).repeat_interleave(64, -1)[..., :q.shape[-1]]


def _check(x):
    p = ops.pack8(x)
    q, k = _reference(x)
    assert p.q.shape == x.shape and p.dtype == x.dtype
    assert torch.equal(p.q.double(), q)
    assert torch.equal(p.scale.double(), k + 127)
    back = ops.unpack8(p)
    assert back.dtype == x.dtype
    # Every q s but one is representable: |q| <= 127 has 7 bits and s >= 2^-126.
    # The one is 64 * 2^122 = 2^128, for |v| > 127/128 * 2^128 (there s = 2^122 and
    # 63.5 < |v| / s < 64), which the type rounds to infinity.
    assert torch.equal(back, _restored(x).to(x.dtype))
    # half a step of the block's scale
    err = (back.double() - x.double()).abs()
    s = torch.exp2(k).repeat_interleave(64, -1)[..., :x.shape[-1]]
    assert (err <= s / 2)[back.isfinite()].all()
    assert (x.double().abs()[~back.isfinite()] > 127 / 128 * 2.0 ** 128).all()


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [(1,), (63,), (64,), (65,), (1, 1), (3, 64), (7, 100), (2, 3, 130),
                                   (129, 2048), (1000, 7), (1, 100000), (517, 1536), (0, 64), (5, 0)])
def test_shapes(shape, dt):
    print(f"pack8 {shape} {dt}", flush=True)
    x = torch.randn(shape, generator=_gen(sum(shape)), device=DEV).to(dt)
    if x.numel() == 0:
        p = ops.pack8(x)
        assert p.q.shape == x.shape and ops.unpack8(p).shape == x.shape
        return
    _check(x)


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
def test_values(dt):
    """Every magnitude from subnormals to the largest, zeros, halves, and blocks
    whose maximum lies next to 127 * 2^k."""
    print(f"pack8 values {dt}", flush=True)
    g = _gen(1)
    x = torch.randn(400, 64, generator=g, device=DEV)
    x *= torch.exp2(torch.linspace(-149, 124, 400, device=DEV).round())[:, None]
    _check(x.to(dt))
    assert (ops.unpack8(ops.pack8(torch.zeros(3, 70, device=DEV, dtype=dt))) == 0).all()
    info = torch.finfo(dt)
    edges = [127.0, 126.5, 127.0 * (1 + info.eps), 127.5, 128.0, 64.0, 63.75, 1.984375,
             1.984375 * (1 + info.eps), info.max, info.tiny, info.tiny / 2, info.smallest_normal]
    rows = torch.zeros(2 * len(edges), 64, device=DEV, dtype=F32)
    for i, e in enumerate(edges):
        rows[2 * i, 17] = e
        rows[2 * i + 1, 63] = -e
        rows[2 * i:2 * i + 2, 5] = e / 3
    _check(rows.to(dt))
    # halves go to the even integer
    h = torch.arange(-63, 64, device=DEV, dtype=F32)[:63] + 0.5
    block = torch.cat([h, torch.tensor([100.0], device=DEV)]).to(dt)
    assert torch.equal(ops.pack8(block).q[:63].double(), torch.round(block[:63].double()))
    _check(block)


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
def test_blocks_that_are_not_finite(dt):
    print(f"pack8 not finite {dt}", flush=True)
    x = torch.randn(4, 200, generator=_gen(2), device=DEV).to(dt)
    clean = ops.unpack8(ops.pack8(x))
    x[0, 3], x[1, 199], x[2, 64] = float("nan"), float("inf"), float("-inf")
    got = ops.unpack8(ops.pack8(x))
    bad = torch.zeros(4, 200, dtype=torch.bool, device=DEV)
    bad[0, :64] = bad[1, 192:] = bad[2, 64:128] = True
    assert got[bad].isnan().all()
    assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("shape", [(4, 128), (3, 100)], ids=["whole", "ragged"])
@pytest.mark.parametrize("bits", [0x7fc00001, 0x7fc000ff, 0xffffffff, 0x7f800001, 0xff80007f,
                                  0x7f800000])
def test_any_nan_makes_the_block_nan(bits, shape):
    """A NaN's payload stays out of q: every q of its block is 0, every value NaN."""
    print(f"pack8 NaN {bits:#x} {shape}", flush=True)
    x = torch.randn(shape, generator=_gen(7), device=DEV)
    clean = ops.pack8(x)
    raw = x.view(torch.int32)
    raw[0, 5] = raw[2, 64] = raw[2, 99] = bits - (1 << 32 if bits >> 31 else 0)
    p = ops.pack8(x)
    bad = torch.zeros(shape, dtype=torch.bool, device=DEV)
    bad[0, :64] = bad[2, 64:128] = True
    assert p.scale[0, 0] == p.scale[2, 1] == 255
    assert (p.q[bad] == 0).all() and torch.equal(p.q[~bad], clean.q[~bad])
    back = ops.unpack8(p)
    assert back[bad].isnan().all() and back[~bad].isfinite().all()


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
def test_strides_and_alignment(dt):
    print(f"pack8 strides {dt}", flush=True)
    x = torch.randn(33, 300, generator=_gen(3), device=DEV).to(dt)
    for view in (x[:, 1:65], x[::2, ::3], x.t(), x[5:], x[:, :256]):
        _check(view)
    flat = torch.randn(64 * 33 + 1, generator=_gen(4), device=DEV).to(dt)
    _check(flat[1:].view(33, 64))      # contiguous, off the vectors' alignment
    assert torch.equal(ops.unpack8(ops.pack8(flat[1:].view(33, 64))),
                       ops.unpack8(ops.pack8(flat[1:].clone().view(33, 64))))
    p = ops.pack8(x)
    odd = torch.empty(p.q.numel() + 1, device=DEV, dtype=torch.int8)
    odd[1:] = p.q.reshape(-1)
    assert torch.equal(ops.unpack8(ops.Packed8(odd[1:].view(p.q.shape), p.scale, dt)),
                       ops.unpack8(p))


def test_more_values_than_32_bits_count():
    print("pack8 large", flush=True)
    rows, cols = 33000, 65600            # 2.16e9 values
    x = torch.empty(rows, cols, device=DEV, dtype=BF)
    x[:] = torch.randn(1, cols, generator=_gen(5), device=DEV).to(BF)
    x[-1] = torch.randn(cols, generator=_gen(6), device=DEV).to(BF) * 3
    p = ops.pack8(x)
    back = ops.unpack8(p)
    assert torch.equal(back[-1].double(), _restored(x[-1]))
    assert torch.equal(back[:-1], back[:1].expand(rows - 1, cols))
    assert torch.equal(back[0].double(), _restored(x[0]))


def test_streams_and_graph():
    print("pack8 streams", flush=True)
    x = torch.randn(300, 1000, generator=_gen(7), device=DEV).to(BF)
    want = ops.unpack8(ops.pack8(x))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ops.unpack8(ops.pack8(x))
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.unpack8(ops.pack8(held))
    for i in range(3):
        held.copy_(torch.randn(300, 1000, generator=_gen(8 + i), device=DEV).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.unpack8(ops.pack8(held)))


def test_refusals_on_the_gpu():
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.pack8(torch.zeros(4, 64, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError, match="at least one dimension"):
        ops.pack8(torch.tensor(1.0, device=DEV))
    p = ops.pack8(torch.zeros(4, 70, device=DEV))
    for bad in (ops.Packed8(p.q, p.scale[:, :1], F32), ops.Packed8(p.q.view(torch.uint8), p.scale, F32),
                ops.Packed8(p.q[:3], p.scale, F32), ops.Packed8(p.q, p.scale.cpu(), F32)):
        with pytest.raises((ValueError, RuntimeError), match="not a packed tensor|GPU only"):
            ops.unpack8(bad)


# --------------------------------------------------------- the fused GEMMs

def _layer(seed, T, H, E, K, I, skew=0.0, wdt=F32):
    g = _gen(seed)
    x = torch.randn(T, H, generator=g, device=DEV).to(BF)
    w1 = (torch.randn(E, 2 * I, H, generator=g, device=DEV) * 0.05).to(BF)
    w2 = (torch.randn(E, H, I, generator=g, device=DEV) * 0.05).to(BF)
    logits = torch.randn(T, E, generator=g, device=DEV)
    if skew:
        logits[:, :2] += skew
    w, idx = torch.softmax(logits, -1).topk(K, dim=-1)
    dout = torch.randn(T, H, generator=g, device=DEV).to(BF)
    return x, idx, w.to(wdt), w1, w2, dout


def _split(q, S, I):
    """(gate_up q int8 [S,2I], scale bytes [S,2I/64]) from the packed buffer."""
    v = q[:S * 2 * I].view(torch.int8).view(S, I // 8, 2, 8)
    s = q[S * 2 * I:].view(S, I // 64, 2)
    return (torch.cat([v[:, :, 0].reshape(S, I), v[:, :, 1].reshape(S, I)], 1),
            torch.cat([s[:, :, 0], s[:, :, 1]], 1))


GEMMS = [  # T, H, E, K, I, skew: rows per expert choose the tile heights of 64, 128 and 256
    (1, 64, 4, 2, 64, 0), (37, 128, 8, 3, 192, 0), (300, 256, 16, 4, 320, 0), (515, 192, 2, 2, 832, 0),
    (700, 128, 8, 2, 768, 4.0), (1111, 256, 2, 2, 128, 0),
]


@pytest.mark.parametrize("T,H,E,K,I,skew", GEMMS)
def test_gemms_keep_gate_up_in_8_bits(T, H, E, K, I, skew):
    print(f"pack8 gemms {T} {H} {E} {K} {I}", flush=True)
    x, idx, w, w1, w2, dout = _layer(T, T, H, E, K, I, skew)
    idx[::7, 0] = E     # sentinels: rows behind the last expert's
    plan = ops.permute(idx, E)
    S, n = T * K, int(plan.offsets[E])
    gu, act = ops.gemm_gate_up_swiglu(x, plan, w1)
    q, act8 = ops.gemm_gate_up_swiglu(x, plan, w1, pack8=True)
    assert torch.equal(act8[:n], act[:n])
    got_q, got_s = _split(q, S, I)
    p = ops.pack8(gu[:n])
    assert torch.equal(got_q[:n], p.q) and torch.equal(got_s[:n], p.scale)
    restored = torch.zeros_like(gu)
    restored[:n] = ops.unpack8(p)
    for wd in (w, w.to(BF)):
        want = ops.gemm_down_backward_fused(dout, plan, w2, restored, wd)
        have = ops.gemm_down_backward_fused(dout, plan, w2, q, wd)
        # the same products: d_gate_up and w * act with one rounding here, three
        # there; the weight's gradient, a sum of g * act, with act's two there
        for a, b, rows in zip(have[:2], want[:2], (n, n)):
            a, b = a[:rows].double(), b[:rows].double()
            assert ((a - b).abs() <= 4.05 * U * b.abs()).all()
        y = ops.gemm_down_backward_fused(dout.abs(), plan, w2.abs(), restored.abs(), wd)[2]
        uw = torch.finfo(wd.dtype).eps / 2
        assert ((have[2] - want[2]).double().abs()
                <= (2.05 * U * y.double() + 2 * uw * want[2].double().abs())).all()


def test_sentinel_rows_are_left_alone():
    from moe_amd import _lib
    print("pack8 gemm sentinels", flush=True)
    T, H, E, K, I = 90, 128, 4, 2, 128
    x, idx, w, w1, w2, dout = _layer(3, T, H, E, K, I)
    idx[::3] = E + 1
    plan = ops.permute(idx, E)
    S, n = T * K, int(plan.offsets[E])
    q = torch.full((S, 2 * I), 0x5A, device=DEV, dtype=torch.uint8)
    s = torch.full((S, I // 32), 0x5A, device=DEV, dtype=torch.uint8)
    act = torch.full((S, I), 7.0, device=DEV, dtype=BF)
    _lib.call("moe_amd_gemm_gate_up_swiglu_pack8", x.data_ptr(), plan.row_src.data_ptr(), K,
              plan.offsets.data_ptr(), plan.tile_plan.data_ptr(), w1.data_ptr(), T, S, E, H, I, 1,
              q.data_ptr(), s.data_ptr(), act.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (q[n:] == 0x5A).all() and (s[n:] == 0x5A).all() and (act[n:] == 7).all()
    assert (s[:n] != 0x5A).all()       # exponents near 2^-6, not 2^-37


def test_not_finite_gate_up_is_not_hidden():
    print("pack8 gemm not finite", flush=True)
    T, H, E, K, I = 40, 128, 4, 2, 128
    x, idx, w, w1, w2, dout = _layer(4, T, H, E, K, I)
    leaf = x.clone().requires_grad_(True)
    want = torch.autograd.grad(experts_forward(leaf, idx, w, w1, w2, "int8"), leaf, dout)[0]
    leaf.data[11, 5] = float("inf")
    got = torch.autograd.grad(experts_forward(leaf, idx, w, w1, w2, "int8"), leaf, dout)[0]
    others = torch.arange(T, device=DEV) != 11
    assert torch.equal(got[others], want[others]) and got[11].isnan().all()


# --------------------------------------------------------------- the layers

def _grads(fn, tensors, dout):
    leaves = [t.detach().clone().requires_grad_(True) for t in tensors]
    out = fn(*leaves)
    return (out.detach(),) + torch.autograd.grad(out, leaves, dout)


def _formula(x, idx, w, w1, w2, dout, keep):
    """{name: (value, bound)} in 64 bits.  Roundings to bf16 on the way, each
    U relative: d_gate, d_up and w act one, d_x's rows one and itself one, every
    gradient its own; sums of n products n V relative to the
    sum of their magnitudes; the sigmoid's hardware exp and reciprocal 8 V."""
    T, H = x.shape
    E, I, K = w1.shape[0], w2.shape[2], idx.shape[1]
    plan = ops.permute(idx, E)
    gu, _ = ops.gemm_gate_up_swiglu(x, plan, w1)
    gu = _restored(gu)[plan.slot.long()]        # by token and k
    xk = _restored(x) if keep == "int8_all" else x.double()
    dx, tx = torch.zeros(2, T, H, device=DEV, dtype=torch.float64)
    dw, tw = torch.zeros(2, T, K, device=DEV, dtype=torch.float64)
    d1, t1 = torch.zeros(2, *w1.shape, device=DEV, dtype=torch.float64)
    d2, t2 = torch.zeros(2, *w2.shape, device=DEV, dtype=torch.float64)
    for e in range(E):
        t, k = torch.nonzero(idx == e, as_tuple=True)
        n = len(t)
        m1, m2, do = w1[e].double(), w2[e].double(), dout[t].double()
        wk = w[t, k].double()[:, None]
        gate, up = gu[t * K + k].split(I, 1)
        sig = torch.sigmoid(gate)
        act, dsig = gate * sig * up, sig * (1 + gate * (1 - sig))
        g, tg = do @ m2, H * V * (do.abs() @ m2.abs())
        dgu = torch.cat([g * wk * up * dsig, g * wk * gate * sig], 1)
        # relative to (1 + |gate|) sig: dsig itself may cancel
        mag = torch.cat([g.abs() * wk * up.abs() * sig * (1 + gate.abs()), dgu[:, I:].abs()], 1)
        tgu = 1.01 * U * dgu.abs() + 16 * V * mag + torch.cat(
            [tg * wk * (up * dsig).abs(), tg * wk * (gate * sig).abs()], 1)
        rows = dgu @ m1
        trows = tgu @ m1.abs() + 2 * I * V * (dgu.abs() @ m1.abs())
        dx.index_add_(0, t, rows)
        tx.index_add_(0, t, trows + U * (rows.abs() + trows))
        dw[t, k] = (g * act).sum(1)
        tw[t, k] = (((I + 16) * V) * (g * act).abs() + tg * act.abs()).sum(1)
        d1[e] = dgu.t() @ xk[t]
        t1[e] = tgu.t() @ xk[t].abs() + n * V * (dgu.abs().t() @ xk[t].abs())
        aw = act * wk
        d2[e] = do.t() @ aw
        t2[e] = (1.01 * U + (n + 16) * V) * (do.abs().t() @ aw.abs())
    tx = tx + K * V * dx.abs()
    res = {"dx": (dx, tx + U * (dx.abs() + tx)), "dw1": (d1, t1 + U * (d1.abs() + t1)),
           "dw2": (d2, t2 + U * (d2.abs() + t2))}
    uw = torch.finfo(w.dtype).eps / 2
    res["dw"] = (dw, tw + uw * (dw.abs() + tw))
    return res


@pytest.mark.parametrize("keep", ["int8", "int8_all"])
@pytest.mark.parametrize("T,H,E,K,I,wdt", [(1, 64, 2, 1, 64, F32), (45, 128, 6, 3, 192, BF),
                                          (200, 256, 8, 2, 128, F32), (611, 128, 2, 2, 64, BF)])
def test_gradients_against_the_formulas(T, H, E, K, I, wdt, keep):
    print(f"int8 gradients {T} {H} {E} {K} {I} {keep}", flush=True)
    x, idx, w, w1, w2, dout = _layer(T + 1, T, H, E, K, I, wdt=wdt)
    ref = _formula(x, idx, w, w1, w2, dout, keep)
    out, dx, dw, d1, d2 = _grads(lambda *a: experts_forward(a[0], idx, *a[1:], keep),
                                 (x, w, w1, w2), dout)
    assert torch.equal(out, experts_forward(x, idx, w, w1, w2))
    for name, got in (("dx", dx), ("dw", dw), ("dw1", d1), ("dw2", d2)):
        val, tol = ref[name]
        over = ((got.double() - val).abs() / tol.clamp(min=1e-300)).max()
        assert ((got.double() - val).abs() <= tol).all(), f"{name}: {float(over):.2f} bounds"


def test_gradients_against_differences():
    """Inputs whose gate_up the 8 bits hold exactly: x one-hot, gate_up
    multiples of 1/32 with 64 <= 32 max < 128 in every block.  Then the gradient
    is the function's own, and a central difference in 64 bits along a direction
    (truncation below 1e-6 of it at h = 1e-4) shows it to the bf16 roundings: at
    most seven on the way to a gradient, 7 U of the sum of the products' sizes."""
    print("int8 differences", flush=True)
    T, H, E, K, I = 48, 64, 3, 2, 128
    g = _gen(9)
    x = torch.nn.functional.one_hot(torch.arange(T, device=DEV) % H, H).to(BF)
    k = torch.randint(-40, 41, (E, 2 * I, H), generator=g, device=DEV)
    k[:, ::64] = torch.randint(64, 128, (E, 2 * I // 64, H), generator=g, device=DEV)
    w1 = (k.float() / 32).to(BF)
    w2 = (torch.randn(E, H, I, generator=g, device=DEV) * 0.1).to(BF)
    idx = torch.rand(T, E, generator=g, device=DEV).argsort(1)[:, :K].contiguous()
    w = torch.rand(T, K, generator=g, device=DEV).to(BF)
    dout = torch.randn(T, H, generator=g, device=DEV).to(BF)
    _, dx, dw, d1, d2 = _grads(lambda *a: experts_forward(a[0], idx, *a[1:], "int8"),
                               (x, w, w1, w2), dout)

    def f(x, w, w1, w2):
        gu = torch.einsum("th,tknh->tkn", x, w1[idx])
        act = gu[..., :I] * torch.sigmoid(gu[..., :I]) * gu[..., I:]
        y = torch.einsum("tki,tkhi->tkh", act, w2[idx])
        return (y * w[..., None] * dout.double()[:, None]).sum()

    base = [t.double() for t in (x, w, w1, w2)]
    for i, grad in enumerate((dx, dw, d1, d2)):
        v = torch.randn(base[i].shape, generator=g, device=DEV, dtype=torch.float64)
        hi = [b + 1e-4 * v if j == i else b for j, b in enumerate(base)]
        lo = [b - 1e-4 * v if j == i else b for j, b in enumerate(base)]
        num = (f(*hi) - f(*lo)) / 2e-4
        have = (grad.double() * v).sum()
        assert (have - num).abs() <= 7 * U * (grad.double() * v).abs().sum() + 1e-6 * num.abs()


@pytest.mark.parametrize("keep", ["int8", "int8_all"])
def test_one_node_layer_and_its_parts(keep):
    """The softmax layer's one node against the same kernels called apart."""
    print(f"int8 layer {keep}", flush=True)
    T, H, E, K, I = 333, 256, 16, 4, 192
    x, _, _, w1, w2, dout = _layer(21, T, H, E, K, I)
    wr = (torch.randn(E, H, generator=_gen(22), device=DEV) * 0.05).to(BF)
    fn = lambda x, wr, w1, w2, **kw: moe_layer(x, wr, w1, w2, K, gating="hip", **kw)[0]  # noqa: E731
    out, dx, dr, d1, d2 = _grads(lambda *a: fn(*a, saved_activations=keep), (x, wr, w1, w2), dout)
    out0, dx0, dr0, d10, d20 = _grads(fn, (x, wr, w1, w2), dout)
    assert torch.equal(out, out0)
    logits = ops.router_linear(x, wr)
    probs, w, idx = ops.router_softmax_topk(logits, K)
    plan = ops.permute(idx, E)
    gu8, _ = ops.gemm_gate_up_swiglu(x, plan, w1, pack8=True)
    xk = ops.unpack8(ops.pack8(x)) if keep == "int8_all" else x
    dgu, aw, dw = ops.gemm_down_backward_fused(dout, plan, w2, gu8, w)
    dl = ops.router_softmax_topk_backward(probs, idx, dw, None, True, BF)
    rows = ops.gemm_gate_up_backward_dx(dgu, plan, w1)
    assert torch.equal(dx, ops.gather_backward(rows, plan, ops.router_linear_backward_dx(dl, wr)))
    assert torch.equal(dr, ops.router_linear_backward_dw(dl, xk))
    assert torch.equal(d1, ops.gemm_gate_up_backward_dw(dgu, xk, plan, w1.shape))
    assert torch.equal(d2, ops.gemm_down_backward_dw_gathered(dout, aw, plan, w2.shape))
    # a step is at most 2/64 of its block's maximum, so half a step 1/64 of it; the
    # gradients move with it, not by more than that share of their own size
    for a, b in ((dx, dx0), (d1, d10), (d2, d20)):
        assert (a.double() - b.double()).norm() / b.double().norm() <= 1 / 64 + 4 * U


def test_main_grad_and_frozen_parts():
    print("int8 main_grad", flush=True)
    T, H, E, K, I = 256, 128, 8, 2, 128
    x, idx, w, w1, w2, dout = _layer(31, T, H, E, K, I)
    _, _, _, d1, d2 = _grads(lambda *a: experts_forward(a[0], idx, *a[1:], "int8_all"),
                             (x, w, w1, w2), dout)
    p1, p2 = (t.clone().requires_grad_(True) for t in (w1, w2))
    p1.main_grad, p2.main_grad = torch.zeros_like(w1), torch.zeros_like(w2)
    experts_forward(x, idx, w, p1, p2, "int8_all").backward(dout)
    assert p1.grad is None and torch.equal(p1.main_grad, d1) and torch.equal(p2.main_grad, d2)
    # weights alone, hidden states alone, and no gradient at all
    q1 = w1.clone().requires_grad_(True)
    experts_forward(x, idx, w, q1, w2, "int8_all").backward(dout)
    assert torch.equal(q1.grad, d1)
    leaf = x.clone().requires_grad_(True)
    a = torch.autograd.grad(experts_forward(leaf, idx, w, w1, w2, "int8"), leaf, dout)[0]
    b = torch.autograd.grad(experts_forward(leaf, idx, w, w1, w2, "int8_all"), leaf, dout)[0]
    assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(experts_forward(x, idx, w, w1, w2, "int8"),
                           experts_forward(x, idx, w, w1, w2))


def test_no_tokens():
    x, idx, w, w1, w2, dout = _layer(5, 4, 64, 2, 1, 64)
    leaf = x[:0].clone().requires_grad_(True)
    out = experts_forward(leaf, idx[:0], w[:0], w1, w2, "int8_all")
    assert torch.autograd.grad(out, leaf, dout[:0])[0].shape == (0, 64)


def _saved_bytes(fn):
    seen = {}

    def note(t):
        seen[t.data_ptr()] = t.nbytes
        return t

    with torch.autograd.graph.saved_tensors_hooks(note, lambda t: t):
        out = fn()
    del out
    return sum(seen.values())


def test_memory_kept():
    print("int8 memory", flush=True)
    T, H, E, K, I = 512, 256, 4, 4, 256
    x, idx, w, w1, w2, _ = _layer(41, T, H, E, K, I)
    x.requires_grad_(True)
    size = {k: _saved_bytes(lambda: experts_forward(x, idx, w, w1, w2, k))
            for k in ("exact", "int8", "int8_all")}
    gu, xs = T * K * 2 * I * 2, T * H * 2
    assert size["exact"] - size["int8"] == gu - gu * 65 // 128
    assert size["int8"] - size["int8_all"] == xs - xs * 65 // 128


def test_block_and_hf_model_train_with_it():
    print("int8 hf", flush=True)
    torch.manual_seed(0)
    blk = SparseMoeBlock(128, 4, 2, 64).to(DEV, BF)
    with torch.no_grad():
        for p in blk.parameters():
            p.normal_(0, 0.1)
    h = torch.randn(3, 5, 128, device=DEV, dtype=BF)
    grads = []
    for keep in ("exact", "int8"):
        blk.saved_activations = keep
        blk.zero_grad()
        blk(h).float().square().sum().backward()
        grads.append([p.grad.double() for p in blk.parameters()])
    for a, b in zip(*grads):
        assert (a - b).norm() <= (1 / 64 + 4 * U) * a.norm() and not torch.equal(a, b)

    from transformers import Qwen3MoeConfig, Qwen3MoeForCausalLM
    cfg = Qwen3MoeConfig(vocab_size=64, hidden_size=128, intermediate_size=128,
                         moe_intermediate_size=64, num_hidden_layers=2, num_attention_heads=2,
                         num_key_value_heads=1, head_dim=64, num_experts=8,
                         num_experts_per_tok=2, norm_topk_prob=True, decoder_sparse_step=1,
                         max_position_embeddings=64)
    m = Qwen3MoeForCausalLM(cfg).to(DEV, BF)
    ids = torch.randint(0, 64, (2, 16), device=DEV)
    hf.install(m)
    loss = m(ids, labels=ids).loss
    hf.install(m, saved_activations="int8")
    assert all(b.saved_activations == "int8" for b in hf.expert_banks(m))
    loss8 = m(ids, labels=ids).loss
    assert torch.equal(loss, loss8)     # the forward is the same
    loss8.backward()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters() if p.grad is not None)


@pytest.mark.parametrize("keep", ["int8", "int8_all"])
def test_compiled_and_opcheck(keep):
    print(f"int8 compile {keep}", flush=True)
    T, H, E, K, I = 64, 128, 4, 2, 64
    x, idx, w, w1, w2, dout = _layer(51, T, H, E, K, I)
    fn = lambda *a: experts_forward(a[0], idx, *a[1:], keep)  # noqa: E731
    eager = _grads(fn, (x, w, w1, w2), dout)
    compiled = _grads(torch.compile(fn, fullgraph=True, backend="aot_eager"), (x, w, w1, w2), dout)
    assert all(torch.equal(a, b) for a, b in zip(eager, compiled))
    utils = ("test_schema", "test_faketensor", "test_autograd_registration")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, w1, w2)]
    torch.library.opcheck(torch.ops.moe_amd.experts_fwd.default,
                          (leaves[0], idx, *leaves[1:], True, keep), test_utils=utils)
    torch.library.opcheck(torch.ops.moe_amd.pack8.default, (x,), test_utils=utils[:2])
    q, s = torch.ops.moe_amd.pack8(x)
    torch.library.opcheck(torch.ops.moe_amd.unpack8.default, (q, s, BF), test_utils=utils[:2])


def test_wrong_packed_gate_up_is_refused():
    T, H, E, K, I = 8, 64, 2, 1, 64
    x, idx, w, w1, w2, dout = _layer(61, T, H, E, K, I)
    plan = ops.permute(idx, E)
    q, _ = ops.gemm_gate_up_swiglu(x, plan, w1, pack8=True)
    with pytest.raises(ValueError, match="packed gate_up"):
        ops.gemm_down_backward_fused(dout, plan, w2, q[:-1], w)
