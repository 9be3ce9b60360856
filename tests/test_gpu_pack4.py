"""Weights in 4 bits: pack4 and unpack4 against the definition, every value equal."""
from __future__ import annotations

import pytest
import torch

from moe_amd import library, ops  # noqa: F401
from pack4_oracle import MAGNITUDES, held, tiles

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _check(w, packed=None):
    p = packed or ops.pack4(w)
    ref = held(w)
    torch.testing.assert_close(tiles(p.q, p.scale, p.shape), ref, rtol=0, atol=0, equal_nan=True)
    back = ops.unpack4(p)
    assert back.shape == w.shape and back.dtype == p.dtype
    torch.testing.assert_close(back.double().cpu(), ref, rtol=0, atol=0, equal_nan=True)
    return p


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("shape", [(16, 128), (1, 1), (1, 31), (3, 33), (16, 127), (17, 129),
                                   (37, 1000), (250, 64), (2, 3, 20, 40), (5, 48, 192),
                                   (3, 2048, 17), (1, 7, 5000)])
def test_values(dt, shape):
    g = torch.Generator(device=DEV).manual_seed(1)
    w = torch.randn(shape, generator=g, device=DEV)
    w *= torch.exp2(torch.randint(-20, 20, (*shape[:-1], 1), generator=g, device=DEV).float())
    _check(w.to(dt))


@pytest.mark.parametrize("dt", [BF, F32])
def test_borders(dt):
    """Halves of every step, the limits of a scale, signs, and values a step off."""
    rows = []
    for top in (4.0, 6.0, 7.0, 7.03125, 7.97, 3.5, 3.515625):
        for k in (-126, -124, -20, 0, 60, 120):
            b = torch.tensor([0.0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2490234375, 0.251953125,
                              0.74609375, 0.75390625, 1.2421875, 1.2578125, 2.484375, 2.515625,
                              3.484375, 3.515625, 4.96875, 5.03125, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0,
                              6.0, 6.96875, 1e-3, 0.126, top], dtype=torch.float64).clamp(max=top)
            sign = torch.where(torch.arange(32) % 3 == 0, -1.0, 1.0)
            rows.append(b * sign * 2.0 ** k)
    w = torch.stack(rows)
    w = w[w.abs().amax(-1) < 1.5 * 2.0 ** 127]
    _check(w.to(dt).to(DEV))


def test_small_and_large():
    tiny = torch.tensor([2.0 ** -149, 2.0 ** -130, 2.0 ** -127, 1.5 * 2.0 ** -127, 2.0 ** -126,
                         -2.0 ** -128, 2.0 ** -125, 0.0] * 4)
    w = torch.stack([tiny, tiny * 0, tiny.clamp(max=2.0 ** -127)]).to(DEV)
    _check(w)
    _check(w.to(BF))
    big = torch.full((2, 32), 1.5 * 2.0 ** 127, device=DEV)   # 6 steps of 2^125
    _check(big)
    _check(big.to(BF))
    most = torch.full((1, 32), torch.finfo(F32).max, device=DEV)
    assert torch.isinf(ops.unpack4(ops.pack4(most))).all()


@pytest.mark.parametrize("dt", [BF, F32])
def test_not_finite(dt):
    w = torch.ones(40, 300, device=DEV, dtype=dt)
    w[3, 40], w[17, 299], w[39, 0] = torch.inf, torch.nan, -torch.inf
    p = _check(w)
    nan = torch.isnan(ops.unpack4(p))
    assert nan[3, 32:64].all() and nan[17, 288:].all() and nan[39, :32].all()
    assert int(nan.sum()) == 32 + 12 + 32


@pytest.mark.parametrize("dt", [BF, F32])
def test_every_code_and_scale(dt):
    """unpack4 of all codes under all scale bytes."""
    q = torch.arange(256, device=DEV, dtype=torch.uint8).repeat(16 * 4)
    scale = torch.arange(16 * 64, device=DEV).to(torch.uint8)
    p = ops.Packed4(q.view(16, 1, 1, 1024), scale.view(16, 1, 1, 64), (16, 16, 128), dt)
    ref = tiles(p.q, p.scale, p.shape)
    ref[ref.abs() >= 2.0 ** 128] *= torch.inf
    torch.testing.assert_close(ops.unpack4(p).double().cpu(), ref, rtol=0, atol=0, equal_nan=True)
    assert len(MAGNITUDES) == 8


def test_padding_is_zero():
    p = ops.pack4(torch.ones(2, 17, 130, device=DEV))
    whole = tiles(p.q, p.scale, (2, 32, 256))
    assert (whole[:, :17, :130] == 1).all()
    whole[:, :17, :130] = 0
    assert (whole == 0).all()


def test_strides_alignment_and_dtype():
    g = torch.Generator(device=DEV).manual_seed(2)
    base = torch.randn(70, 261, generator=g, device=DEV)
    _check(base.t())
    _check(base[::2, 1:200])
    for dt in (BF, F32):
        flat = base.to(dt).reshape(-1)
        _check(flat[1:1 + 40 * 256].view(40, 256))       # not aligned to 16 bytes
    p = ops.pack4(base, dtype=BF)
    assert p.dtype == BF
    _check(base, p)


@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0, 4, 4), (2, 0, 64)])
def test_empty(shape):
    p = ops.pack4(torch.zeros(shape, device=DEV))
    assert ops.unpack4(p).shape == shape


def test_stream_graph_and_ops():
    g = torch.Generator(device=DEV).manual_seed(3)
    w = torch.randn(3, 96, 320, generator=g, device=DEV, dtype=BF)
    ref = held(w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        back = ops.unpack4(ops.pack4(w))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            again = ops.unpack4(ops.pack4(w))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(back.double().cpu(), ref)
    for k in range(3):
        w.copy_(torch.randn(w.shape, generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again.double().cpu(), held(w)), k
    q, scale = torch.ops.moe_amd.pack4(w)
    assert torch.equal(torch.ops.moe_amd.unpack4(q, scale, 96, 320, BF).double().cpu(), held(w))
    torch.library.opcheck(torch.ops.moe_amd.pack4.default, (w,))
    torch.library.opcheck(torch.ops.moe_amd.unpack4.default, (q, scale, 96, 320, BF))
