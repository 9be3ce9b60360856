"""Weights in 4 bits from the definition, in 64 bits on the CPU: what a block
holds, and the weight that tiles hold, place by place."""
from __future__ import annotations

import torch

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def held(w: torch.Tensor) -> torch.Tensor:
    """The values that w [..., K] has once packed, 64 bits."""
    v = w.double().cpu()
    out = torch.empty_like(v)
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64)
    for j in range(0, v.shape[-1], 32):
        b = v[..., j:j + 32]
        a = b.abs().amax(-1, keepdim=True)
        s = torch.full_like(a, 2.0 ** -125)
        for _ in range(260):  # the smallest power of two that will do
            s = torch.where(a > 7 * s, 2 * s, s)
        u = (b.abs() / s).clamp(max=6)
        up = (u[..., None] > grid).sum(-1)          # the first magnitude >= u
        lo = (up - 1).clamp(min=0)
        closer = grid[up] - u - (u - grid[lo])      # negative: the upper one is nearer
        code = torch.where((closer < 0) | ((closer == 0) & (up % 2 == 0)), up, lo)
        r = torch.copysign(grid[code] * s, b)
        out[..., j:j + 32] = torch.where(torch.isfinite(b).all(-1, keepdim=True), r, torch.nan)
    return out


def tiles(q: torch.Tensor, scale: torch.Tensor, shape) -> torch.Tensor:
    """The weight [..., N, K] of tiles, 64 bits; a scale byte of 255 is NaN."""
    q, scale = q.cpu(), scale.cpu()
    N, K = shape[-2:]
    r, c = torch.arange(N)[:, None], torch.arange(K)[None, :]
    byte = q[..., r // 16, c // 128, c % 128 // 32 * 256 + r % 16 * 16 + c % 32 // 2].long()
    code = torch.where(c % 2 == 0, byte & 15, byte >> 4)
    b = scale[..., r // 16, c // 128, r % 16 * 4 + c % 128 // 32].double()
    s = torch.where(b == 255, torch.nan, torch.exp2(b - 127))
    v = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), dtype=torch.float64)
    return v[code] * s
