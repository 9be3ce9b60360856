"""The expert layer in 64 bits with the roundings that a form of it makes, and how
far that form's outputs may then be from it in the 2-norm.

Tolerance.  Against a reference that makes the form's own rounding of act, an output
differs by its rounding to bf16 and by what the form does in fp32 or finer.  The first
is computed, from the reference itself.  Of the rest, in the 2-norm and relative to the
output: fp32 sums of n products, sqrt(n) 2^-24 each way at most 2^-17 for n up to 2^14,
which also put an act on another side of a border between two bf16 values in one of
2^8 / 2^17 cases or fewer, a step of 2^-7 each: 2^-4.5 2^-7 = 2^-11.5; y in fp16, half a
step of which is 2^-11 of a value and a sixth of it less in the mean square (/ sqrt 3);
y = sum of w y has no smaller 2-norm than its terms'.  These are independent of each
other and of the output's rounding (2^-8 / sqrt 3 of a value that begins a power of two,
1.65e-3 of normal values in the mean): sqrt(1.65e-3^2 + 3.5e-4^2 + 2.8e-4^2) is 1.04 of
it.  A further rounding to bf16 makes it 1.4.  The limit is 1.2.
"""
from __future__ import annotations

import torch

LIMIT = 1.2


def layer(x, idx, w, w1, w2, act_bf16, planted=()):
    """out [T, H] in 64 bits of weights w1 [E, 2I, H], w2 [E, H, I] (a tensor or
    anything that an expert's id indexes); act_bf16: act is rounded.  ``planted``: names of
    what is rounded to bf16 besides: gate_up, silu, act, y, w, wy."""
    def bf(name, v):
        return v.bfloat16().double() if name in planted else v
    out = torch.zeros(x.shape, device=x.device, dtype=torch.float64)
    for e in torch.unique(idx).tolist():
        if not 0 <= e < len(w1):
            continue
        t, k = torch.nonzero(idx == e, as_tuple=True)
        gu = bf("gate_up", x[t].double() @ w1[e].double().t().contiguous())
        gate, up = gu.chunk(2, 1)
        act = bf("act", bf("silu", gate * torch.sigmoid(gate)) * up)
        if act_bf16:
            act = act.bfloat16().double()
        y = bf("y", act @ w2[e].double().t().contiguous())
        out.index_add_(0, t, bf("wy", y * bf("w", w[t, k].double())[:, None]))
    return out


def distance(got, ref):
    """|got - ref| in units of the output's own rounding, in the 2-norm over all values."""
    own = (ref.bfloat16().double() - ref).norm()
    return float((got.double() - ref).norm() / own)
