"""The workloads that expert banks in 4 bits are measured on: their inputs,
their plain forms in elementary torch operations and their values in 64 bits.

  few      the whole MoE layer (router + experts) for a few tokens, its bank in
           4 bits: moe_amd.few.moe_layer_few
  experts  the experts alone for a few tokens, routing given, some entries of it
           padding (ids outside [0, E)): moe_amd.few.experts_forward_few
  prompt   the experts for a whole prompt, products grouped by expert with
           ragged sizes, routing given: moe_amd.experts_forward
  pack     a weight packed to 4 bits and restored: moe_amd.ops.pack4, unpack4

A packed weight w [..., N, K] holds, for 32 consecutive values v of a row (zeros
follow where 32 does not divide K), a power of two s and a code a value: s is the
smallest power of two that is at least 2^-125 and has max|v| <= 7 s, the code
a sign (bit 3) and the magnitude of v / s rounded to 0, 1/2, 1, 3/2, 2, 3, 4
or 6 (bits 0 to 2 count them), halves to the even code.  Codes and scales lie in
tiles of 16 rows by 128 columns (zeros follow where those do not divide N and K):

  q      uint8 [..., N/16, K/128, 1024]: by block of 32 columns, row, two values
         a byte, the first one in its low half
  scale  uint8 [..., N/16, K/128, 64]: by row, block of 32 columns; s = 2^(b-127)

Layer shapes are those of moe_amd/configs.py.
"""
from __future__ import annotations

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One token of one request through the L layer: the latency of a decode step.
        dict(name="few4_l_1", op="few", T=1, H=2048, E=128, K=8, I=768, router="softmax"),
        # A small batch of requests, one token each.
        dict(name="few4_l_13", op="few", T=13, H=2048, E=128, K=8, I=768, router="softmax"),
        # A full decode batch: every expert of the L layer has a few rows.
        dict(name="few4_l_64", op="few", T=64, H=2048, E=128, K=8, I=768, router="softmax"),
        # The global bank of 1792 experts behind the sigmoid router with its selection bias.
        dict(name="few4_retrofit_64", op="few", T=64, H=2048, E=1792, K=8, I=768,
             router="sigmoid"),
        # Experts alone behind a caller's router, one token (XS).
        dict(name="experts4_xs_1", op="experts", T=1, H=1024, E=128, K=4, I=768, skew=0.0,
             pad=0.0),
        # Experts alone, a ragged batch with padded entries and a few popular experts.
        dict(name="experts4_l_37", op="experts", T=37, H=2048, E=128, K=8, I=768, skew=2.0,
             pad=0.15),
        # A short prompt of odd length through the global bank (XS): 16 rows an expert.
        dict(name="prompt4_xs_509", op="prompt", T=509, H=1024, E=128, K=4, I=768, skew=0.0),
        # A prompt through the L layer, 64 rows an expert.
        dict(name="prompt4_l_1021", op="prompt", T=1021, H=2048, E=128, K=8, I=768, skew=0.0),
        # A batch of long prompts with skewed routing: from a few rows to thousands an expert.
        dict(name="prompt4_l_16384", op="prompt", T=16384, H=2048, E=128, K=8, I=768, skew=2.0),
        # A prompt through the global bank of 1792 experts, 9 rows each: its weights are the work.
        dict(name="prompt4_retrofit_2048", op="prompt", T=2048, H=2048, E=1792, K=8, I=768,
             skew=0.0),
        # A weight of odd sizes.
        dict(name="pack4_1021", op="pack", B=1, N=1021, C=1000, dtype="bf16"),
        # Sixteen experts' gate_up_proj, from an fp32 checkpoint.
        dict(name="pack4_bank", op="pack", B=16, N=1536, C=2048, dtype="f32"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["few", "few", "experts", "prompt", "prompt", "pack"])
    if op == "pack":
        return dict(op=op, B=rng.randint(1, 4), N=_spread(rng, 1, 4000), C=_spread(rng, 1, 3000),
                    dtype=rng.choice(["bf16", "f32"]))
    case = dict(op=op, H=64 * rng.randint(4, 32), I=64 * rng.randint(2, 12), K=rng.randint(1, 8))
    if op == "prompt":
        return dict(case, T=_spread(rng, 1, 12000), E=8 * rng.randint(1, 16),
                    skew=rng.choice([0.0, 2.0]))
    case.update(T=_spread(rng, 1, 64), E=8 * rng.randint(2, 64))
    if op == "few":
        return dict(case, router=rng.choice(["softmax", "sigmoid"]))
    return dict(case, skew=rng.choice([0.0, 2.0]), pad=rng.choice([0.0, 0.2]))


def _routing(g, T, E, K, skew):
    """Top-K of random logits, whose largest offsets follow a Zipf law."""
    logits = torch.randn(T, E, generator=g, device=DEV)
    if skew:
        rank = torch.randperm(E, generator=g, device=DEV).float() + 1.0
        logits += skew * rank.pow(-1.1)
    w, idx = torch.softmax(logits, -1).topk(K, dim=-1)
    return w / w.sum(-1, keepdim=True), idx


def _bank(g, E, N, C):
    """A bank [E, N, C] of weights ~ N(0, 0.02) in 4 bits: (q, scale)."""
    parts = []
    for e in range(0, E, 64):
        w = torch.randn(min(64, E - e), N, C, generator=g, device=DEV) * 0.02
        parts.append(_tiles(*_codes(w)))
    return tuple(torch.cat(p) for p in zip(*parts))


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    if c["op"] == "pack":
        # rows of different size, as a trained weight has
        x = torch.randn(c["B"], c["N"], c["C"], generator=g, device=DEV)
        x *= torch.rand(c["B"], c["N"], 1, generator=g, device=DEV) * 0.04
        return dict(c, x=x.to(DTYPES[c["dtype"]]))
    T, H, E, K, I = c["T"], c["H"], c["E"], c["K"], c["I"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.bfloat16)

    s = dict(c, x=normal(T, H), w1=_bank(g, E, 2 * I, H), w2=_bank(g, E, H, I))
    if c["op"] == "few":
        s["wr"] = normal(E, H).mul_(0.02)
        if c["router"] == "sigmoid":
            s["bias"] = (torch.rand(E, generator=g, device=DEV) - 0.5) * 0.1
        return s
    w, idx = _routing(g, T, E, K, c["skew"])
    s["w"], s["idx"] = w, idx
    if c["op"] == "experts":
        s["idx"] = torch.where(torch.rand(T, K, generator=g, device=DEV) < c["pad"], E, idx)
    else:
        s["most"] = int(torch.bincount(idx.reshape(-1), minlength=E).max())
    return s


# ------------------------------------------------------------ plain forms

def _two_to(k):
    """2^k, k a whole number from -126 to 127, fp32, exact."""
    return ((k.int() + 127) << 23).view(torch.float32)


def _codes(v):
    """(codes, scale bytes) of v [..., C]: [..., C/32, 32] and [..., C/32], C
    padded to a multiple of 32 with zeros."""
    b = torch.nn.functional.pad(v.float(), (0, -v.shape[-1] % 32)).unflatten(-1, (-1, 32))
    a = b.abs()
    m, e = torch.frexp(a.amax(-1))
    # m 2^e <= 7 2^k, m in [1/2, 1): k = e - 3, or e - 2 where m > 7/8
    k = torch.where(m > 7 / 8, e - 2, e - 3).clamp(min=-125)
    a = a * _two_to(-k)[..., None]
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5.0))
    return code + 8 * (b < 0).to(torch.uint8), (k + 127).to(torch.uint8)


def _tiles(code, scale):
    """(q, scale) in tiles of 16 rows by 128 columns."""
    *lead, N, B, _ = code.shape
    n, b = -N % 16, -B % 4
    code = torch.nn.functional.pad(code, (0, 0, 0, b, 0, n))
    scale = torch.nn.functional.pad(scale, (0, b, 0, n))
    q = code[..., 0::2] + 16 * code[..., 1::2]
    q = q.unflatten(-2, (-1, 4)).unflatten(-4, (-1, 16))       # [.., N/16, 16, K/128, 4, 16]
    scale = scale.unflatten(-1, (-1, 4)).unflatten(-3, (-1, 16))
    return (q.movedim(-4, -2).flatten(-3).contiguous(),
            scale.movedim(-3, -2).flatten(-2).contiguous())


def _restored(q, scale, N, C):
    """The weight [..., N, C] that tiles (q, scale) hold, fp32."""
    one = torch.tensor(MAGNITUDES + tuple(-v for v in MAGNITUDES), device=q.device)
    byte = torch.arange(256, device=q.device)
    pairs = torch.stack([one[byte & 15], one[byte >> 4]], -1)
    v = pairs[q.int()].flatten(-2).unflatten(-1, (4, 16, 32))   # [.., N/16, K/128, 4, 16, 32]
    s = _two_to(scale.int() - 127).unflatten(-1, (16, 4))
    v = (v * s.transpose(-1, -2)[..., None]).movedim(-2, -4)
    return v.flatten(-3).flatten(-3, -2)[..., :N, :C]


def _plain_router(s):
    """(weights fp32 [T,K], index [T,K]); logits in 64 bits, since routing
    decides on the border between two of them."""
    logits = s["x"].double() @ s["wr"].double().t().contiguous()
    K = s["K"]
    if s["router"] == "softmax":
        # the layer's logits have the model's type, as its linear returns them
        p = torch.softmax(logits.bfloat16().float(), -1)
        p, idx = torch.sort(p, dim=-1, descending=True, stable=True)
        w, idx = p[:, :K], idx[:, :K]
        return w / w.sum(-1, keepdim=True), idx
    score = torch.sigmoid(logits)
    idx = torch.sort(score + s["bias"].double(), dim=-1, descending=True, stable=True)[1][:, :K]
    w = score.gather(1, idx)
    return (w / (w.sum(-1, keepdim=True) + 1e-20)).float(), idx


def _plain_few(s, w, idx):
    """The experts of a few tokens: every routed row with its own copy of its
    expert's weights."""
    T, K = idx.shape
    H, I = s["H"], s["I"]
    e = idx.reshape(-1)
    real = e < s["E"]
    e = torch.where(real, e, 0)
    xs = s["x"].float().repeat_interleave(K, 0)
    gu = torch.bmm(_restored(s["w1"][0][e], s["w1"][1][e], 2 * I, H), xs[:, :, None])[:, :, 0]
    act = gu[:, :I] / (1 + torch.exp(-gu[:, :I])) * gu[:, I:]
    y = torch.bmm(_restored(s["w2"][0][e], s["w2"][1][e], H, I), act[:, :, None])[:, :, 0]
    y = torch.where(real[:, None], y, 0) * w.float().reshape(-1, 1)
    return y.view(T, K, H).sum(1).to(s["x"].dtype)


def _plain_prompt(s):
    """The experts of many tokens: rows sorted by expert into [E, most, ...]."""
    E, H, I, K, most = s["E"], s["H"], s["I"], s["K"], s["most"]
    e = s["idx"].reshape(-1)
    order = torch.argsort(e, stable=True)
    es = e[order]
    count = torch.bincount(e, minlength=E)
    place = torch.arange(e.numel(), device=DEV) - (count.cumsum(0) - count)[es]
    xe = torch.zeros(E, most, H, device=DEV)
    xe[es, place] = s["x"].float()[order // K]
    gu = torch.bmm(xe, _restored(*s["w1"], 2 * I, H).transpose(1, 2).contiguous())
    act = gu[..., :I] / (1 + torch.exp(-gu[..., :I])) * gu[..., I:]
    y = torch.bmm(act, _restored(*s["w2"], H, I).transpose(1, 2).contiguous())
    rows = torch.empty(e.numel(), H, device=DEV)
    rows[order] = y[es, place]
    return (rows * s["w"].reshape(-1, 1)).view(-1, K, H).sum(1).to(s["x"].dtype)


# -------------------------------------------------------------------- run

def run(state):
    s = state
    if own:
        return _own(s)
    if s["op"] == "few":
        return _plain_few(s, *_plain_router(s))
    if s["op"] == "experts":
        return _plain_few(s, s["w"], s["idx"])
    if s["op"] == "prompt":
        return _plain_prompt(s)
    return _restored(*_tiles(*_codes(s["x"])), s["N"], s["C"]).to(s["x"].dtype)


def _own(s):
    from moe_amd import ops
    if s["op"] == "pack":
        return ops.unpack4(ops.pack4(s["x"]))
    E, H, I = s["E"], s["H"], s["I"]
    w1 = ops.Packed4(*s["w1"], (E, 2 * I, H), torch.bfloat16)
    w2 = ops.Packed4(*s["w2"], (E, H, I), torch.bfloat16)
    if s["op"] == "few":
        from moe_amd.few import moe_layer_few
        return moe_layer_few(s["x"], s["wr"], w1, w2, s["K"], router=s["router"],
                             expert_bias=s.get("bias"))
    if s["op"] == "experts":
        from moe_amd.few import experts_forward_few
        return experts_forward_few(s["x"], s["idx"], s["w"], w1, w2)
    from moe_amd import experts_forward
    return experts_forward(s["x"], s["idx"], s["w"], w1, w2)


# ------------------------------------------------------------------- work

def work(case):
    c = case
    if c["op"] == "pack":
        n = c["B"] * c["N"] * c["C"]
        q = n // 2 + c["B"] * c["N"] * -(-c["C"] // 32)
        return {"bytes": 2 * n * (4 if c["dtype"] == "f32" else 2) + 2 * q, "flops": 12 * n}
    T, H, E, K, I = c["T"], c["H"], c["E"], c["K"], c["I"]
    S = T * K * (1 - c.get("pad", 0.0))
    active = E * (1 - (1 - 1 / E) ** S)  # experts with a row, routing being even
    n = active * 3 * H * I * 17 / 32 + 2 * T * H * 2
    flops = 6 * S * H * I
    if c["op"] == "few":
        n += E * H * 2
        flops += 2 * T * E * H
    return {"bytes": int(n), "flops": int(flops)}


# ------------------------------------------------- the definition in 64 bits

def _held(v):
    """What the packed form holds of v [..., C], block by block, from the
    definition: of the values that 4 bits can hold, the nearest."""
    grid = torch.tensor(MAGNITUDES, device=v.device, dtype=torch.float64)
    out = torch.empty_like(v)
    for j in range(0, v.shape[-1], 32):
        b = v[..., j:j + 32]
        a = b.abs().amax(-1, keepdim=True)
        k = torch.floor(torch.log2(torch.where(a > 0, a, 1) / 7)) - 1
        for _ in range(3):  # the smallest k with a <= 7 * 2^k
            k = torch.where(a > 7 * torch.exp2(k), k + 1, k)
        s = torch.exp2(k.clamp(min=-125))
        u = b.abs() / s
        hi = torch.bucketize(u, grid).clamp(max=7)     # grid[hi - 1] < u <= grid[hi]
        lo = (hi - 1).clamp(min=0)
        up, down = grid[hi] - u, u - grid[lo]
        code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
        out[..., j:j + 32] = torch.copysign(grid[code] * s, b)
    return out


def _weight(bank, e, N, C):
    """Expert e's weight [N, C] from its tiles, a place at a time, 64 bits."""
    q, scale = bank[0][e], bank[1][e]
    r = torch.arange(N, device=q.device)[:, None]
    c = torch.arange(C, device=q.device)[None, :]
    byte = q[r // 16, c // 128, (c % 128) // 32 * 256 + r % 16 * 16 + c % 32 // 2].long()
    code = torch.where(c % 2 == 0, byte % 16, byte // 16)
    grid = torch.tensor(MAGNITUDES, device=q.device, dtype=torch.float64)
    s = torch.exp2(scale[r // 16, c // 128, r % 16 * 4 + c % 128 // 32].double() - 127)
    return grid[code % 8] * torch.where(code < 8, 1.0, -1.0) * s


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "pack":
        return _held(s["x"].double())
    x, H, I, E, K = s["x"].double(), s["H"], s["I"], s["E"], s["K"]
    if s["op"] == "few":
        logits = torch.stack([x @ r.double() for r in s["wr"]], 1)
        if s["router"] == "softmax":
            score = torch.softmax(logits.bfloat16().double(), -1)
            rank = score
        else:
            score = 1 / (1 + torch.exp(-logits))
            rank = score + s["bias"].double()
        idx = torch.argsort(-rank, dim=-1, stable=True)[:, :K]
        w = score.gather(1, idx)
        w = w / (w.sum(-1, keepdim=True) + (1e-20 if s["router"] == "sigmoid" else 0.0))
    else:
        idx, w = s["idx"], s["w"].double()
    out = torch.zeros_like(x)
    for e in torch.unique(idx).tolist():
        if e >= E:
            continue
        t, k = torch.nonzero(idx == e, as_tuple=True)
        gu = x[t] @ _weight(s["w1"], e, 2 * I, H).t()
        act = gu[:, :I] / (1 + torch.exp(-gu[:, :I])) * gu[:, I:]
        out.index_add_(0, t, act @ _weight(s["w2"], e, H, I).t() * w[t, k, None])
    return out
