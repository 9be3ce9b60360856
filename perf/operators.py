"""The workloads that the few-token expert layer and the 8-bit activation
checkpoints are measured on: their inputs, their plain forms in elementary
torch operations and their values in 64 bits.

  few      the whole MoE layer (router + experts) for a few tokens:
           moe_amd.few.moe_layer_few
  experts  the experts alone for a few tokens, routing given, some entries
           of it padding (ids outside [0, E)): moe_amd.few.experts_forward_few
  train    the expert layer forward and backward with its kept activations
           in 8 bits: moe_amd.experts.experts_forward(saved_activations=...)
  pack     a tensor packed to 8 bits and restored: moe_amd.ops.pack8, unpack8

A packed tensor holds, for 64 consecutive values v of a row (the last block
may be shorter), a power of two s and the integers q = rint(v / s), halves to
even: s is the smallest power of two that is at least 2^-126 and has
max|v| / s <= 127.  What is restored, q * s, is exact in bf16 and in fp32.

Layer shapes are those of moe_amd/configs.py.
"""
from __future__ import annotations

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One token of one request through the L layer: the latency of a decode step.
        dict(name="few_l_1", op="few", T=1, H=2048, E=128, K=8, I=768, dtype="bf16",
             router="softmax"),
        # A small batch of requests, one token each.
        dict(name="few_l_13", op="few", T=13, H=2048, E=128, K=8, I=768, dtype="bf16",
             router="softmax"),
        # A full decode batch: every expert of the L layer has a few rows.
        dict(name="few_l_64", op="few", T=64, H=2048, E=128, K=8, I=768, dtype="bf16",
             router="softmax"),
        # The global bank of 1792 experts behind the sigmoid router with its selection bias.
        dict(name="few_retrofit_64", op="few", T=64, H=2048, E=1792, K=8, I=768, dtype="bf16",
             router="sigmoid"),
        # The fp32 layer (XS standard), a handful of tokens.
        dict(name="few_xs_f32_5", op="few", T=5, H=1024, E=16, K=4, I=768, dtype="f32",
             router="softmax"),
        # Experts alone behind a caller's router, one token.
        dict(name="experts_xs_1", op="experts", T=1, H=1024, E=128, K=4, I=768, dtype="bf16",
             skew=0.0, pad=0.0),
        # Experts alone, a ragged batch with padded entries and a few popular experts.
        dict(name="experts_l_37", op="experts", T=37, H=2048, E=128, K=8, I=768, dtype="bf16",
             skew=2.0, pad=0.15),
        # A short ragged sequence through one layer of the global bank (XS), gate_up kept in 8 bits.
        dict(name="train_xs_509", op="train", T=509, H=1024, E=128, K=4, I=768, skew=0.0,
             keep="int8"),
        # A micro-batch through the L layer with skewed routing, gate_up kept in 8 bits.
        dict(name="train_l_8192", op="train", T=8192, H=2048, E=128, K=8, I=768, skew=2.0,
             keep="int8"),
        # The same layer at a larger micro-batch, hidden states kept in 8 bits too.
        dict(name="train_l_16384", op="train", T=16384, H=2048, E=128, K=8, I=768, skew=0.0,
             keep="int8_all"),
        # The hidden states of a short ragged batch, packed and restored.
        dict(name="pack_1021", op="pack", rows=1021, cols=2048, dtype="bf16"),
        # The gate_up of a whole micro-batch (S = 131072 routed rows), fp32.
        dict(name="pack_131072", op="pack", rows=131072, cols=1536, dtype="f32"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["few", "few", "experts", "train", "train", "pack"])
    if op == "pack":
        return dict(op=op, rows=_spread(rng, 1, 60000), cols=_spread(rng, 1, 3000),
                    dtype=rng.choice(["bf16", "f32"]))
    case = dict(op=op, H=64 * rng.randint(4, 32), I=64 * rng.randint(2, 12))
    if op == "train":
        return dict(case, T=_spread(rng, 1, 8000), E=8 * rng.randint(1, 16), K=rng.randint(1, 8),
                    skew=rng.choice([0.0, 2.0]), keep=rng.choice(["int8", "int8_all"]))
    case.update(T=_spread(rng, 1, 64), E=8 * rng.randint(2, 64), K=rng.randint(1, 8),
                dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]))
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


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    if c["op"] == "pack":
        # activations: rows of different size, as a gate_up has over its experts
        x = torch.randn(c["rows"], c["cols"], generator=g, device=DEV)
        x *= torch.rand(c["rows"], 1, generator=g, device=DEV) * 4
        return dict(c, x=x.to(DTYPES[c["dtype"]]))
    T, H, E, K, I = c["T"], c["H"], c["E"], c["K"], c["I"]
    dt = DTYPES[c.get("dtype", "bf16")]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dt)

    s = dict(c, x=normal(T, H), w1=normal(E, 2 * I, H).mul_(0.02), w2=normal(E, H, I).mul_(0.02))
    if c["op"] == "few":
        s["wr"] = normal(E, H).mul_(0.02)
        if c["router"] == "sigmoid":
            s["bias"] = (torch.rand(E, generator=g, device=DEV) - 0.5) * 0.1
        return s
    w, idx = _routing(g, T, E, K, c["skew"])
    s["w"], s["idx"] = w.to(dt), idx
    if c["op"] == "experts":
        s["idx"] = torch.where(torch.rand(T, K, generator=g, device=DEV) < c["pad"], E, idx)
        return s
    s["dout"] = normal(T, H)
    s["most"] = int(torch.bincount(idx.reshape(-1), minlength=E).max())
    for name in ("x", "w", "w1", "w2"):
        s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------ plain forms

def _restored(v):
    """What a packed and restored `v` (..., n) holds, fp32 or fp64."""
    n = v.shape[-1]
    b = torch.nn.functional.pad(v, (0, -n % 64)).unflatten(-1, (-1, 64))
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    # m * 2^e <= 127 * 2^k, m in [1/2, 1): k = e - 7, or e - 6 where m > 127/128
    k = torch.where(m > 127 / 128, e - 6, e - 7).clamp(min=-126)
    s = torch.ldexp(torch.ones_like(m), k)
    return (torch.round(b / s) * s).flatten(-2)[..., :n]


def _plain_router(s):
    """(weights fp32 [T,K], index [T,K]); logits in 64 bits, since routing
    decides on the border between two of them."""
    logits = s["x"].double() @ s["wr"].double().t().contiguous()
    K = s["K"]
    if s["router"] == "softmax":
        # the layer's logits have the model's type, as its linear returns them
        p = torch.softmax(logits.to(s["x"].dtype).float(), -1)
        p, idx = torch.sort(p, dim=-1, descending=True, stable=True)
        w, idx = p[:, :K], idx[:, :K]
        return w / w.sum(-1, keepdim=True), idx
    score = torch.sigmoid(logits)
    idx = torch.sort(score + s["bias"].double(), dim=-1, descending=True, stable=True)[1][:, :K]
    w = score.gather(1, idx)
    return (w / (w.sum(-1, keepdim=True) + 1e-20)).float(), idx


def _plain_experts(x, idx, w, w1, w2):
    """The experts of a few tokens: every routed row with its own copy of its
    expert's weights."""
    T, K = idx.shape
    E, H, I = w2.shape
    e = idx.reshape(-1)
    real = e < E
    e = torch.where(real, e, 0)
    xs = x.float().repeat_interleave(K, 0)
    gu = torch.bmm(w1[e].float(), xs[:, :, None])[:, :, 0]
    act = gu[:, :I] / (1 + torch.exp(-gu[:, :I])) * gu[:, I:]
    y = torch.bmm(w2[e].float(), act[:, :, None])[:, :, 0]
    y = torch.where(real[:, None], y, 0) * w.float().reshape(-1, 1)
    return y.view(T, K, H).sum(1).to(x.dtype)


@torch.no_grad()
def _plain_train(s):
    """(out, dx, dw, dW1, dW2): rows sorted by expert into [E, most, ...]."""
    x, w, w1, w2 = (s[k].float() for k in ("x", "w", "w1", "w2"))
    dout, E, I, most, K = s["dout"].float(), s["E"], s["I"], s["most"], s["K"]
    e = s["idx"].reshape(-1)
    S = e.numel()
    order = torch.argsort(e, stable=True)
    es = e[order]
    count = torch.bincount(e, minlength=E)
    place = torch.arange(S, device=DEV) - (count.cumsum(0) - count)[es]
    tok = order // K

    def rows(v):  # [S, n] in expert order -> [E, most, n]
        r = v.new_zeros(E, most, v.shape[-1])
        r[es, place] = v
        return r

    def back(r):  # [E, most, n] -> [S, n] in token order
        v = torch.empty(S, r.shape[-1], device=DEV, dtype=r.dtype)
        v[order] = r[es, place]
        return v

    xe = rows(x[tok])
    # the layer's gate_up has its type (bf16): that is what is packed
    gu = torch.bmm(xe, w1.transpose(1, 2)).bfloat16().float()
    act = gu[..., :I] * torch.sigmoid(gu[..., :I]) * gu[..., I:]
    y = back(torch.bmm(act, w2.transpose(1, 2)))
    wf = w.reshape(-1, 1)
    out = (y * wf).view(-1, K, x.shape[1]).sum(1)
    # backward, from the restored gate_up
    gu = _restored(gu)
    gate, up = gu[..., :I], gu[..., I:]
    sig = torch.sigmoid(gate)
    act = gate * sig * up
    do = rows(dout[tok])
    wr = rows(wf[order])
    g = torch.bmm(do, w2)
    dw = back((g * act).sum(-1, keepdim=True)).view(-1, K)
    da = g * wr
    dgu = torch.cat([da * up * (sig + gate * sig * (1 - sig)), da * gate * sig], -1)
    dw2 = torch.bmm((do * wr).transpose(1, 2), act)
    dx = back(torch.bmm(dgu, w1)).view(-1, K, x.shape[1]).sum(1)
    if s["keep"] == "int8_all":
        xe = rows(_restored(x)[tok])
    dw1 = torch.bmm(dgu.transpose(1, 2), xe)
    return tuple(v.bfloat16() for v in (out, dx, dw, dw1, dw2))


# -------------------------------------------------------------------- run

def run(state):
    s = state
    if own:
        return _own(s)
    if s["op"] == "few":
        w, idx = _plain_router(s)
        return _plain_experts(s["x"], idx, w, s["w1"], s["w2"])
    if s["op"] == "experts":
        return _plain_experts(s["x"], s["idx"], s["w"], s["w1"], s["w2"])
    if s["op"] == "train":
        return _plain_train(s)
    return _restored(s["x"].float()).to(s["x"].dtype)


def _own(s):
    if s["op"] == "few":
        from moe_amd.few import moe_layer_few
        return moe_layer_few(s["x"], s["wr"], s["w1"], s["w2"], s["K"], router=s["router"],
                             expert_bias=s.get("bias"))
    if s["op"] == "experts":
        from moe_amd.few import experts_forward_few
        return experts_forward_few(s["x"], s["idx"], s["w"], s["w1"], s["w2"])
    if s["op"] == "train":
        from moe_amd import experts_forward
        out = experts_forward(s["x"], s["idx"], s["w"], s["w1"], s["w2"],
                              saved_activations=s["keep"])
        grads = torch.autograd.grad(out, (s["x"], s["w"], s["w1"], s["w2"]), s["dout"])
        return (out.detach(),) + grads
    from moe_amd import ops
    return ops.unpack8(ops.pack8(s["x"]))


# ------------------------------------------------------------------- work

def work(case):
    c = case
    b = 4 if c.get("dtype") == "f32" else 2
    if c["op"] == "pack":
        n = c["rows"] * c["cols"]
        q = n + c["rows"] * -(-c["cols"] // 64)
        return {"bytes": 2 * n * b + 2 * q, "flops": 4 * n}
    T, H, E, K, I = c["T"], c["H"], c["E"], c["K"], c["I"]
    S = T * K
    if c["op"] == "train":
        # inputs, weights and outputs, gradients of both, the packed gate_up written and read
        n = 2 * (4 * T * H + 2 * 3 * E * H * I + 2 * S) + 2 * S * 2 * I * 65 // 64
        return {"bytes": n, "flops": 18 * S * H * I}
    S = S * (1 - c.get("pad", 0.0))
    active = E * (1 - (1 - 1 / E) ** S)  # experts with a row, routing being even
    n = active * 3 * H * I * b + 2 * T * H * b
    flops = 6 * S * H * I
    if c["op"] == "few":
        n += E * H * b
        flops += 2 * T * E * H
    return {"bytes": int(n), "flops": int(flops)}


# ------------------------------------------------- the definition in 64 bits

def _blocks8(v):
    """q * s of the packed form, block by block, from the definition."""
    out = torch.empty_like(v)
    for j in range(0, v.shape[-1], 64):
        b = v[..., j:j + 64]
        a = b.abs().amax(-1, keepdim=True)
        k = torch.floor(torch.log2(torch.where(a > 0, a, 1) / 127)) - 1
        for _ in range(3):  # the smallest k with a <= 127 * 2^k
            k = torch.where(a > 127 * torch.exp2(k), k + 1, k)
        s = torch.exp2(k.clamp(min=-126))
        out[..., j:j + 64] = torch.round(b / s) * s
    return out


def _exact_rows(x, w1, w2, I):
    """(gate, up) of x's rows through one expert, 64 bits."""
    gu = x @ w1.double().t()
    return gu[:, :I], gu[:, I:]


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "pack":
        return _blocks8(s["x"].double())
    x, I, E, K = s["x"].detach().double(), s["I"], s["E"], s["K"]
    if s["op"] == "few":
        logits = torch.stack([x @ r.double() for r in s["wr"]], 1)
        if s["router"] == "softmax":
            score = torch.softmax(logits.to(s["x"].dtype).double(), -1)
            rank = score
        else:
            score = 1 / (1 + torch.exp(-logits))
            rank = score + s["bias"].double()
        idx = torch.argsort(-rank, dim=-1, stable=True)[:, :K]
        w = score.gather(1, idx)
        w = w / (w.sum(-1, keepdim=True) + (1e-20 if s["router"] == "sigmoid" else 0.0))
    else:
        idx, w = s["idx"], s["w"].detach().double()
    out = torch.zeros_like(x)
    used = [e for e in torch.unique(idx).tolist() if e < E]
    if s["op"] in ("few", "experts"):
        for e in used:
            t, k = torch.nonzero(idx == e, as_tuple=True)
            g, u = _exact_rows(x[t], s["w1"][e], s["w2"][e], I)
            y = (g / (1 + torch.exp(-g)) * u) @ s["w2"][e].double().t()
            out.index_add_(0, t, y * w[t, k, None])
        return out
    dout = s["dout"].double()
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    dw1 = torch.zeros(s["w1"].shape, device=DEV, dtype=torch.float64)
    dw2 = torch.zeros(s["w2"].shape, device=DEV, dtype=torch.float64)
    kept = _blocks8(x) if s["keep"] == "int8_all" else x
    for e in used:
        t, k = torch.nonzero(idx == e, as_tuple=True)
        m1, m2 = s["w1"][e].detach().double(), s["w2"][e].detach().double()
        g, u = _exact_rows(x[t], m1, m2, I)
        g, u = g.bfloat16().double(), u.bfloat16().double()
        wk = w[t, k, None]
        out.index_add_(0, t, (g / (1 + torch.exp(-g)) * u) @ m2.t() * wk)
        g, u = _blocks8(g), _blocks8(u)
        sig = 1 / (1 + torch.exp(-g))
        act = g * sig * u
        d = dout[t] @ m2
        dw[t, k] = (d * act).sum(-1)
        d = d * wk
        dgu = torch.cat([d * u * sig * (1 + g * (1 - sig)), d * g * sig], 1)
        dx.index_add_(0, t, dgu @ m1)
        dw1[e] = dgu.t() @ kept[t]
        dw2[e] = (dout[t] * wk).t() @ act
    return out, dx, dw, dw1, dw2
