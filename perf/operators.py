"""Attention with modified scores and what stands in front of it, as calls that
can be timed and checked.

Four operators: the rotary embedding in either pair layout, over part of the
head, at given positions (`rotary`); the norm of each query and key head with
that rotation in one pass (`qk_norm`); attention whose scores are capped, get a
bias by distance, or are masked by documents or a prefix, with key heads shared
by query heads (`attn`); and the same attention for the newest token of each
sequence over its cache (`decode`).

With `own` false, `run` computes them in plain torch operations in float32,
rounded once; with `own` true it calls the framework.  `exact` restates each in
float64.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # One new token of 16 sequences, each at its own position, between the
        # projection and the cache: nothing but latency.
        dict(name="rotary_token_half_bf16", kind="rotary", dtype="bfloat16", S=1, B=16, H=32, Hk=8,
             D=128, R=128, interleaved=False, positions="each", grad=False),
        # Training with half of each head rotated (half layout), shared key heads.
        dict(name="rotary_partial_half_bf16_s2048", kind="rotary", dtype="bfloat16", S=2048, B=4,
             H=32, Hk=8, D=128, R=64, interleaved=False, positions="none", grad=True),
        # Packed documents whose positions start over, odd length, full precision.
        dict(name="rotary_packed_fp32_s1000", kind="rotary", dtype="float32", S=1000, B=3, H=12,
             Hk=12, D=64, R=64, interleaved=True, positions="each", grad=True),
        # One new token of 64 sequences of a model that normalises queries and keys.
        dict(name="qk_norm_token_bf16", kind="qk_norm", dtype="bfloat16", S=1, B=64, H=16, Hk=8,
             D=128, R=128, interleaved=False, positions="each", grad=False),
        # A layer of the 12-head model's train step.
        dict(name="qk_norm_bf16_s1024", kind="qk_norm", dtype="bfloat16", S=1024, B=8, H=12, Hk=12,
             D=64, R=64, interleaved=True, positions="none", grad=True),
        # The largest of these: a long context with shared key heads, fp16.
        dict(name="qk_norm_fp16_s4096_d128", kind="qk_norm", dtype="float16", S=4096, B=4, H=32,
             Hk=8, D=128, R=128, interleaved=False, positions="none", grad=True),
        # Prefill of a model with capped scores: the forward alone.
        dict(name="attn_cap_bf16_s4096_d128", kind="attn", dtype="bfloat16", B=1, H=32, Hk=8,
             S=4096, D=128, causal=True, cap=50.0, bias=False, docs=0, pack=0, prefix=False,
             grad=False),
        # A layer of the 12-head model's train step with distance biases in
        # place of the rotary embedding.
        dict(name="attn_bias_bf16_s1024", kind="attn", dtype="bfloat16", B=8, H=12, Hk=12, S=1024,
             D=64, causal=True, cap=0.0, bias=True, docs=0, pack=0, prefix=False, grad=True),
        # Training on sequences packed from documents of many lengths, with a
        # padded end: long context, shared key heads.
        dict(name="attn_docs_bf16_s4096_d128", kind="attn", dtype="bfloat16", B=2, H=16, Hk=4,
             S=4096, D=128, causal=True, cap=0.0, bias=False, docs=9, pack=1, prefix=False,
             grad=True),
        # Full-precision training with a bidirectional prefix, no whole tiles.
        dict(name="attn_prefix_fp32_s1000", kind="attn", dtype="float32", B=2, H=12, Hk=12, S=1000,
             D=64, causal=True, cap=0.0, bias=False, docs=0, pack=0, prefix=True, grad=True),
        # Serving: the newest token of 32 sequences of different lengths.
        dict(name="decode_bf16_b32_s4096", kind="decode", dtype="bfloat16", B=32, H=32, Hk=8,
             S=4096, D=128, cap=0.0, bias=False, lengths=True, pack=2),
        # One long sequence of a model with capped scores: few rows, a long axis.
        dict(name="decode_cap_bf16_b1_s65536", kind="decode", dtype="bfloat16", B=1, H=16, Hk=4,
             S=65536, D=128, cap=30.0, bias=False, lengths=False, pack=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    Hk = rng.choice([1, 2, 4, 8, 12])
    return Hk * rng.choice([1, 1, 2, 3, 4, 8]), Hk


def draw(rng):
    kind = rng.choice(["rotary", "qk_norm", "attn", "attn", "attn", "decode"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    H, Hk = _heads(rng)
    if kind in ("rotary", "qk_norm"):
        D = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        S, B = _log_int(rng, 1, 8192), rng.choice([1, 2, 3, 4, 8, 16])
        while B > 1 and S * B * (H + Hk) * D > 1 << 25:
            B -= 1
        S = min(S, max(1, (1 << 25) // (B * (H + Hk) * D)))
        return dict(kind=kind, dtype=dtype, S=S, B=B, H=H, Hk=Hk, D=D,
                    R=D if rng.random() < 0.6 else rng.choice([D // 2, 2 * rng.randint(1, D // 2)]),
                    interleaved=rng.random() < 0.5, positions=rng.choice(["none", "row", "each"]),
                    grad=rng.random() < 0.7)
    if kind == "decode":
        S, B = _log_int(rng, 1, 65536), rng.choice([1, 2, 4, 7, 16, 32])
        D = rng.choice([64, 128, 128, 96])
        while B > 1 and S * B * Hk * D > 1 << 26:
            B -= 1
        S = min(S, (1 << 26) // (B * Hk * D))
        return dict(kind=kind, dtype=dtype, B=B, H=H, Hk=Hk, S=S, D=D,
                    cap=rng.choice([0.0, 0.0, 30.0]), bias=rng.random() < 0.3,
                    lengths=rng.random() < 0.7, pack=rng.randrange(1 << 20))
    D = rng.choice([32, 64, 64, 80, 128, 128])
    S, B = _log_int(rng, 1, 8192), rng.choice([1, 2, 3, 4, 8])
    if rng.random() < 0.4:
        S = max(1, S // 64 * 64)
    causal, grad = rng.random() < 0.75, rng.random() < 0.7
    # products and scores of all heads: no more than the largest listed case has
    most = (13e9 if dtype == "float32" else 137e9) / ((7 if grad else 2) * (1 if causal else 2) * D)
    most = int(min(most, 1 << 29))
    while B > 1 and B * H * S * S > most:
        B -= 1
    S = min(S, math.isqrt(most // (B * H)))
    docs = rng.choice([0, 0, rng.randint(1, 12)])
    return dict(kind=kind, dtype=dtype, B=B, H=H, Hk=Hk, S=S, D=D, causal=causal,
                cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.random() < 0.3, docs=docs,
                pack=rng.randrange(1 << 20), prefix=causal and rng.random() < 0.3, grad=grad)


# --------------------------------------------------------------------------
# inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _spans(c):
    """The documents of each sequence, [(id, first, end)], the rest padding: by
    the case alone, as the work depends on them."""
    rng, spans = random.Random(c["pack"]), []
    for _ in range(c["B"]):
        end = c["S"] - int(c["S"] * rng.choice([0, 0.02, 0.1]))
        cuts = sorted(rng.randint(0, end) for _ in range(c["docs"] - 1))
        spans.append([(i, a, b) for i, (a, b) in enumerate(zip([0] + cuts, cuts + [end]))])
    return spans


def _prefixes(c):
    rng = random.Random(c["pack"] + 1)
    return [rng.randint(0, c["S"] // 2) for _ in range(c["B"])]


def _lengths(c):
    rng = random.Random(c["pack"])
    return [rng.randint(max(1, c["S"] // 8), c["S"]) if c["lengths"] else c["S"]
            for _ in range(c["B"])]


def _document_ids(c):
    ids = torch.full((c["B"], c["S"]), -1, dtype=torch.int32)
    for b, spans in enumerate(_spans(c)):
        for i, first, end in spans:
            ids[b, first:end] = i
    return ids.cuda()


def _slopes(H):
    return (2.0 ** (-8.0 * torch.arange(1, H + 1, dtype=torch.float32) / H)).cuda()


def _rotary_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    S, B, H, Hk, D, R = (c[n] for n in ("S", "B", "H", "Hk", "D", "R"))
    qkv = _randn(g, (S, B, (H + 2 * Hk) * D), dt)  # the fused projection they are cut from
    T = S + 64 if c["positions"] == "none" else 8192
    freqs = 1.0 / (10000.0 ** (torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R))
    a = torch.outer(torch.arange(T, device="cuda", dtype=torch.float64), freqs)
    x = dict(q=qkv[..., : H * D].view(S, B, H, D),
             k=qkv[..., H * D: (H + Hk) * D].view(S, B, Hk, D),
             cos=a.cos().to(dt), sin=a.sin().to(dt), pos=None)
    if c["positions"] != "none":
        x["pos"] = torch.randint(0, T, (S, B) if c["positions"] == "each" else (S,), generator=g,
                                 device="cuda")
    if c["kind"] == "qk_norm":
        x["wq"], x["wk"] = ((1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dt)
                            for _ in range(2))
    if c["grad"]:
        x["dq"], x["dk"] = _randn(g, (S, B, H, D), dt), _randn(g, (S, B, Hk, D), dt)
    return x


def _attn_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    B, H, Hk, S, D = (c[n] for n in ("B", "H", "Hk", "S", "D"))

    # [S, B, heads, D] as the projections give them, seen as [B, heads, S, D];
    # scores of a few units, so that a cap has something to do
    def heads(n, scale):
        return _randn(g, (S, B, n, D), dt, scale).permute(1, 2, 0, 3)

    return dict(q=heads(H, 1.5), k=heads(Hk, 1.5), v=heads(Hk, 1.0),
                do=_randn(g, (B, H, S, D), dt) if c["grad"] else None,
                slopes=_slopes(H) if c["bias"] else None,
                docs=_document_ids(c) if c["docs"] else None,
                prefix=torch.tensor(_prefixes(c), dtype=torch.int32).cuda() if c["prefix"] else None)


def _decode_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    B, H, Hk, S, D = (c[n] for n in ("B", "H", "Hk", "S", "D"))
    return dict(q=_randn(g, (B, H, D), dt, 1.5), k=_randn(g, (B, Hk, S, D), dt, 1.5),
                v=_randn(g, (B, Hk, S, D), dt), slopes=_slopes(H) if c["bias"] else None,
                lengths=torch.tensor(_lengths(c), dtype=torch.int32).cuda() if c["lengths"] else None)


def _inputs(c, seed):
    make = {"attn": _attn_inputs, "decode": _decode_inputs}.get(c["kind"], _rotary_inputs)
    return make(c, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    if case.get("grad"):
        for n in ("q", "k", "v", "wq", "wk"):
            if n in s:
                s[n].requires_grad_()
    return {"case": case, **s}


# --------------------------------------------------------------------------
# the framework's calls


def _own(c, s):
    import gpt_from_scratch_amd as fw

    cap = c.get("cap") or None
    if c["kind"] == "decode":
        return fw.decode_attn(s["q"], s["k"], s["v"], lengths=s["lengths"], softcap=cap,
                              slopes=s["slopes"])
    if c["kind"] == "attn":
        how = dict(causal=c["causal"], softcap=cap, slopes=s["slopes"], document_ids=s["docs"],
                   prefix_lens=s["prefix"])
        if not c["grad"]:
            return fw.scored_attn_forward(s["q"], s["k"], s["v"], **how)
        o = fw.scored_attn(s["q"], s["k"], s["v"], **how)
        return (o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"]))
    how = dict(positions=s["pos"], interleaved=c["interleaved"])
    if c["kind"] == "rotary":
        y, wrt = fw.apply_rotary_qk(s["q"], s["k"], s["cos"], s["sin"], **how), (s["q"], s["k"])
    else:
        y = fw.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], eps=EPS, **how)
        wrt = (s["q"], s["k"], s["wq"], s["wk"])
    return (*y, *torch.autograd.grad(y, wrt, (s["dq"], s["dk"]))) if c["grad"] else y


# --------------------------------------------------------------------------
# the plain forms


def _angles(s, S):
    """cos and sin, [S, 1 or B, 1, R / 2]."""
    pos = s["pos"]
    cos, sin = ((t[:S] if pos is None else t[pos]).float() for t in (s["cos"], s["sin"]))
    return (t[:, None, None] if t.dim() == 2 else t[:, :, None] for t in (cos, sin))


def _turn(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] elements of each head turned by the angles."""
    n = cos.shape[-1]
    a, b = (x[..., : 2 * n: 2], x[..., 1: 2 * n: 2]) if interleaved else (x[..., :n],
                                                                         x[..., n: 2 * n])
    p, q = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((p, q), -1).flatten(-2) if interleaved else torch.cat((p, q), -1)
    return torch.cat((y, x[..., 2 * n:]), -1)


def _plain_rotary(c, s):
    dt, cos_sin = DTYPES[c["dtype"]], tuple(_angles(s, c["S"]))
    back = (cos_sin[0], -cos_sin[1])
    lay, norm = c["interleaved"], c["kind"] == "qk_norm"
    xs = [t.detach().float() for t in (s["q"], s["k"])]
    if not norm:
        ys = [_turn(x, *cos_sin, lay).to(dt) for x in xs]
        if c["grad"]:
            ys += [_turn(t.float(), *back, lay).to(dt) for t in (s["dq"], s["dk"])]
        return tuple(ys)
    ws = [t.detach().float() for t in (s["wq"], s["wk"])]
    rs = [torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) for x in xs]
    ns = [x * r for x, r in zip(xs, rs)]
    ys = [_turn(n * w, *cos_sin, lay).to(dt) for n, w in zip(ns, ws)]
    if not c["grad"]:
        return tuple(ys)
    ds = [_turn(t.float(), *back, lay) for t in (s["dq"], s["dk"])]
    gs = [d * w for d, w in zip(ds, ws)]
    dx = [r * (g - n * (g * n).mean(-1, keepdim=True)) for r, g, n in zip(rs, gs, ns)]
    dw = [(d * n).sum((0, 1, 2)) for d, n in zip(ds, ns)]
    return tuple(ys) + tuple(t.to(dt) for t in dx + dw)


def _visible(c, s):
    """[1 or B, 1, S, S]: which keys each query sees; None if all."""
    i = torch.arange(c["S"], device="cuda")
    see = None
    if c["causal"]:
        see = (i[None, :] <= i[:, None])[None]
        if s["prefix"] is not None:
            see = see | (i[None, :] < s["prefix"][:, None])[:, None]
    if s["docs"] is not None:
        d = s["docs"]
        same = (d[:, :, None] == d[:, None, :]) & (d >= 0)[:, :, None]
        see = same if see is None else see & same
    return None if see is None else see[:, None]


def _capped(z, cap):
    """(scores, their derivative by the uncapped ones or None)."""
    if not cap:
        return z, None
    t = torch.tanh(z / cap)
    return cap * t, 1 - t * t


def _plain_attn(c, s):
    dt, G, D, S = DTYPES[c["dtype"]], c["H"] // c["Hk"], c["D"], c["S"]
    q, k, v = (s[n].detach().float().contiguous() for n in ("q", "k", "v"))
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    scale = 1.0 / math.sqrt(D)
    z, slope = _capped((q @ k.transpose(-1, -2).contiguous()) * scale, c["cap"])
    if c["bias"]:
        i = torch.arange(S, device="cuda", dtype=torch.float32)
        z = z - s["slopes"][:, None, None] * (i[:, None] - i[None, :]).abs()
    see = _visible(c, s)
    if see is not None:
        z = z.masked_fill(~see, -math.inf)
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(z - m)
    total = p.sum(-1, keepdim=True)
    lse = (m + torch.log(total))[..., 0]
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = p @ v
    if not c["grad"]:
        return o.to(dt), lse
    do = s["do"].float()
    dv = p.transpose(-1, -2).contiguous() @ do
    ds = p * (do @ v.transpose(-1, -2).contiguous() - (do * o).sum(-1, keepdim=True))
    if slope is not None:
        ds = ds * slope
    ds = ds * scale
    dk = ds.transpose(-1, -2).contiguous() @ q
    dk, dv = (t.view(c["B"], c["Hk"], G, S, D).sum(2) for t in (dk, dv))
    return tuple(t.to(dt) for t in (o, ds @ k, dk, dv))


def _plain_decode(c, s):
    B, H, Hk, S, D = (c[n] for n in ("B", "H", "Hk", "S", "D"))
    q = s["q"].float().view(B, Hk, H // Hk, D)
    k, v = s["k"].float(), s["v"].float()
    z, _ = _capped((q @ k.transpose(-1, -2).contiguous()) / math.sqrt(D), c["cap"])
    n = (s["lengths"] if s["lengths"] is not None else
         torch.full((B,), S, device="cuda", dtype=torch.int32)).view(B, 1, 1, 1)
    j = torch.arange(S, device="cuda")
    if c["bias"]:
        z = z - s["slopes"].view(Hk, H // Hk, 1) * (n - 1 - j).abs()
    p = torch.exp(z.masked_fill(j >= n, -math.inf) - z.masked_fill(j >= n, -math.inf)
                  .amax(-1, keepdim=True))
    return ((p / p.sum(-1, keepdim=True)) @ v).to(DTYPES[c["dtype"]]).view(B, H, D)


def run(state):
    c = state["case"]
    if own:
        return _own(c, state)
    plain = {"attn": _plain_attn, "decode": _plain_decode}.get(c["kind"], _plain_rotary)
    return plain(c, state)


# --------------------------------------------------------------------------
# what each pass cannot do without


def _pairs(c):
    """Pairs of a query and a key that it sees, all sequences of one head."""
    n = 0
    pre = _prefixes(c) if c["prefix"] else [0] * c["B"]
    for spans, p in zip(_spans(c) if c["docs"] else [[(0, 0, c["S"])]] * c["B"], pre):
        for _, a, b in spans:
            m, w = b - a, max(0, min(p, b) - a)
            # causal pairs, and those above the diagonal whose key lies in the prefix
            n += m * (m + 1) // 2 + w * (w - 1) // 2 if c["causal"] else m * m
    return n


def work(case):
    c = case
    e = 4 if c["dtype"] == "float32" else 2
    H, Hk, D, S, B = (c[n] for n in ("H", "Hk", "D", "S", "B"))
    if c["kind"] in ("rotary", "qk_norm"):
        x = S * B * (H + Hk) * D
        rows = S * B if c["positions"] == "each" else S
        tabs = 2 * min(rows, 8192 if c["positions"] != "none" else rows) * c["R"] // 2 * e
        norm = c["kind"] == "qk_norm"
        moved = (2 + (2 if c["grad"] else 0)) * x * e  # q, k, their gradients: in and out
        return {"bytes": moved + tabs + (2 * D * e * (2 if c["grad"] else 1) if norm else 0),
                "flops": 0}
    if c["kind"] == "decode":
        keys = sum(_lengths(c))
        return {"bytes": 2 * e * Hk * D * keys + 2 * B * H * D * e, "flops": 4.0 * H * D * keys}
    qo, kv = B * H * S * D * e, B * Hk * S * D * e
    ids = 4 * B * S if c["docs"] else 0
    unit = 2.0 * H * D * _pairs(c)
    if not c["grad"]:
        return {"bytes": 2 * qo + 2 * kv + 4 * B * H * S + ids, "flops": 2 * unit}
    return {"bytes": 4 * qo + 4 * kv + ids, "flops": 7 * unit}


# --------------------------------------------------------------------------
# float64


def _pair_product(x, pos, cos, sin, interleaved, sign):
    """Rotation as a product of complex numbers over the pairs."""
    n = cos.shape[1]
    c, s = cos.double()[pos], sign * sin.double()[pos]
    w = torch.complex(c, s)
    w = w[:, None, None] if w.dim() == 2 else w[:, :, None]
    r = x[..., : 2 * n]
    pairs = r.unflatten(-1, (n, 2)) if interleaved else r.unflatten(-1, (2, n)).transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat((y, x[..., 2 * n:]), -1)


def _exact_rotary(c, seed):
    s = _rotary_inputs(c, seed)
    pos = s["pos"] if s["pos"] is not None else torch.arange(c["S"], device="cuda")
    outs, grads, wgrads = [], [], []
    for n in ("q", "k"):
        x = s[n].double().requires_grad_(c["grad"])
        y, wrt = x, (x,)
        if c["kind"] == "qk_norm":
            w = s["w" + n].double().requires_grad_(c["grad"])
            y, wrt = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["D"] + EPS) * w, (x, w)
        y = _pair_product(y, pos, s["cos"], s["sin"], c["interleaved"], 1.0)
        outs.append(y.detach())
        if c["grad"]:
            got = torch.autograd.grad(y, wrt, s["d" + n].double())
            grads.append(got[0])
            wgrads += got[1:]
    return tuple(outs + grads + wgrads)


def _scale(c):
    return c["D"] ** -0.5


def _scores64(q, k, c, slopes, dist):
    """Capped and biased scores of one key head's queries [G, n, D] on keys [m, D]."""
    z = torch.matmul(q, k.t()) * _scale(c)
    if c["cap"]:
        z = torch.tanh(z / c["cap"]) * c["cap"]
    if slopes is not None:
        z = z - slopes.double()[:, None, None] * dist
    return z


def _exact_attn(c, seed):
    if c["B"] * c["H"] * c["S"] ** 2 * c["D"] > 1 << 38:
        return None
    s = _attn_inputs(c, seed)
    B, H, Hk, S, D = (c[n] for n in ("B", "H", "Hk", "S", "D"))
    G = H // Hk
    i = torch.arange(S, device="cuda", dtype=torch.float64)
    dist = (i[:, None] - i[None, :]).abs()
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    o, lse = torch.zeros_like(q).contiguous(), torch.empty(B, H, S, device="cuda", dtype=torch.float64)
    dq, dk, dv = (torch.zeros(t.shape, device="cuda", dtype=torch.float64) for t in (q, k, v))
    for b in range(B):
        hidden = torch.zeros(S, S, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden |= i[None, :] > i[:, None]
            if s["prefix"] is not None:
                hidden[:, : int(s["prefix"][b])] = False
        if s["docs"] is not None:
            d = s["docs"][b]
            hidden |= (d[:, None] != d[None, :]) | (d < 0)[None, :]
        empty = hidden.all(-1)
        for h in range(Hk):
            hs = slice(h * G, (h + 1) * G)
            qg, kg, vg = (t.detach().requires_grad_(c["grad"]) for t in (q[b, hs], k[b, h], v[b, h]))
            z = _scores64(qg, kg, c, s["slopes"][hs] if c["bias"] else None, dist)
            z = z.masked_fill(hidden, -math.inf)
            lse[b, hs] = torch.logsumexp(z.detach(), -1)
            p = torch.softmax(z.masked_fill(empty[:, None], 0.0), -1) * (~empty)[:, None]
            y = torch.matmul(p, vg)
            o[b, hs] = y.detach()
            if c["grad"]:
                dq[b, hs], dk[b, h], dv[b, h] = torch.autograd.grad(y, (qg, kg, vg),
                                                                    s["do"][b, hs].double())
            del z, p, y
    return (o, dq, dk, dv) if c["grad"] else (o, lse)


def _exact_decode(c, seed):
    s = _decode_inputs(c, seed)
    B, H, Hk, S, D = (c[n] for n in ("B", "H", "Hk", "S", "D"))
    G = H // Hk
    o = torch.empty(B, H, D, device="cuda", dtype=torch.float64)
    for b, n in enumerate(_lengths(c)):
        back = torch.arange(n - 1, -1, -1, device="cuda", dtype=torch.float64)
        for h in range(Hk):
            hs = slice(h * G, (h + 1) * G)
            z = _scores64(s["q"][b, hs, None].double(), s["k"][b, h, :n].double(), c,
                          s["slopes"][hs] if c["bias"] else None, back)
            o[b, hs] = torch.matmul(torch.softmax(z, -1), s["v"][b, h, :n].double())[:, 0]
    return o


def exact(case, seed):
    how = {"attn": _exact_attn, "decode": _exact_decode}.get(case["kind"], _exact_rotary)
    return how(case, seed)
