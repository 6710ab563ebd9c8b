"""Plain float64 forms of the rotary, norm and attention operators, and how far a
kernel that computes them in fp32 with stated roundings may be off.

Units: u = torch.finfo(dtype).eps / 2 is the largest relative error of one rounding
to dtype, f = 2^-24 that of fp32.  Every bound below is a sum of worst cases, term
by term, so no margin is added beyond the counts of fp32 operations."""
import math

import torch

F32 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def visible(B, Sq, Sk, causal, docs=None, prefix=None, device="cpu"):
    """[B, Sq, Sk]: which keys each query sees; query i is at position Sk - Sq + i."""
    i = torch.arange(Sk - Sq, Sk, device=device)[:, None]
    j = torch.arange(Sk, device=device)[None, :]
    see = torch.ones(B, Sq, Sk, dtype=torch.bool, device=device)
    if causal:
        see &= j <= i
        if prefix is not None:
            see |= (j < prefix[:, None, None])
    if docs is not None:
        dq = docs[:, Sk - Sq:]
        see &= (dq[:, :, None] == docs[:, None, :]) & (dq >= 0)[:, :, None]
    return see


def attention(q, k, v, do=None, causal=True, softcap=None, slopes=None, docs=None, prefix=None,
              scale=None, dtype=None):
    """float64 results {name: (value, bound)} of o, lse and, with do, dq, dk, dv.
    `dtype`: the kernel's element type (q's by default)."""
    dtype = dtype or q.dtype
    B, H, Sq, D = q.shape
    Hk, Sk = k.shape[1], k.shape[2]
    G = H // Hk
    scale = 1 / math.sqrt(D) if scale is None else scale
    u = unit(dtype) if dtype != torch.float32 else 0.0  # P and dS stay fp32 there
    out = unit(dtype)
    see = visible(B, Sq, Sk, causal, docs, prefix, q.device)[:, None]
    # contents of padding are nobody's business
    q, k, v = (t.double() for t in (q, k, v))
    if docs is not None:
        kp, qp = (docs < 0), (docs[:, Sk - Sq:] < 0)
        k, v = (t.masked_fill(kp[:, None, :, None], 0.0) for t in (k, v))
        q = q.masked_fill(qp[:, None, :, None], 0.0)
        if do is not None:
            do = do.masked_fill(qp[:, None, :, None], 0.0)
    kk, vv = (t.repeat_interleave(G, 1) for t in (k, v))
    z = (q @ kk.transpose(-1, -2)) * scale
    absz = (q.abs() @ kk.abs().transpose(-1, -2)) * scale
    # the product: D fp32 multiply-adds, then two roundings of the scaled score
    ez = (D + 2) * F32 * absz
    t = None
    if softcap:
        t = torch.tanh(z / softcap)
        z = softcap * t
        # |tanh'| <= 1; 1 - 2 / (1 + e): a few roundings of values up to 1 (16-bit
        # types), a few relative ones (fp32)
        ez = ez + softcap * 8 * F32 * (t.abs() + (1.0 if dtype != torch.float32 else 0.4))
    if slopes is not None:
        i = torch.arange(Sk - Sq, Sk, device=q.device, dtype=torch.float64)[:, None]
        j = torch.arange(Sk, device=q.device, dtype=torch.float64)[None, :]
        bias = slopes.double()[:, None, None] * (i - j).abs()
        z = z - bias
        ez = ez + 3 * F32 * bias.abs()
    ez = ez + 4 * F32 * z.abs()  # to log2 units and against the maximum
    z = z.masked_fill(~see, -math.inf)
    ez = ez.masked_fill(~see, 0.0)
    none = ~see.any(-1)
    lse = torch.logsumexp(z, -1)
    p = torch.exp(z - torch.where(none.expand(lse.shape), torch.zeros_like(lse), lse)[..., None])
    # a probability: its score's error and the row's (both at most max ez), the
    # exponential's few roundings, Sk additions in the sum
    e = 2 * ez.amax(-1, keepdim=True) + (8 + Sk) * F32
    e = e + 4 * F32 * torch.nan_to_num(lse, neginf=0.0).abs()[..., None]
    o = p @ vv
    mass = p @ vv.abs()
    # each P rounded by u, and the sum over them as rounded: 2 u of the mass
    tol_o = (2 * u + e) * mass + out * o.abs() + 1e-30
    res = {"o": (o, tol_o), "lse": (lse, (u + e[..., 0]) * 1.01 + 4 * F32 * torch.nan_to_num(
        lse, neginf=0.0).abs())}
    if do is None:
        return res
    do = do.double()
    dp = do @ vv.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # dP: D multiply-adds; delta: from the rounded O, D multiply-adds
    e_dp = (D + 1) * F32 * (do.abs() @ vv.abs().transpose(-1, -2))
    e_delta = (do.abs() * (tol_o + D * F32 * o.abs())).sum(-1, keepdim=True)
    tol_ds = p * ((e + u + 4 * F32) * (dp - delta).abs() + (1 + e) * (e_dp + e_delta))
    if softcap:
        deriv = 1 - t * t
        tol_ds = tol_ds * deriv + ds.abs() * 32 * F32
        ds = ds * deriv
    # smallest fp16 step: what dS and P lose below it
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    tol_ds = (tol_ds + tiny).masked_fill(~see, 0.0)
    n = (Sq * G + 8) * F32

    def grad(val, tol, mag, heads):
        if heads:
            val, tol, mag = (x.view(B, Hk, G, Sk, D).sum(2) for x in (val, tol, mag))
        return val, tol + n * mag + out * val.abs() + tiny + 1e-30

    dsT, tolT = ds.transpose(-1, -2), tol_ds.transpose(-1, -2)
    pT = (p * (u + e) + tiny).masked_fill(~see, 0.0).transpose(-1, -2)
    res["dq"] = grad(scale * (ds @ kk), scale * (tol_ds @ kk.abs()), scale * (ds.abs() @ kk.abs()), 0)
    res["dk"] = grad(scale * (dsT @ q), scale * (tolT @ q.abs()), scale * (dsT.abs() @ q.abs()), 1)
    res["dv"] = grad(p.transpose(-1, -2) @ do, pT @ do.abs(),
                     p.transpose(-1, -2) @ do.abs(), 1)
    return res


def within(name, got, want):
    """got within the bound of want = (value, bound); -inf only where it belongs."""
    val, tol = want
    g = got.detach().double()
    inf = torch.isinf(val)
    assert torch.equal(torch.isinf(g), inf), f"{name}: infinities elsewhere"
    err = (g - val).abs().masked_fill(inf, 0.0)
    assert not torch.isnan(err).any(), f"{name}: NaN"
    over = (err / tol.masked_fill(inf, 1.0)).max()
    assert float(over) <= 1.0, f"{name}: {float(over):.3f} of the bound, off by {float(err.max()):.3e}"


def turn(x, cos, sin, positions, interleaved, inverse=False):
    """x [S, B, H, D] with the first 2 * cos.shape[1] elements turned, float64."""
    S, B = x.shape[:2]
    pos = torch.arange(S, device=x.device) if positions is None else positions.long()
    pos = pos[:, None].expand(S, B) if pos.dim() == 1 else pos
    n = cos.shape[1]
    c, s = cos.double()[pos][:, :, None], sin.double()[pos][:, :, None]
    s = -s if inverse else s
    x = x.double()
    e, o = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    y = x.clone()
    a, b = e * c - o * s, e * s + o * c
    if interleaved:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = a, b
    else:
        y[..., :n], y[..., n:2 * n] = a, b
    return y


def pair_size(x, n, interleaved):
    """|e| + |o| of each element's pair, |x| beyond the turned ones."""
    a = x.abs()
    y = a.clone()
    if interleaved:
        m = a[..., 0:2 * n:2] + a[..., 1:2 * n:2]
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = m, m
    else:
        m = a[..., :n] + a[..., n:2 * n]
        y[..., :n], y[..., n:2 * n] = m, m
    return y


def rotary(x, cos, sin, positions, interleaved, inverse=False):
    """(value, bound): two products and a sum in fp32, one rounding."""
    y = turn(x, cos, sin, positions, interleaved, inverse)
    return y, unit(x.dtype) * y.abs() + 3 * F32 * pair_size(x.double(), cos.shape[1], interleaved) \
        + tiny(x.dtype)


def tiny(dtype):
    """Half the smallest step of the type (flushed or rounded away)."""
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}[dtype]


def norm_rotary(x, w, cos, sin, positions, interleaved, eps, dy=None):
    """{y, dx, dw: (value, bound)} of the normalised and turned heads."""
    D, n, u = x.shape[-1], cos.shape[1], unit(x.dtype)
    X, W = x.double(), w.double()
    r = 1 / torch.sqrt((X * X).mean(-1, keepdim=True) + eps)
    h = X * r
    # r: the sum of D squares in fp32 and three roundings, halved by the root
    er = (D / 2 + 6) * F32
    y = turn(h * W, cos, sin, positions, interleaved)
    res = {"y": (y, u * y.abs() + (er + 5 * F32) * pair_size(h * W, n, interleaved) + tiny(x.dtype))}
    if dy is None:
        return res
    d = turn(dy, cos, sin, positions, interleaved, inverse=True)
    ed = 3 * F32 * pair_size(dy.double(), n, interleaved)
    g = d * W
    m = (g * h).mean(-1, keepdim=True)
    dx = r * (g - h * m)
    em = ((ed * W.abs() * h.abs()) + (er + (D + 4) * F32) * (g * h).abs()).mean(-1, keepdim=True)
    tol = r * (ed * W.abs() + (er + 6 * F32) * (g.abs() + (h * m).abs()) + h.abs() * em
               + 2 * er * (h * m).abs())
    res["dx"] = (dx, u * dx.abs() + tol + tiny(x.dtype))
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    dw = (d * h).sum((0, 1, 2))
    # the additions: at most as deep as the rows are many, and no deeper than 4096
    # in the kernels' fixed order (rows of a group, groups, waves, parts)
    depth = min(rows, 4096) + 8
    tol = (ed * h.abs() + (er + depth * F32) * (d * h).abs()).sum((0, 1, 2))
    res["dw"] = (dw, unit(w.dtype) * dw.abs() + tol + tiny(w.dtype))
    return res
