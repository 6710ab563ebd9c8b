"""Rotary embedding at given positions and the norm in front of it, against float64."""
import pytest
import torch

import scored_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(S, B, H, Hk, D, dtype, seed, device, T=None, R=None, tab=None, layout="qkv"):
    g = torch.Generator().manual_seed(seed)
    R = R or D
    if layout == "qkv":  # cut from a fused projection
        x = torch.randn(S, B, (H + 2 * Hk) * D, generator=g).to(dtype).to(device)
        q, k = x[..., :H * D].view(S, B, H, D), x[..., H * D:(H + Hk) * D].view(S, B, Hk, D)
    elif layout == "bshd":
        q, k = (torch.randn(B, S, n, D, generator=g).to(dtype).to(device).transpose(0, 1)
                for n in (H, Hk))
    elif layout == "odd":  # unaligned rows, every other element
        q, k = (torch.randn(S, B, n, 2 * D + 1, generator=g).to(dtype).to(device)[..., 1::2]
                for n in (H, Hk))
    T = T or S
    freqs = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    a = torch.outer(torch.arange(T, dtype=torch.float64), freqs)
    tab = tab or dtype
    cos, sin = (t.to(tab).to(device) for t in (a.cos(), a.sin()))
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(device) for _ in range(2)]
    dy = [torch.randn(S, B, n, D, generator=g).to(dtype).to(device) for n in (H, Hk)]
    pos = torch.randint(0, T, (S, B), generator=g)
    return q, k, cos, sin, w, dy, pos


SIZES = [  # S, B, H, Hk, D, R
    (1, 1, 1, 1, 64, 64), (1, 7, 12, 4, 128, 128), (5, 2, 3, 1, 64, 32), (37, 3, 5, 5, 80, 80),
    (130, 2, 9, 3, 128, 64), (64, 1, 4, 2, 256, 256), (3, 2, 2, 1, 16, 16), (17, 3, 5, 2, 10, 6),
    (9, 1, 3, 3, 96, 20), (2, 2, 1, 1, 2, 2), (33, 2, 2, 1, 512, 512), (11, 2, 3, 1, 24, 24)]


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_rotary(gpu, size, dtype, interleaved):
    from gpt_from_scratch_amd import apply_rotary_qk
    S, B, H, Hk, D, R = size
    for where in ("none", "row", "each"):
        q, k, cos, sin, _, dy, pos = make(S, B, H, Hk, D, dtype, S + D, gpu, T=S + 5, R=R)
        p = {"none": None, "row": pos[:, 0].to(gpu), "each": pos.int().to(gpu)}[where]
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        y = apply_rotary_qk(q, k, cos, sin, p, interleaved)
        dx = torch.autograd.grad(y, (q, k), dy)
        for i, x in enumerate((q, k)):
            assert y[i].shape == x.shape and y[i].dtype == dtype
            ref.within(f"y{i} {where}", y[i], ref.rotary(x.detach(), cos, sin, p, interleaved))
            ref.within(f"d{i} {where}", dx[i], ref.rotary(dy[i], cos, sin, p, interleaved, True))


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_norm_rotary(gpu, size, dtype, interleaved):
    from gpt_from_scratch_amd import qk_norm_rotary
    S, B, H, Hk, D, R = size
    for where, wt in (("none", dtype), ("each", torch.float32)):
        q, k, cos, sin, w, dy, pos = make(S, B, H, Hk, D, dtype, 2 * S + D, gpu, T=S + 5, R=R)
        p = pos.to(gpu) if where == "each" else None
        w = [t.to(wt).requires_grad_() for t in w]
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        y = qk_norm_rotary(q, k, *w, cos, sin, 1e-5, p, interleaved)
        got = torch.autograd.grad(y, (q, k, *w), dy)
        for i, x in enumerate((q, k)):
            want = ref.norm_rotary(x.detach(), w[i].detach(), cos, sin, p, interleaved, 1e-5, dy[i])
            assert y[i].dtype == dtype and got[2 + i].dtype == wt
            ref.within(f"y{i}", y[i], want["y"])
            ref.within(f"dx{i}", got[i], want["dx"])
            ref.within(f"dw{i}", got[2 + i], want["dw"])


@pytest.mark.parametrize("layout", ["qkv", "bshd", "odd"])
@pytest.mark.parametrize("tab", TYPES)
def test_layouts_and_tables(gpu, layout, tab):
    """Inputs of other strides and alignments, tables of other types and strides:
    the same bits as from dense copies with the same tables."""
    from gpt_from_scratch_amd import apply_rotary_qk, qk_norm_rotary
    q, k, cos, sin, w, dy, pos = make(21, 2, 6, 2, 64, torch.bfloat16, 3, gpu, T=40, tab=tab,
                                      layout=layout)
    pos = pos.to(gpu)
    w = [t.bfloat16() for t in w]
    wide = torch.cat((cos, sin, cos[:, :1]), 1)  # rows of odd length
    tabs = [(cos, sin), (cos.t().contiguous().t(), sin.t().contiguous().t()),
            (wide[:, :32], wide[:, 32:64])]
    base = apply_rotary_qk(q.contiguous(), k.contiguous(), cos, sin, pos)
    normed = qk_norm_rotary(q.contiguous(), k.contiguous(), *w, cos, sin, 1e-6, pos)
    for c, s in tabs:
        for p in (pos, pos.t().contiguous().t(), pos.int()):
            y = apply_rotary_qk(q, k, c, s, p)
            assert all(torch.equal(a, b) for a, b in zip(y, base))
        # the sum of squares may be added in another order
        for i, y in enumerate(qk_norm_rotary(q, k, *w, c, s, 1e-6, pos)):
            x = (q, k)[i]
            ref.within("norm", y, ref.norm_rotary(x, w[i], cos, sin, pos, True, 1e-6)["y"])
            assert float((y != normed[i]).float().mean()) < 0.02
    # gradients of any layout
    qr, kr = (t.detach().requires_grad_() for t in (q, k))
    y = apply_rotary_qk(qr, kr, cos, sin, pos)
    g = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in dy]
    a = torch.autograd.grad(y, (qr, kr), g, retain_graph=True)
    b = torch.autograd.grad(y, (qr, kr), dy, retain_graph=True)
    assert all(torch.equal(x, z) for x, z in zip(a, b))
    one = torch.ones((), device=gpu, dtype=torch.bfloat16)
    c = torch.autograd.grad(y, (qr, kr), [one.expand(t.shape) for t in dy])
    ref.within("ones", c[0], ref.rotary(torch.ones_like(dy[0]), cos, sin, pos, True, True))


def test_matches_apply_rope_qk(gpu):
    """The form both have gives the same bits."""
    from gpt_from_scratch_amd import apply_rope_qk, apply_rotary_qk
    q, k, cos, sin, _, _, _ = make(65, 2, 6, 6, 64, torch.bfloat16, 5, gpu)
    for a, b in zip(apply_rope_qk(q, k, cos, sin), apply_rotary_qk(q, k, cos, sin)):
        assert torch.equal(a, b)


def test_positions_outside_the_tables(gpu):
    from gpt_from_scratch_amd import apply_rotary_qk, qk_norm_rotary
    q, k, cos, sin, w, _, _ = make(6, 1, 2, 1, 64, torch.bfloat16, 7, gpu, T=10, R=32)
    pos = torch.tensor([0, 9, 10, -1, 2 ** 40, -2 ** 60], device=gpu)
    w = [t.bfloat16() for t in w]
    for y in (apply_rotary_qk(q, k, cos, sin, pos),
              qk_norm_rotary(q, k, *w, cos, sin, positions=pos)):
        for t in y:
            assert not torch.isnan(t[:2]).any() and not torch.isnan(t[..., 32:]).any()
            assert torch.isnan(t[2:, ..., :32]).all()


def test_zero_rows_and_eps(gpu):
    from gpt_from_scratch_amd import qk_norm_rotary
    q, k, cos, sin, w, dy, _ = make(4, 2, 3, 1, 64, torch.float32, 8, gpu)
    q = q.detach().clone().zero_().requires_grad_()
    y = qk_norm_rotary(q, k, *w, cos, sin, eps=1e-6)
    assert not y[0].any()
    (dq,) = torch.autograd.grad(y, (q,), dy)
    ref.within("dq", dq, ref.norm_rotary(q.detach(), w[0], cos, sin, None, True, 1e-6, dy[0])["dx"])


def test_gradient_by_differences(gpu):
    """Central differences of the fp32 operator along random directions.  f is the
    sum over N outputs of y * dy, its value off by at most a few F32 per term; the
    difference divides that by h, and h^2 of the third derivative stays below it."""
    from gpt_from_scratch_amd import qk_norm_rotary
    q, k, cos, sin, w, dy, pos = make(7, 2, 3, 2, 64, torch.float32, 9, gpu, T=20, R=32)
    pos = pos.to(gpu)
    xs = [t.detach().clone().requires_grad_() for t in (q, k, *w)]

    def f(args):
        y = qk_norm_rotary(*args, cos, sin, 1e-6, pos, False)
        return sum((a.double() * b.double()).sum() for a, b in zip(y, dy))

    grads = torch.autograd.grad(f(xs), xs)
    h = 2.0 ** -6
    g = torch.Generator().manual_seed(1)
    for i in range(4):
        v = torch.randn(xs[i].shape, generator=g).to(gpu)
        v = v / v.norm()
        with torch.no_grad():
            at = [f([x + s * h * v if j == i else x for j, x in enumerate(xs)]) for s in (1, -1)]
        diff = (at[0] - at[1]) / (2 * h)
        want = (grads[i].double() * v.double()).sum()
        size = sum((a.double() * b.double()).abs().sum() for a, b in
                   zip(qk_norm_rotary(*xs, cos, sin, 1e-6, pos, False), dy))
        # 40 roundings per term at worst, both values; h^2 / 6 of a third derivative
        # of at most 6 * 64 |dy| |v|^3 / |x|^3 < 6 per row
        tol = 40 * ref.F32 * size / h + h * h
        assert abs(float(diff - want)) <= float(tol)


def test_streams_and_graph(gpu):
    """Another stream than the default one, and captured calls replayed on new
    contents with eager work in between."""
    from gpt_from_scratch_amd import qk_norm_rotary
    q, k, cos, sin, w, dy, _ = make(50, 2, 4, 2, 128, torch.bfloat16, 11, gpu)
    w = [t.bfloat16().requires_grad_() for t in w]
    q, k = (t.detach().clone().requires_grad_() for t in (q, k))

    def call():
        y = qk_norm_rotary(q, k, *w, cos, sin)
        return tuple(t.detach() for t in y) + torch.autograd.grad(y, (q, k, *w), dy)

    want = call()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = call()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, call()))


def test_captured_backward_of_live_leaves_is_refused(gpu):
    """While an eager graph of the same leaves is alive, a captured backward would
    leave the capture: an error instead, and the process goes on."""
    from gpt_from_scratch_amd import apply_rotary_qk, qk_norm_rotary, scored_attn
    q, k, cos, sin, w, dy, _ = make(16, 2, 4, 2, 64, torch.bfloat16, 12, gpu)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, *(t.bfloat16() for t in w))]

    def attn():
        b = [t.permute(1, 2, 0, 3) for t in (q, k, k)]
        b[0] = x4
        return (scored_attn(*b),)

    x4 = q.permute(1, 2, 0, 3).contiguous().requires_grad_()
    for call, wrt, g in ((lambda: apply_rotary_qk(*leaves[:2], cos, sin), leaves[:2], dy),
                         (lambda: qk_norm_rotary(*leaves, cos, sin), leaves, dy),
                         (attn, [x4], [torch.ones_like(x4)])):
        alive = call()
        with pytest.raises(RuntimeError, match="captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(call(), wrt, g)
        torch.cuda.synchronize()
        # without it, or outside a capture, as ever
        want = torch.autograd.grad(call(), wrt, g)
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(call(), wrt, g)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
