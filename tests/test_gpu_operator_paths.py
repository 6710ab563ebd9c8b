"""Rotary embedding and attention with modified scores: sizes that fill the GPU, the
autograd functions in Python against the nodes in C++, tensors handed over twice and
saved tensors that went elsewhere in between."""
import pytest
import torch

import scored_ref as ref
import test_scored_checks as checks
from test_gpu_scored_attn import documents, randn, run

pytestmark = pytest.mark.gpu

# Grids of more than 512 tiles: no waves share a row, chains are not split; the
# float64 form holds [B, H, S, S].
LARGE = {
    "plain_64": dict(size=(4, 16, 4, 1100, 1100, 64)),
    "plain_128": dict(size=(2, 16, 4, 1500, 1500, 128)),
    "cap_bias": dict(size=(2, 12, 12, 1500, 1500, 64), cap=30.0, bias=1.0),
    "full_128": dict(size=(3, 8, 2, 1409, 1409, 128), causal=False, cap=50.0),
    "docs_64": dict(size=(5, 8, 8, 1300, 1300, 64), docs="packed"),
    "docs_128": dict(size=(3, 12, 4, 1300, 1300, 128), docs="packed", bias=1.0),
    "mixed": dict(size=(3, 12, 4, 1300, 1300, 64), docs="mixed", causal=False),
    "prefix": dict(size=(3, 12, 12, 1025, 1025, 128), prefix=700),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("name", list(LARGE))
def test_large_grids(gpu, name, dtype):
    run(LARGE[name], dtype, gpu)


def _attn_inputs(gpu, dtype, B=2, H=4, Hk=2, S=200, D=64):
    q = randn((B, H, S, D), 1, dtype, gpu).requires_grad_()
    k, v = (randn((B, Hk, S, D), i, dtype, gpu).requires_grad_() for i in (2, 3))
    slopes = (0.5 ** torch.arange(1, H + 1, dtype=torch.float32)).to(gpu)
    return (q, k, v), randn((B, H, S, D), 4, dtype, gpu), slopes, documents(B, S, "packed", 5, gpu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("which", ["plain", "cap", "slopes", "docs", "prefix", "all"])
def test_scored_attn_python_path(gpu, dtype, which):
    from gpt_from_scratch_amd import ScoredAttn, scored_attn
    x, do, slopes, ids = _attn_inputs(gpu, dtype)
    pre = torch.tensor([50, 0], dtype=torch.int32, device=gpu)
    on = lambda n, v: v if which in (n, "all") else None  # noqa: E731
    how = (True, on("cap", 20.0), on("slopes", slopes), on("docs", ids), on("prefix", pre))
    a = scored_attn(*x, *how, 0.2)
    b = ScoredAttn.apply(*x, *how, 0.2)
    assert type(a.grad_fn) is not type(b.grad_fn)
    assert torch.equal(a, b)
    for g, h in zip(torch.autograd.grad(a, x, do), torch.autograd.grad(b, x, do)):
        assert torch.equal(g, h)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("positions", [False, True])
def test_rotary_python_path(gpu, interleaved, positions):
    from gpt_from_scratch_amd import QKNormRotary, RotaryQK, apply_rotary_qk, qk_norm_rotary
    S, B, D = 37, 2, 64
    q, k = (randn((S, B, n, D), n, torch.bfloat16, gpu).requires_grad_() for n in (6, 3))
    wq, wk = (randn((D,), i, torch.float32, gpu).requires_grad_() for i in (8, 9))
    a = torch.rand(90, 16, generator=torch.Generator().manual_seed(1)).to(gpu) * 6
    cos, sin = a.cos(), a.sin()
    pos = torch.randint(0, 90, (S, B), generator=torch.Generator().manual_seed(2)).to(gpu) \
        if positions else None
    dy = [randn(t.shape, 20 + i, torch.bfloat16, gpu) for i, t in enumerate((q, k))]
    pairs = [(apply_rotary_qk(q, k, cos, sin, pos, interleaved),
              RotaryQK.apply(q, k, cos, sin, pos, interleaved), (q, k)),
             (qk_norm_rotary(q, k, wq, wk, cos, sin, 1e-5, pos, interleaved),
              QKNormRotary.apply(q, k, wq, wk, cos, sin, pos, interleaved, 1e-5), (q, k, wq, wk))]
    for x, y, leaves in pairs:
        assert type(x[0].grad_fn) is not type(y[0].grad_fn)
        assert all(torch.equal(s, t) for s, t in zip(x, y))
        for g, h in zip(torch.autograd.grad(x, leaves, dy), torch.autograd.grad(y, leaves, dy)):
            assert g.dtype == h.dtype and torch.equal(g, h)


def test_one_output_unused(gpu):
    """Only q's (or k's) result has a gradient: the other's is zero."""
    from gpt_from_scratch_amd import apply_rotary_qk, qk_norm_rotary
    S, B, D = 20, 2, 64
    q, k = (randn((S, B, n, D), n, torch.bfloat16, gpu).requires_grad_() for n in (4, 2))
    w = randn((D,), 3, torch.float32, gpu).requires_grad_()
    a = torch.rand(S, 32, generator=torch.Generator().manual_seed(1)).to(gpu)
    dy = [randn(t.shape, 20 + i, torch.bfloat16, gpu) for i, t in enumerate((q, k))]
    for f in (lambda: apply_rotary_qk(q, k, a.cos(), a.sin()),
              lambda: qk_norm_rotary(q, k, w, w, a.cos(), a.sin())):
        both = torch.autograd.grad(f(), (q, k), dy)
        for i in (0, 1):
            got = torch.autograd.grad(f()[i], (q, k), dy[i], allow_unused=True)
            assert torch.equal(got[i], both[i])
            assert got[1 - i] is None or not got[1 - i].any()


def test_the_same_tensor_twice(gpu):
    from gpt_from_scratch_amd import apply_rotary_qk, decode_attn, qk_norm_rotary, scored_attn
    x = randn((2, 3, 150, 64), 1, torch.float32, gpu).requires_grad_()
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    do = randn(x.shape, 2, torch.float32, gpu)
    o, p = scored_attn(x, x, x, softcap=20.0), scored_attn(*parts, softcap=20.0)
    assert torch.equal(o, p)
    got, = torch.autograd.grad(o, x, do)
    g = torch.autograd.grad(p, parts, do)
    torch.testing.assert_close(got, g[0] + g[1] + g[2], rtol=0,
                               atol=4 * ref.F32 * float(sum(t.abs().max() for t in g)))
    with torch.no_grad():
        assert torch.equal(decode_attn(x[:, :, 0], x, x), decode_attn(x[:, :, 0].clone(), x, x.clone()))
    y = randn((20, 2, 4, 64), 3, torch.bfloat16, gpu)
    w = randn((64,), 4, torch.bfloat16, gpu)
    a = torch.rand(20, 32, generator=torch.Generator().manual_seed(1)).to(gpu)
    for f in (lambda q, k: apply_rotary_qk(q, k, a.cos(), a.sin()),
              lambda q, k: qk_norm_rotary(q, k, w, w, a.cos(), a.sin())):
        assert torch.equal(*f(y, y)) and torch.equal(f(y, y)[0], f(y, y.clone())[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_saved_tensors_kept_on_the_host(gpu, dtype):
    from gpt_from_scratch_amd import qk_norm_rotary, scored_attn
    x, do, slopes, ids = _attn_inputs(gpu, dtype)
    S, B = 30, 2
    q, k = (randn((S, B, n, 64), n, dtype, gpu).requires_grad_() for n in (4, 2))
    w = randn((64,), 3, torch.float32, gpu).requires_grad_()
    a = torch.rand(S, 32, generator=torch.Generator().manual_seed(1)).to(gpu)
    dy = [randn(t.shape, 20 + i, dtype, gpu) for i, t in enumerate((q, k))]

    def grads():
        o = scored_attn(*x, softcap=20.0, slopes=slopes, document_ids=ids)
        y = qk_norm_rotary(q, k, w, w, a.cos(), a.sin())
        return lambda: torch.autograd.grad(o, x, do) + torch.autograd.grad(y, (q, k, w), dy)

    want = grads()()
    with torch.autograd.graph.save_on_cpu():
        later = grads()
    assert all(torch.equal(s, t) for s, t in zip(later(), want))


def test_changed_inputs_are_noticed(gpu):
    """What the backward reads may not change in between."""
    from gpt_from_scratch_amd import qk_norm_rotary, scored_attn
    (q, k, v), do, _, _ = _attn_inputs(gpu, torch.bfloat16)
    o = scored_attn(q, k, v)
    with torch.no_grad():
        k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(o, (q, k, v), do)
    x = randn((9, 2, 4, 64), 1, torch.bfloat16, gpu).requires_grad_()
    w = randn((64,), 3, torch.float32, gpu).requires_grad_()
    a = torch.rand(9, 32).to(gpu)
    y = qk_norm_rotary(x, x, w, w, a.cos(), a.sin())
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, (x, w), [t.detach() for t in y])


def test_second_derivatives_are_refused(gpu):
    from gpt_from_scratch_amd import scored_attn
    x, do, _, _ = _attn_inputs(gpu, torch.float32)
    o = scored_attn(*x)
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(o, x[:1], do.requires_grad_(), create_graph=True)
        torch.autograd.grad(g.sum(), do)


def test_gradients_of_some_inputs(gpu):
    from gpt_from_scratch_amd import scored_attn
    x, do, _, ids = _attn_inputs(gpu, torch.bfloat16)
    want = torch.autograd.grad(scored_attn(*x, document_ids=ids), x, do)
    for i in range(3):
        y = [t if i == j else t.detach() for j, t in enumerate(x)]
        got, = torch.autograd.grad(scored_attn(*y, document_ids=ids), y[i], do)
        assert torch.equal(got, want[i])
    # a gradient that is one value expanded, and one of other strides
    o = scored_attn(*x, document_ids=ids)
    got = torch.autograd.grad(o.sum(), x, retain_graph=True)
    dense = torch.autograd.grad(o, x, torch.ones_like(o), retain_graph=True)
    assert all(torch.equal(s, t) for s, t in zip(got, dense))
    turned = torch.autograd.grad(o, x, do.transpose(1, 2).contiguous().transpose(1, 2))
    assert all(torch.equal(s, t) for s, t in zip(turned, want))


def test_prefixes_of_any_value(gpu):
    """Negative ones are none, ones past the end are all keys."""
    from gpt_from_scratch_amd import scored_attn
    x, do, _, _ = _attn_inputs(gpu, torch.bfloat16)
    x = [torch.cat((t, t)).detach().requires_grad_() for t in x]
    do = torch.cat((do, do))
    pre = torch.tensor([-2 ** 31, -1, 2 ** 31 - 1, 200], dtype=torch.int32, device=gpu)
    o = scored_attn(*x, prefix_lens=pre)
    want = ref.attention(*(t.detach() for t in x), do, prefix=pre)
    for n, g in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, x, do))):
        ref.within(n, g, want[n])


def test_more_rows_than_one_wave_each(gpu):
    """Heads of 4 elements, which no 16-byte chunk holds: 7e7 rows, past 2^32 threads."""
    from gpt_from_scratch_amd import apply_rotary_qk
    S, H = 1 << 21, 31
    q, k = (randn((8, 1, n, 4), n, torch.float32, gpu).repeat(S // 8, 1, 1, 1) for n in (H, 2))
    a = torch.rand(8, 2, generator=torch.Generator().manual_seed(1)).to(gpu).repeat(S // 8, 1)
    cos, sin = a.cos(), a.sin()
    for x, y in zip((q, k), apply_rotary_qk(q, k, cos, sin)):
        first = ref.rotary(x[:8], cos[:8], sin[:8], None, True)
        ref.within("first", y[:8], first)
        assert torch.equal(y, y[:8].repeat(S // 8, 1, 1, 1))


def _moved(kw, device):
    out = {n: t.detach().to(device).requires_grad_(t.requires_grad)
           if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
    return out


@pytest.mark.parametrize("kw,error,text", [c for c in checks.ROTARY if c[0]])
def test_rotary_refuses_on_the_gpu(gpu, kw, error, text):
    from gpt_from_scratch_amd import apply_rotary_qk, qk_norm_rotary
    a = _moved(checks._rotary(**kw), gpu)
    with pytest.raises(error, match=text):
        apply_rotary_qk(**a)
    w = torch.ones(a["q"].shape[-1], device=gpu)
    with pytest.raises(error, match=text):
        qk_norm_rotary(q_weight=w, k_weight=w, **a)


@pytest.mark.parametrize("kw,error,text", [c for c in checks.ATTN + checks.MASKS if c[0]] + [
    checks.SLOPES_GRAD, (dict(k=torch.zeros(2, 0, 32, 64), v=torch.zeros(2, 0, 32, 64)), ValueError,
                         "no size 0")])
def test_scored_attn_refuses_on_the_gpu(gpu, kw, error, text):
    from gpt_from_scratch_amd import scored_attn, scored_attn_forward
    a = _moved(checks._attn(**kw), gpu)
    with pytest.raises(error, match=text):
        scored_attn(**a)
    if text != checks.SLOPES_GRAD[2]:
        with pytest.raises(error, match=text):
            scored_attn_forward(**a)


@pytest.mark.parametrize("which", ["k", "v", "slopes", "document_ids", "prefix_lens"])
def test_tensors_elsewhere_are_refused(gpu, which):
    from gpt_from_scratch_amd import scored_attn
    a = checks._attn(slopes=torch.zeros(4), document_ids=torch.zeros(2, 32, dtype=torch.int32),
                     prefix_lens=torch.zeros(2, dtype=torch.int32))
    b = _moved(a, gpu)
    scored_attn(**b)
    b[which] = a[which]
    with pytest.raises(RuntimeError):
        scored_attn(**b)


def test_batches_past_32_bits(gpu):
    """Sequences 2^31 elements apart: forward, backward, rotation and norm."""
    from gpt_from_scratch_amd import qk_norm_rotary, scored_attn
    B, S, D, far = 2, 70, 64, 2 ** 31 + 64

    def apart(n, seed):
        big = torch.empty(far + n * S * D, dtype=torch.bfloat16, device=gpu)
        t = big.as_strided((S, B, n, D), (n * D, far, D, 1))
        t.copy_(randn((S, B, n, D), seed, torch.bfloat16, gpu))
        return t

    q, k, v, g = (apart(n, i) for i, n in enumerate((4, 2, 2, 4)))
    w = randn((D,), 9, torch.float32, gpu)
    a = torch.rand(S, D // 2, generator=torch.Generator().manual_seed(1)).to(gpu)

    def call(q, k, v, g):
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        qr, kr = qk_norm_rotary(x[0], x[1], w, w, a.cos(), a.sin())
        o = scored_attn(qr.permute(1, 2, 0, 3), kr.permute(1, 2, 0, 3), x[2].permute(1, 2, 0, 3))
        direct = scored_attn(*(t.permute(1, 2, 0, 3) for t in x), softcap=20.0)
        do = g.permute(1, 2, 0, 3)
        return (o, *torch.autograd.grad(o, x, do), direct, *torch.autograd.grad(direct, x, do))

    for s, t in zip(call(q, k, v, g), call(*(t.contiguous() for t in (q, k, v, g)))):
        assert torch.equal(s, t)


def test_two_threads(gpu):
    """Two host threads, each on its own stream: the bits of one after the other."""
    import threading
    from gpt_from_scratch_amd import decode_attn, qk_norm_rotary, scored_attn
    a = torch.rand(300, 32, generator=torch.Generator().manual_seed(1)).to(gpu)
    cos, sin = a.cos(), a.sin()
    w = randn((64,), 9, torch.float32, gpu)
    data = []
    for i in range(2):
        x = [randn((300, 2, n, 64), 10 * i + n, torch.bfloat16, gpu) for n in (8, 2, 2)]
        data.append((x, documents(2, 300, "packed", i, gpu), randn((2, 8, 300, 64), 40 + i,
                                                                     torch.bfloat16, gpu)))

    def work(x, ids, do):
        x = [t.detach().requires_grad_() for t in x]
        q, k = qk_norm_rotary(x[0], x[1], w, w, cos, sin)
        q, k, v = (t.permute(1, 2, 0, 3) for t in (q, k, x[2]))
        o = scored_attn(q, k, v, document_ids=ids)
        with torch.no_grad():
            d = decode_attn(q[:, :, -1], k, v)
        return (o.detach(), d, *torch.autograd.grad(o, x, do))

    want = [work(*d) for d in data]
    torch.cuda.synchronize()
    bad = []

    def run_on(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                got = work(*data[i])
                st.synchronize()
                if not all(torch.equal(s, t) for s, t in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=run_on, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
