"""Attention with modified scores and its single-token form, against float64."""
import pytest
import torch

import scored_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def randn(shape, seed, dtype, device, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(device)


def heads(B, n, S, D, seed, dtype, device, layout, std=1.0):
    if layout == "dense":
        return randn((B, n, S, D), seed, dtype, device, std)
    if layout == "model":  # [S, B, heads, D] as the projections give them
        return randn((S, B, n, D), seed, dtype, device, std).permute(1, 2, 0, 3)
    if layout == "odd":  # rows that are not 16-byte aligned: copied
        return randn((B, n, S, D + 3), seed, dtype, device, std)[..., 1:D + 1]
    assert layout == "strided"  # a part of a wider tensor, every other row
    return randn((B, 2 * S, n, 2 * D), seed, dtype, device, std)[:, ::2, :, D:].transpose(1, 2)


def documents(B, S, kind, seed, device):
    """[B, S] ids: "packed" in order with padding behind, "random" in any order,
    "mixed" interleaved with padding between, "one" document, "empty" sequences."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.zeros(B, S, dtype=torch.int32)
    for b in range(B):
        if kind == "packed":
            end = S - int(torch.randint(0, max(1, S // 4), (1,), generator=g))
            cuts = torch.randint(0, end + 1, (5,), generator=g).sort().values
            ids[b] = torch.bucketize(torch.arange(S), cuts, right=True) + 7
            ids[b, end:] = -1
        elif kind == "random":
            ids[b] = torch.randint(0, 3, (S,), generator=g)
        elif kind == "mixed":
            ids[b] = torch.randint(-2, 4, (S,), generator=g)
            ids[b, S // 3: S // 2] = -2 ** 31
        elif kind == "empty":
            ids[b] = -1 if b % 2 == 0 else 2 ** 31 - 1
    return ids.to(device)


def run(c, dtype, device, seed=1, grad=True):
    from gpt_from_scratch_amd import scored_attn, scored_attn_forward
    B, H, Hk, Sq, Sk, D = c["size"]
    lay = c.get("layout", "model")
    q = heads(B, H, Sq, D, seed, dtype, device, lay, 1.5)
    k, v = (heads(B, Hk, Sk, D, seed + i, dtype, device, lay, s) for i, s in ((1, 1.5), (2, 1.0)))
    do = randn((B, H, Sq, D), seed + 3, dtype, device)
    how = dict(causal=c.get("causal", True), softcap=c.get("cap"))
    if c.get("bias"):
        how["slopes"] = (2.0 ** -torch.arange(1, H + 1, dtype=torch.float32)).to(device) * c["bias"]
    if c.get("docs"):
        how["document_ids"] = documents(B, Sk, c["docs"], seed, device)
    if c.get("prefix") is not None:
        how["prefix_lens"] = torch.tensor([(c["prefix"] + 29 * b) for b in range(B)],
                                          dtype=torch.int32, device=device)
    if c.get("scale"):
        how["softmax_scale"] = c["scale"]
    q, k, v = (t.detach().requires_grad_(grad) for t in (q, k, v))
    got = {}
    got["o"], got["lse"] = (t.clone() for t in scored_attn_forward(q, k, v, **how))
    if grad:
        o = scored_attn(q, k, v, **how)
        assert torch.equal(o, got["o"])
        got.update(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)))
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            assert got[n].shape == t.shape and got[n].dtype == dtype
    want = ref.attention(q.detach(), k.detach(), v.detach(), do if grad else None, how["causal"],
                         how["softcap"], how.get("slopes"), how.get("document_ids"),
                         how.get("prefix_lens"), how.get("softmax_scale"))
    for n in got:
        ref.within(n, got[n], want[n])
    return got


CASES = {
    # sizes: one token, ends of tiles, head counts and dims
    "s1": dict(size=(2, 3, 1, 1, 1, 64)),
    "s2": dict(size=(1, 2, 2, 2, 2, 8)),
    "s31": dict(size=(1, 4, 2, 31, 31, 16)),
    "s33": dict(size=(2, 2, 2, 33, 33, 128)),
    "s63": dict(size=(1, 6, 2, 63, 63, 40), layout="dense"),
    "s64": dict(size=(1, 2, 1, 64, 64, 64)),
    "s65": dict(size=(2, 3, 3, 65, 65, 80), layout="odd"),
    "s127": dict(size=(1, 2, 2, 127, 127, 96), layout="strided"),
    "s128": dict(size=(1, 8, 1, 128, 128, 128)),
    "s129": dict(size=(1, 5, 5, 129, 129, 72)),
    "s300": dict(size=(2, 4, 2, 300, 300, 64), layout="strided"),
    "s1000": dict(size=(1, 3, 1, 1000, 1000, 128)),
    "full_s200": dict(size=(2, 2, 1, 200, 200, 32), causal=False),
    "full_s129": dict(size=(1, 4, 4, 129, 129, 128), causal=False),
    # queries at the end of longer keys
    "late_1": dict(size=(2, 4, 2, 1, 333, 64)),
    "late_70": dict(size=(1, 2, 2, 70, 200, 128)),
    "late_full": dict(size=(1, 4, 2, 130, 131, 64), causal=False),
    "late_docs": dict(size=(2, 2, 1, 150, 301, 64), docs="packed"),
    "late_mixed": dict(size=(2, 2, 1, 77, 301, 128), docs="mixed", prefix=40, bias=1.0),
    # scores
    "cap": dict(size=(1, 4, 2, 300, 300, 128), cap=30.0),
    "cap_tight": dict(size=(1, 2, 2, 200, 200, 64), cap=1.5, causal=False),
    "cap_far": dict(size=(1, 2, 1, 130, 130, 64), cap=20.0, scale=2.0),
    "bias": dict(size=(2, 6, 2, 300, 300, 64), bias=1.0),
    "bias_full": dict(size=(1, 4, 4, 257, 257, 128), bias=1.0, causal=False),
    "bias_up": dict(size=(1, 3, 3, 150, 150, 64), bias=-0.25),
    "cap_bias": dict(size=(1, 4, 2, 190, 190, 128), cap=20.0, bias=1.0),
    "cap_bias_64": dict(size=(1, 4, 2, 190, 190, 64), cap=20.0, bias=1.0, causal=False),
    "scale": dict(size=(1, 2, 2, 100, 100, 64), scale=0.37),
    # masks
    "prefix_0": dict(size=(2, 2, 2, 130, 130, 64), prefix=0),
    "prefix_63": dict(size=(3, 2, 1, 200, 200, 64), prefix=63),
    "prefix_64": dict(size=(2, 2, 1, 300, 300, 128), prefix=64),
    "prefix_over": dict(size=(2, 2, 2, 100, 100, 64), prefix=90),
    "prefix_bias": dict(size=(1, 2, 2, 200, 200, 64), prefix=100, bias=1.0, cap=50.0),
    "packed": dict(size=(3, 4, 2, 500, 500, 64), docs="packed"),
    "packed_128": dict(size=(2, 2, 1, 500, 500, 128), docs="packed", cap=50.0),
    "packed_full": dict(size=(2, 2, 2, 400, 400, 64), docs="packed", causal=False),
    "random": dict(size=(2, 2, 2, 150, 150, 128), docs="random"),
    "mixed": dict(size=(2, 4, 2, 300, 300, 64), docs="mixed", bias=1.0),
    "mixed_full": dict(size=(2, 2, 2, 200, 200, 128), docs="mixed", causal=False),
    "one_doc": dict(size=(1, 2, 2, 300, 300, 64), docs="one"),
    "empty": dict(size=(3, 2, 1, 140, 140, 64), docs="empty"),
    "prefix_docs": dict(size=(2, 3, 1, 300, 300, 128), docs="packed", prefix=100),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", list(CASES))
def test_scored_attn(gpu, name, dtype):
    run(CASES[name], dtype, gpu)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_keys(gpu, dtype):
    """More than 64 key tiles, so that the list of live tiles is looked up twice."""
    run(dict(size=(1, 2, 1, 70, 9000, 64), docs="packed"), dtype, gpu, grad=dtype != torch.float32)
    run(dict(size=(1, 1, 1, 200, 4500, 128), causal=False, cap=30.0), dtype, gpu)


def test_many_documents_as_if_alone(gpu):
    """A long packed sequence: each document gives what it gives alone, within the
    bounds of both (the two calls may split their sums differently)."""
    from gpt_from_scratch_amd import scored_attn_forward
    D, S = 64, 2048
    q, k, v = (randn((1, 4, S, D), i, torch.bfloat16, gpu) for i in range(3))
    ids = (torch.arange(S, dtype=torch.int32, device=gpu) // 256)[None]
    o, lse = scored_attn_forward(q, k, v, document_ids=ids)
    for a in range(0, S, 256):
        part = [t[:, :, a:a + 256] for t in (q, k, v)]
        want = ref.attention(*part)
        for got in ((o[:, :, a:a + 256], lse[:, :, a:a + 256]), scored_attn_forward(*part)):
            ref.within("o", got[0], want["o"])
            ref.within("lse", got[1], want["lse"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_padding_may_hold_anything(gpu, dtype, bad):
    """Rows of negative document id in q, k, v and do: no effect on any other row,
    zeros for their own."""
    from gpt_from_scratch_amd import scored_attn
    B, H, Hk, S, D = 2, 4, 2, 200, 64
    for kind in ("packed", "mixed"):
        ids = documents(B, S, kind, 3, gpu)
        pad = (ids < 0)[:, None, :, None]
        assert pad.any()
        q, k, v, do = (randn((B, n, S, D), i, dtype, gpu) for i, n in enumerate((H, Hk, Hk, H)))
        res = []
        for fill in (0.0, bad):
            x = [t.masked_fill(pad, fill).requires_grad_() for t in (q, k, v)]
            o = scored_attn(*x, document_ids=ids)
            res.append((o, *torch.autograd.grad(o, x, do.masked_fill(pad, fill))))
        for a, b in zip(*res):
            assert torch.equal(a, b)
            assert not a.masked_select(pad.expand(a.shape)).any()


def test_masked_scores_of_the_lowest_value(gpu):
    """Scores of -inf for visible keys weigh nothing; a row's first tiles may hold
    nothing else."""
    from gpt_from_scratch_amd import scored_attn_forward
    S, D = 300, 64
    q = torch.zeros(1, 1, S, D, device=gpu, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    k, v = (randn((1, 1, S, D), i, torch.bfloat16, gpu) for i in (1, 2))
    k[..., :, 0] = 1.0
    k[:, :, :130, 0] = -torch.inf
    o, lse = scored_attn_forward(q, k, v)
    assert not o[:, :, :130].any() and torch.isneginf(lse[:, :, :130]).all()
    mean = v[0, 0, 130:].double().cumsum(0) / torch.arange(1, S - 129, device=gpu)[:, None]
    # equal weights: P = 1 exactly, O rounded once
    err = (o[0, 0, 130:].double() - mean).abs()
    assert bool((err <= 2.0 ** -8 * mean.abs() + 2.0 ** -20).all())


def test_broadcast_inputs(gpu):
    """One key head seen by all through a zero stride, and a gradient of ones."""
    from gpt_from_scratch_amd import scored_attn
    B, H, S, D = 2, 4, 130, 64
    q = randn((B, H, S, D), 1, torch.bfloat16, gpu).requires_grad_()
    k1, v1 = (randn((B, 1, S, D), i, torch.bfloat16, gpu).requires_grad_() for i in (2, 3))
    do = torch.ones((), device=gpu, dtype=torch.bfloat16).expand(B, H, S, D)
    o = scored_attn(q, k1.expand(B, H, S, D), v1.expand(B, H, S, D))
    shared = scored_attn(q, k1, v1)
    assert torch.equal(o, shared)
    want = ref.attention(q.detach(), k1.detach(), v1.detach(), do)
    for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(shared, (q, k1, v1), do)):
        ref.within(n, g, want[n])
    # the sum over heads by autograd: each head's gradient rounded once more
    g = torch.autograd.grad(o, (k1, v1), do)
    full = ref.attention(q.detach(), k1.detach().expand(B, H, S, D), v1.detach().expand(B, H, S, D), do)
    for n, a in zip(("dk", "dv"), g):
        val, tol = full[n]
        ref.within(n, a, (val.sum(1, keepdim=True), tol.sum(1, keepdim=True)
                          + 4 * 2.0 ** -8 * val.abs().sum(1, keepdim=True)))


def test_repeats_bit_for_bit(gpu):
    c = dict(size=(2, 8, 2, 700, 700, 128), docs="packed", cap=30.0)
    a, b = (run(c, torch.bfloat16, gpu) for _ in range(2))
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_agrees_with_flash_attn(gpu):
    """The form both have."""
    from gpt_from_scratch_amd import apply_flash_attn, scored_attn
    x = [randn((2, 3, 257, 64), i, torch.bfloat16, gpu).requires_grad_() for i in range(3)]
    do = randn((2, 3, 257, 64), 9, torch.bfloat16, gpu)
    want = ref.attention(*(t.detach() for t in x), do)
    for f in (apply_flash_attn, scored_attn):
        o = f(*x)
        for n, g in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, x, do))):
            ref.within(n, g, want[n])


def test_gradient_by_differences(gpu):
    """Central differences of the fp32 forward, h = 2^-5 along unit directions.  The
    forward's bound summed over the outputs, twice, over 2 h, and h^2 / 6 times a
    third derivative: with |v| = 1 a score moves by at most scale |x_row| |v_row| (x
    either of q, k), a few units, and its third power enters once per output."""
    from gpt_from_scratch_amd import scored_attn
    B, H, Hk, S, D = 1, 2, 1, 90, 64
    how = dict(softcap=5.0, slopes=torch.tensor([0.1, 0.02], device=gpu),
               document_ids=documents(B, S, "packed", 5, gpu),
               prefix_lens=torch.tensor([20], dtype=torch.int32, device=gpu))
    x = [randn((B, n, S, D), i, torch.float32, gpu).requires_grad_()
         for i, n in enumerate((H, Hk, Hk))]
    do = randn((B, H, S, D), 4, torch.float32, gpu)

    def f(q, k, v):
        return (scored_attn(q, k, v, **how).double() * do.double()).sum()

    grads = torch.autograd.grad(f(*x), x)
    want = ref.attention(*(t.detach() for t in x), do, softcap=5.0, slopes=how["slopes"],
                         docs=how["document_ids"], prefix=how["prefix_lens"])
    noise = float((want["o"][1] * do.abs().double()).sum())
    h, g = 2.0 ** -5, torch.Generator().manual_seed(2)
    for i in range(3):
        u = torch.randn(x[i].shape, generator=g).to(gpu)
        u = u / u.norm()
        with torch.no_grad():
            a, b = (f(*(t + s * h * u if j == i else t for j, t in enumerate(x))) for s in (1, -1))
        diff, dot = float((a - b) / (2 * h)), float((grads[i].double() * u.double()).sum())
        assert abs(diff - dot) <= noise / h + h * h * 10


def test_streams_and_graph(gpu):
    from gpt_from_scratch_amd import decode_attn, scored_attn
    B, H, Hk, S, D = 2, 4, 2, 300, 64
    x = [randn((B, n, S, D), i, torch.bfloat16, gpu).requires_grad_()
         for i, n in enumerate((H, Hk, Hk))]
    do = randn((B, H, S, D), 4, torch.bfloat16, gpu)
    ids = documents(B, S, "packed", 6, gpu)
    lens = torch.tensor([300, 77], dtype=torch.int32, device=gpu)

    def call():
        o = scored_attn(*x, document_ids=ids, softcap=20.0)
        with torch.no_grad():
            d = decode_attn(x[0][:, :, -1], x[1], x[2], lens)
        return (o.detach(), d, *torch.autograd.grad(o, x, do))

    want = call()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = call()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):  # two graphs, each with its own workspaces
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    for seed in range(3):
        with torch.no_grad():
            x[0].copy_(randn(x[0].shape, 50 + seed, torch.bfloat16, gpu))
            ids.copy_(documents(B, S, "mixed", 60 + seed, gpu))
            lens.copy_(torch.tensor([17 * seed, 300 - seed], dtype=torch.int32))
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        want = call()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_chain(gpu):
    """The operators as a layer uses them: the fused projection, norms and rotation
    at positions that start over in each document, attention within documents; and
    the last token of each sequence alone gives the same row."""
    from gpt_from_scratch_amd import decode_attn, qk_norm_rotary, scored_attn
    S, B, H, Hk, D = 200, 2, 6, 2, 64
    n = (H + 2 * Hk) * D
    qkv = randn((S, B, n), 1, torch.float32, gpu).requires_grad_()
    w = [(1 + 0.1 * randn((D,), 2 + i, torch.float32, gpu)).requires_grad_() for i in range(2)]
    ids = torch.zeros(B, S, dtype=torch.int32, device=gpu)
    ids[0, 80:] = 1
    ids[1, 130:] = 5
    pos = torch.arange(S, device=gpu)[:, None].repeat(1, B)
    pos[80:, 0] -= 80
    pos[130:, 1] -= 130
    a = torch.outer(torch.arange(S, dtype=torch.float64),
                    10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    cos, sin = (t.float().to(gpu) for t in (a.cos(), a.sin()))
    do = randn((B, H, S, D), 5, torch.float32, gpu)

    def parts(x):
        x = x.view(S, B, H + 2 * Hk, D)
        return x[:, :, :H], x[:, :, H:H + Hk], x[:, :, H + Hk:]

    q, k, v = parts(qkv)
    q, k = qk_norm_rotary(q, k, *w, cos, sin, 1e-6, pos, interleaved=False)
    bhsd = [t.permute(1, 2, 0, 3) for t in (q, k, v)]
    o = scored_attn(*bhsd, document_ids=ids, softcap=30.0)
    got = torch.autograd.grad(o, (qkv, *w), do)
    # the same in float64, gradients by autograd
    x64, w64 = qkv.detach().double().requires_grad_(), [t.detach().double().requires_grad_() for t in w]
    q6, k6, v6 = parts(x64)
    q6, k6 = (ref.turn(t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * u, cos, sin, pos,
                       False) for t, u in ((q6, w64[0]), (k6, w64[1])))
    q6, k6, v6 = (t.permute(1, 2, 0, 3) for t in (q6, k6, v6))
    z = (q6 @ k6.repeat_interleave(3, 1).transpose(-1, -2)) / 8
    z = 30 * torch.tanh(z / 30)
    z = z.masked_fill(~ref.visible(B, S, S, True, ids, None, gpu)[:, None], -torch.inf)
    o6 = torch.softmax(z, -1) @ v6.repeat_interleave(3, 1)
    want = torch.autograd.grad(o6, (x64, *w64), do.double())
    # fp32 throughout: the norm of the difference against that of the value, a chain
    # of products over 64, 200 and 64 terms whose roundings add up as sqrt(n), with a
    # condition of a few; 200 * F32 = 1.2e-5
    for a, b in zip((o, *got), (o6, *want)):
        assert float((a.double() - b).norm() / b.norm()) < 200 * ref.F32
    with torch.no_grad():
        # sequence 0's second document as a cache, its last token alone
        d = decode_attn(bhsd[0][:1, :, -1], bhsd[1][:1, :, 80:], bhsd[2][:1, :, 80:], softcap=30.0)
    assert float((d - o[:1, :, -1]).norm() / d.norm()) < 200 * ref.F32


DECODE = {
    "s1": dict(size=(2, 4, 2, 1, 64)),
    "s31": dict(size=(1, 3, 3, 31, 8)),
    "s33": dict(size=(3, 8, 1, 33, 128)),
    "s128": dict(size=(1, 6, 2, 128, 96), layout="dense"),
    "s129": dict(size=(2, 4, 4, 129, 64), layout="odd"),
    "s1000": dict(size=(2, 8, 2, 1000, 128), bias=1.0),
    "group_40": dict(size=(2, 80, 2, 300, 64)),  # more heads to a key head than one operand's columns
    "group_33": dict(size=(1, 33, 1, 700, 128), cap=20.0),
    "s5000": dict(size=(1, 4, 1, 5000, 128), cap=30.0),
    "many": dict(size=(9, 16, 4, 900, 64), cap=10.0, bias=1.0, layout="strided"),
    "s20000": dict(size=(1, 2, 1, 20000, 40)),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", list(DECODE))
def test_decode(gpu, name, dtype):
    from gpt_from_scratch_amd import decode_attn
    c = DECODE[name]
    B, H, Hk, S, D = c["size"]
    lay = c.get("layout", "model")
    q = heads(B, H, 1, D, 1, dtype, gpu, lay, 1.5)[:, :, 0]
    k, v = (heads(B, Hk, S, D, 1 + i, dtype, gpu, lay, s) for i, s in ((1, 1.5), (2, 1.0)))
    slopes = (2.0 ** -torch.arange(1, H + 1, dtype=torch.float32)).to(gpu) if c.get("bias") else None
    g = torch.Generator().manual_seed(S)
    some = torch.randint(0, S + 1, (B,), generator=g, dtype=torch.int32)
    some[0] = 0 if B > 1 else S
    for lengths in (None, some, torch.full((B,), S + 5, dtype=torch.int32) - 6 * (torch.arange(B) % 2).int()):
        kk, vv = k, v
        if lengths is not None:
            lengths = lengths.to(gpu)
            # behind the last key: anything
            past = torch.arange(S, device=gpu)[None, None, :, None] >= lengths[:, None, None, None]
            kk, vv = (t.masked_fill(past, float("nan")) for t in (k, v))
        o = decode_attn(q, kk, vv, lengths, c.get("cap"), slopes)
        assert o.shape == (B, H, D) and o.dtype == dtype
        for b in range(B):
            n = S if lengths is None else min(max(int(lengths[b]), 0), S)
            if n == 0:
                assert not o[b].any()
                continue
            want = ref.attention(q[b:b + 1, :, None], k[b:b + 1, :, :n], v[b:b + 1, :, :n],
                                 softcap=c.get("cap"), slopes=slopes)["o"]
            ref.within(f"o[{b}]", o[b:b + 1, :, None], want)


def test_offsets_past_32_bits(gpu):
    """A cache of 2.2e9 elements: the last sequence's keys lie past any 32-bit offset."""
    from gpt_from_scratch_amd import decode_attn, scored_attn_forward
    B, Hk, S, D = 9, 2, 1 << 20, 120
    k = torch.empty(B, Hk, S, D, dtype=torch.bfloat16, device=gpu)
    assert k.numel() > 2 ** 31
    v = torch.empty_like(k)
    n = 500
    k[-1, :, S - n:] = randn((Hk, n, D), 1, torch.bfloat16, gpu)
    v[-1, :, S - n:] = randn((Hk, n, D), 2, torch.bfloat16, gpu)
    q = randn((1, 4, D), 3, torch.bfloat16, gpu)
    # the last keys of the last sequence alone, and all of it with zero keys before
    kk, vv = k[-1:, :, S - n:], v[-1:, :, S - n:]
    want = ref.attention(q[:, :, None], kk, vv)["o"]
    ref.within("decode", decode_attn(q, kk, vv)[:, :, None], want)
    ref.within("forward", scored_attn_forward(q[:, :, None], kk, vv)[0], want)
    k[-1, :, :S - n].zero_()
    v[-1, :, :S - n].zero_()
    k[-1, ..., 0] = 0.0
    k[-1, :, :S - n, 0] = -1e4
    q[..., 0] = 1.0
    want = ref.attention(q[:, :, None], k[-1:, :, S - n:], v[-1:, :, S - n:])["o"]
    ref.within("whole", decode_attn(q, k[-1:], v[-1:])[:, :, None], want)
