"""What rotary embedding, attention with modified scores and decoding refuse before
any launch (no GPU needed): through the Python functions, and through the C ABI."""
import ctypes

import pytest
import torch

from gpt_from_scratch_amd import (_lib, apply_rotary_qk, decode_attn, qk_norm_rotary, scored_attn,
                                  scored_attn_forward)


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


# ---- Python ---------------------------------------------------------------------

def _rotary(**kw):
    a = dict(q=_t(8, 2, 4, 64), k=_t(8, 2, 2, 64), cos=_t(8, 32), sin=_t(8, 32), positions=None)
    a.update(kw)
    return a


ROTARY = [
    (dict(q=_t(8, 2, 64)), ValueError, "must be"),
    (dict(k=_t(9, 2, 2, 64)), ValueError, "must be"),
    (dict(k=_t(8, 1, 2, 64)), ValueError, "must be"),
    (dict(k=_t(8, 2, 2, 32)), ValueError, "must be"),
    (dict(k=_t(8, 2, 0, 64)), ValueError, "empty"),
    (dict(k=_t(8, 2, 2, 64, dtype=torch.float16)), TypeError, "share a dtype"),
    (dict(q=_t(8, 2, 4, 64, dtype=torch.float64), k=_t(8, 2, 2, 64, dtype=torch.float64)),
     TypeError, "dtype"),
    (dict(cos=_t(8)), ValueError, "cos and sin"),
    (dict(cos=_t(8, 16)), ValueError, "cos and sin"),
    (dict(cos=_t(8, 32, dtype=torch.float32)), ValueError, "cos and sin"),
    (dict(cos=_t(8, 33), sin=_t(8, 33)), ValueError, "angles"),
    (dict(cos=_t(8, 0), sin=_t(8, 0)), ValueError, "angles"),
    (dict(cos=_t(7, 32), sin=_t(7, 32)), ValueError, "rows for 8 positions"),
    (dict(positions=torch.arange(8.)), TypeError, "int32 or int64"),
    (dict(positions=torch.arange(8, dtype=torch.int16)), TypeError, "int32 or int64"),
    (dict(positions=torch.arange(7)), ValueError, "positions must be"),
    (dict(positions=torch.zeros(2, 8, dtype=torch.int64)), ValueError, "positions must be"),
    (dict(cos=_t(0, 32), sin=_t(0, 32), positions=torch.arange(8)), ValueError, "without rows"),
    ({}, RuntimeError, "GPU|device"),
]


@pytest.mark.parametrize("kw,error,text", ROTARY)
def test_rotary_refuses(kw, error, text):
    a = _rotary(**kw)
    with pytest.raises(error, match=text):
        apply_rotary_qk(**a)
    w = _t(a["q"].shape[-1], dtype=torch.float32)
    with pytest.raises(error, match=text):
        qk_norm_rotary(q_weight=w, k_weight=w, **a)


@pytest.mark.parametrize("kw,error,text", [
    (dict(q_weight=_t(32)), ValueError, "q_weight"),
    (dict(k_weight=_t(1, 64)), ValueError, "k_weight"),
    (dict(k_weight=_t(64, dtype=torch.float32)), TypeError, "share a dtype"),
    (dict(q_weight=torch.zeros(64, dtype=torch.int32)), TypeError, "dtype"),
])
def test_norm_refuses(kw, error, text):
    a = dict(_rotary(), q_weight=_t(64), k_weight=_t(64))
    a.update(kw)
    with pytest.raises(error, match=text):
        qk_norm_rotary(**a)


def test_norm_refuses_long_heads():
    with pytest.raises(ValueError, match="at most 512"):
        qk_norm_rotary(_t(1, 1, 1, 520), _t(1, 1, 1, 520), _t(520), _t(520), _t(1, 4), _t(1, 4))


def _attn(**kw):
    a = dict(q=_t(2, 4, 16, 64), k=_t(2, 2, 32, 64), v=_t(2, 2, 32, 64))
    a.update(kw)
    return a


ATTN = [
    (dict(q=_t(4, 16, 64)), ValueError, "must be"),
    (dict(v=_t(2, 2, 32, 32)), ValueError, "must be"),
    (dict(q=_t(1, 4, 16, 64)), ValueError, "multiple of Hk"),
    (dict(q=_t(2, 3, 16, 64)), ValueError, "multiple of Hk"),
    (dict(q=_t(2, 4, 0, 64)), ValueError, "no size 0"),
    (dict(q=_t(2, 4, 33, 64)), ValueError, "more queries"),
    (dict(v=_t(2, 2, 32, 64, dtype=torch.float16)), TypeError, "share a dtype"),
    (dict(q=_t(2, 4, 16, 60), k=_t(2, 2, 32, 60), v=_t(2, 2, 32, 60)), ValueError, "head dim"),
    (dict(q=_t(2, 4, 16, 136), k=_t(2, 2, 32, 136), v=_t(2, 2, 32, 136)), ValueError, "head dim"),
    (dict(softcap=0.0), ValueError, "softcap"),
    (dict(softcap=-1.0), ValueError, "softcap"),
    (dict(softcap=float("inf")), ValueError, "softcap"),
    (dict(softcap=1e-60), ValueError, "softcap"),       # 0 in fp32: would mean none
    (dict(softcap=2e4), ValueError, "softcap"),
    (dict(softmax_scale=0.0), ValueError, "softmax_scale"),
    (dict(softmax_scale=float("nan")), ValueError, "softmax_scale"),
    (dict(slopes=torch.zeros(2)), ValueError, "slopes"),
    (dict(slopes=torch.zeros(4, dtype=torch.bfloat16)), ValueError, "slopes"),
]
SLOPES_GRAD = (dict(slopes=torch.zeros(4, requires_grad=True)), ValueError, "slopes take no grad")
MASKS = [
    (dict(document_ids=torch.zeros(2, 32)), ValueError, "document_ids"),
    (dict(document_ids=torch.zeros(2, 32, dtype=torch.int64)), ValueError, "document_ids"),
    (dict(document_ids=torch.zeros(2, 16, dtype=torch.int32)), ValueError, "document_ids"),
    (dict(prefix_lens=torch.zeros(1, dtype=torch.int32)), ValueError, "prefix_lens"),
    (dict(prefix_lens=torch.zeros(2, dtype=torch.int64)), ValueError, "prefix_lens"),
    (dict(prefix_lens=torch.zeros(2, dtype=torch.int32), causal=False), ValueError, "causal"),
    ({}, RuntimeError, "GPU|device"),
]


@pytest.mark.parametrize("call", [scored_attn, scored_attn_forward])
@pytest.mark.parametrize("kw,error,text", ATTN + MASKS)
def test_scored_attn_refuses(call, kw, error, text):
    with pytest.raises(error, match=text):
        call(**_attn(**kw))


def test_scored_attn_refuses_slopes_with_gradients():
    kw, error, text = SLOPES_GRAD
    with pytest.raises(error, match=text):
        scored_attn(**_attn(**kw))


@pytest.mark.parametrize("kw,error,text", [c for c in ATTN if "q" not in c[0] or c[2] == "head dim"] + [
    SLOPES_GRAD,
    (dict(lengths=torch.zeros(2)), ValueError, "lengths"),
    (dict(lengths=torch.zeros(2, 1, dtype=torch.int32)), ValueError, "lengths"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError, "lengths"),
    (dict(k=_t(2, 2, 0, 64), v=_t(2, 2, 0, 64)), ValueError, "no size 0"),
    (dict(q=_t(4, 16, 64)), ValueError, "multiple of Hk"),
    (dict(q=_t(2, 3, 1, 64)), ValueError, "multiple of Hk"),
    (dict(q=_t(2, 4)), ValueError, "must be"),
    (dict(k=_t(2, 2, 32, 64).requires_grad_()), RuntimeError, "no backward"),
    ({}, RuntimeError, "GPU|device"),
])
def test_decode_refuses(kw, error, text):
    a = _attn(**kw)
    if a["q"].dim() == 4:
        a["q"] = a["q"].sum(2)
    with pytest.raises(error, match=text):
        decode_attn(**a)


# ---- C ABI: addresses that are never read, since the checks come first -----------

P = ctypes.c_void_p(1 << 20)
BAD, UNSUPPORTED = 1, 2


def _s(*v):
    return (ctypes.c_int64 * len(v))(*v)


ROW = _s(512, 256, 64, 1)


def _how(**kw):
    h = _lib.Rotary(2, 8, 2, 4, 2, 64, 64, 1, 1 << 20, 1 << 20, (32, 1), (32, 1), 8)
    for k, v in kw.items():
        setattr(h, k, v)
    return h


@pytest.mark.parametrize("kw,code", [
    (dict(tab_dtype=5), BAD), (dict(S=0), BAD), (dict(B=-1), BAD), (dict(Hk=0), BAD),
    (dict(R=0), BAD), (dict(R=63), BAD), (dict(R=66), BAD), (dict(cos_tab=None), BAD),
    (dict(sin_tab=None), BAD), (dict(table_rows=7), BAD), (dict(table_rows=0), BAD),
    (dict(positions=1 << 20, pos_bytes=2), BAD), (dict(positions=1 << 20, table_rows=0), BAD),
    (dict(S=1 << 28, B=16, table_rows=1 << 28), UNSUPPORTED),
])
def test_rotary_c_refuses(kw, code):
    lib, h = _lib.lib(), _how(**kw)
    assert lib.mi_rotary_qk(2, h, 0, P, ROW, P, ROW, P, ROW, P, ROW, None) == code
    assert lib.mi_qk_norm_rotary(2, 0, h, 1e-6, P, ROW, P, ROW, P, P, P, ROW, P, ROW, None) == code
    assert lib.mi_qk_norm_rotary_bwd(2, 0, h, 1e-6, P, ROW, P, ROW, P, P, P, ROW, P, ROW, P, ROW, P,
                                     ROW, P, P, P, 1 << 40, None) == code


def test_rotary_c_refuses_pointers_and_workspaces():
    lib, h = _lib.lib(), _how()
    assert lib.mi_rotary_qk(9, h, 0, P, ROW, P, ROW, P, ROW, P, ROW, None) == BAD
    assert lib.mi_rotary_qk(2, None, 0, P, ROW, P, ROW, P, ROW, P, ROW, None) == BAD
    assert lib.mi_rotary_qk(2, h, 0, None, ROW, P, ROW, P, ROW, P, ROW, None) == BAD
    assert lib.mi_rotary_qk(2, h, 0, P, ROW, P, ROW, P, ROW, P, None, None) == BAD
    norm = [P, ROW, P, ROW, P, P, P, ROW, P, ROW]
    assert lib.mi_qk_norm_rotary(2, 7, h, 1e-6, *norm, None) == BAD
    assert lib.mi_qk_norm_rotary(2, 0, h, -1.0, *norm, None) == BAD
    assert lib.mi_qk_norm_rotary(2, 0, h, float("nan"), *norm, None) == BAD
    assert lib.mi_qk_norm_rotary(2, 0, _how(D=520), 1e-6, *norm, None) == UNSUPPORTED
    n = lib.mi_qk_norm_rotary_workspace(h)
    assert n > 0 and lib.mi_qk_norm_rotary_workspace(None) == 0
    bwd = norm + [P, ROW, P, ROW, P, P]
    assert lib.mi_qk_norm_rotary_bwd(2, 0, h, 1e-6, *bwd, P, n - 1, None) == BAD
    assert lib.mi_qk_norm_rotary_bwd(2, 0, h, 1e-6, *bwd, None, n, None) == BAD


def _fwd(lib, dtype=2, sizes=(1, 2, 2, 64, 64, 64), scale=0.1, mods=None, q=P, st=ROW, o_lo=None,
         lse=P, tiles=P, ws=P, n=1 << 40):
    mods = mods or _lib.ScoreMods(1, 0.0)
    return lib.mi_sattn_fwd(dtype, *sizes, scale, mods, q, st, P, ROW, P, ROW, P, ROW, o_lo, lse,
                            tiles, ws, n, None)


def _bwd(lib, dtype=2, sizes=(1, 2, 2, 64, 64, 64), scale=0.1, mods=None, q=P, st=ROW, o_lo=None,
         lse=P, tiles=P, ws=P, n=1 << 40):
    mods = mods or _lib.ScoreMods(1, 0.0)
    return lib.mi_sattn_bwd(dtype, *sizes, scale, mods, q, st, P, ROW, P, ROW, P, ROW, o_lo, P, ROW,
                            lse, tiles, ws, n, P, ROW, P, ROW, P, ROW, None)


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("call", [_fwd, _bwd])
@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), BAD), (dict(sizes=(0, 2, 2, 64, 64, 64)), BAD),
    (dict(sizes=(1, 2, 2, 0, 64, 64)), BAD), (dict(sizes=(1, 3, 2, 64, 64, 64)), BAD),
    (dict(sizes=(1, 2, 2, 65, 64, 64)), BAD), (dict(sizes=(1, 2, 2, 64, 64, 60)), UNSUPPORTED),
    (dict(sizes=(1, 2, 2, 64, 64, 136)), UNSUPPORTED),
    (dict(sizes=(1, 1, 1, 1, (1 << 24) + 1, 64)), UNSUPPORTED),
    (dict(sizes=(1 << 16, 1 << 15, 1, 1, 1, 64)), UNSUPPORTED),
    (dict(sizes=(1 << 12, 1 << 12, 1, 1, 1, 64)), UNSUPPORTED),  # 2^32 threads
    (dict(sizes=(1 << 10, 1 << 10, 1 << 10, 1, 1 << 10, 8)), UNSUPPORTED),
    (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD), (dict(scale=NAN), BAD), (dict(scale=INF), BAD),
    (dict(mods=_lib.ScoreMods(1, -1.0)), BAD), (dict(mods=_lib.ScoreMods(1, NAN)), BAD),
    (dict(mods=_lib.ScoreMods(1, INF)), BAD), (dict(mods=_lib.ScoreMods(1, 2e4)), BAD),
    (dict(mods=_lib.ScoreMods(1, 1e-8)), BAD),
    (dict(mods=_lib.ScoreMods(0, 0.0, None, None, 1 << 20)), BAD),
    (dict(mods=_lib.ScoreMods(1, 0.0, None, 1 << 20), tiles=None), BAD),
    (dict(mods=_lib.ScoreMods(1, 0.0, None, 1 << 20), tiles=ctypes.c_void_p((1 << 20) + 4)), BAD),
    (dict(q=None), BAD), (dict(q=ctypes.c_void_p((1 << 20) + 2)), UNSUPPORTED),
    (dict(st=_s(512, 256, 64, 2)), BAD), (dict(st=_s(512, 256, 68, 1)), UNSUPPORTED),
    (dict(st=_s(512, 256, 1 << 22, 1)), UNSUPPORTED), (dict(lse=None), BAD),
    (dict(dtype=0, o_lo=P), UNSUPPORTED), (dict(o_lo=ctypes.c_void_p((1 << 20) + 2)), UNSUPPORTED),
])
def test_sattn_c_refuses(call, kw, code):
    assert call(_lib.lib(), **kw) == code


def test_sattn_c_workspaces():
    lib = _lib.lib()
    size = (2, 1, 2, 2, 4096, 4096, 64)  # long rows and few heads: split, partial sums
    assert lib.mi_sattn_bwd_workspace(*size) > 0
    for call, want in ((_fwd, lib.mi_sattn_fwd_workspace), (_bwd, lib.mi_sattn_bwd_workspace)):
        n = want(*size)
        assert n >= 0
        if n:
            assert call(lib, sizes=size[1:], n=0) == BAD
            assert call(lib, sizes=size[1:], ws=None) == BAD
            assert call(lib, sizes=size[1:], ws=ctypes.c_void_p((1 << 20) + 4)) == BAD
        assert want(2, 1, 3, 2, 64, 64, 64) == 0  # what the call would refuse
    assert _bwd(lib, sizes=size[1:], n=lib.mi_sattn_bwd_workspace(*size) - 1) == BAD
    assert lib.mi_sattn_tiles(2, 65, 129) == 4 * 2 * (2 + 3)
    assert lib.mi_sattn_tiles(0, 64, 64) == 0


def test_decode_c_refuses():
    lib = _lib.lib()

    def call(dtype=2, sizes=(1, 2, 2, 64, 64), scale=0.1, cap=0.0, q=P, qs=_s(128, 64, 1), kst=ROW,
             ws=P, n=1 << 40):
        return lib.mi_decode_attn(dtype, *sizes, scale, cap, None, None, q, qs, P, kst, P, ROW, P,
                                  _s(128, 64, 1), ws, n, None)
    assert call(dtype=-1) == BAD
    assert call(sizes=(1, 3, 2, 64, 64)) == BAD
    assert call(sizes=(1, 2, 2, 0, 64)) == BAD
    assert call(sizes=(1, 2, 2, 64, 12)) == UNSUPPORTED
    assert call(scale=NAN) == BAD and call(cap=-2.0) == BAD and call(cap=INF) == BAD
    assert call(q=None) == BAD
    assert call(q=ctypes.c_void_p((1 << 20) + 8)) == UNSUPPORTED
    assert call(qs=_s(128, 64, 2)) == BAD and call(qs=_s(128, 60, 1)) == UNSUPPORTED
    assert call(kst=_s(512, 256, 60, 1)) == UNSUPPORTED
    big = (1, 8, 8, 65536, 128)
    n = lib.mi_decode_workspace(2, *big)
    assert n > 0
    assert call(sizes=big, n=n - 1) == BAD and call(sizes=big, ws=None) == BAD
