"""Tables for long contexts (no GPU needed), against the formulas in Python floats."""
import math

import pytest
import torch

from gpt_from_scratch_amd import RotaryEmbedding, RotaryScaling

EPS = torch.finfo(torch.float32).eps / 2


def _freq(i, dim, base, s):
    f = base ** (-2 * i / dim)
    if s.trained_positions is None:
        return f / s.factor
    keep = (s.trained_positions * f / (2 * math.pi) - s.slow) / (s.fast - s.slow)
    keep = min(max(keep, 0.0), 1.0)
    return f * keep + f / s.factor * (1 - keep)


@pytest.mark.parametrize("scaling", [
    RotaryScaling(4.0), RotaryScaling(1.0), RotaryScaling(8.0, 2048),
    RotaryScaling(32.0, 4096, 16.0, 2.0), RotaryScaling(2.5, 1)])
@pytest.mark.parametrize("dim,base", [(64, 10000.0), (128, 500000.0), (2, 10000.0)])
def test_scaled_tables(scaling, dim, base):
    e = RotaryEmbedding(dim, 8, base, device="cpu", scaling=scaling)
    x = torch.empty(1)
    n = 70001
    cos, sin = e(x, n)
    size = 1.0 if scaling.trained_positions is None else 0.1 * math.log(scaling.factor) + 1
    assert cos.shape == sin.shape == (n, dim // 2) and cos.dtype == torch.float32
    for i in {0, 1 % (dim // 2), dim // 4, dim // 2 - 1}:
        f = _freq(i, dim, base, scaling)
        assert abs(e.freqs[i].item() - f) <= 1.01 * EPS * f
        for s in (0, 1, 17, 2047, 65535, n - 1):
            # float64 angles: off by a few 2^-53 of up to 7e4 radians, then one rounding
            tol = size * (EPS + 1e-9)
            assert abs(cos[s, i].item() - size * math.cos(s * f)) <= tol
            assert abs(sin[s, i].item() - size * math.sin(s * f)) <= tol


def test_unscaled_tables_keep_their_values():
    a = RotaryEmbedding(64, 128, device="cpu")
    t = torch.outer(torch.arange(128, dtype=torch.float32),
                    1.0 / (10000.0 ** (torch.arange(0, 64, 2, dtype=torch.float32) / 64)))
    assert torch.equal(a.cos_cached, t.cos()) and torch.equal(a.sin_cached, t.sin())
    assert set(a.state_dict()) == {"freqs"}


def test_a_factor_of_one_changes_only_roundings():
    a = RotaryEmbedding(64, 128, device="cpu")
    b = RotaryEmbedding(64, 128, device="cpu", scaling=RotaryScaling(1.0, 128))
    # fp32 angles: a frequency off by 2^-23 (power and quotient), a product by 2^-24
    torch.testing.assert_close(a.cos_cached, b.cos_cached, rtol=0, atol=128 * 4 * EPS)


@pytest.mark.parametrize("bad", [
    RotaryScaling(0.5), RotaryScaling(float("inf")), RotaryScaling(float("nan")),
    RotaryScaling(2.0, 0), RotaryScaling(2.0, 128, 1.0, 1.0), RotaryScaling(2.0, 128, 4.0, 0.0)])
def test_refusals(bad):
    with pytest.raises(ValueError, match="scaling"):
        RotaryEmbedding(64, 128, device="cpu", scaling=bad)
