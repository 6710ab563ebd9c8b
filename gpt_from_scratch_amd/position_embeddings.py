"""Rotary tables: the counterpart of core/position_embeddings.py.

``RotaryEmbedding(head_dim, max_position_embeddings=2048, base=10000.0,
device=None)`` builds, in fp32,

    freqs[i]  = 1 / base ** (2i / head_dim)                 (:19)
    cos[s, i] = cos(s * freqs[i]),  sin[s, i] = sin(s * freqs[i])   (:34-40)

and ``forward(x, seq_len)`` returns the first ``seq_len`` rows cast to
``x.dtype`` (:45-51).  Unlike the reference, a ``seq_len`` beyond the cached
length regrows the cache (the reference's regrow call passes three arguments to
a one-argument method, :48 vs :29, and raises ``TypeError``).

``scaling=RotaryScaling(factor)`` gives the tables of a context ``factor`` times
the trained one, with all positions divided by ``factor``; with
``trained_positions`` = L, pair i keeps its speed where it makes at least ``fast``
turns within L positions, is slowed by ``factor`` where it makes at most ``slow``,
and by a mean of both in between (Peng et al. 2023, "YaRN", eqs. 17-20):

    t_i = L freqs[i] / 2 pi,   g_i = clamp((t_i - slow) / (fast - slow), 0, 1)
    freqs'[i] = freqs[i] (g_i + (1 - g_i) / factor)

and cos and sin are multiplied by ``0.1 ln(factor) + 1`` (eq. 22: q . k by its
square).  Scaled tables are computed in float64: a position of 10^5 in fp32 puts
the angle off by up to 0.004.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
import torch.nn as nn


class RotaryScaling(NamedTuple):
    factor: float
    trained_positions: Optional[int] = None
    fast: float = 32.0
    slow: float = 1.0


class RotaryEmbedding(nn.Module):
    def __init__(self, head_dim, max_position_embeddings=2048, base=10000.0, device=None,
                 scaling: Optional[RotaryScaling] = None):
        super().__init__()
        if scaling is not None:
            scaling = RotaryScaling(*scaling)
            if not 1.0 <= scaling.factor < math.inf:
                raise ValueError(f"the scaling factor must be 1 or more; got {scaling.factor}")
            if scaling.trained_positions is not None and (
                    scaling.trained_positions < 1 or not 0 < scaling.slow < scaling.fast):
                raise ValueError(f"scaling needs trained_positions of 1 or more and "
                                 f"0 < slow < fast; got {scaling}")
        self.scaling = scaling
        self.head_dim = head_dim
        self.max_position_embeddings = max_position_embeddings
        self.base = base
        if device is None:
            device = torch.cuda.current_device() if torch.cuda.is_available() else "cpu"
        freqs = 1.0 / (self.base ** (torch.arange(0, self.head_dim, 2, device=device,
                                                  dtype=torch.float32) / self.head_dim))
        if scaling is not None:
            freqs = self._scaled_freqs(device)
        self.register_buffer("freqs", freqs.to(torch.float32))
        self.max_seq_len_cached = 0
        self._set_cos_sin_cache(self.max_position_embeddings)

    def _scaled_freqs(self, device):
        factor, trained, fast, slow = self.scaling
        freqs = float(self.base) ** (-torch.arange(0, self.head_dim, 2, device=device,
                                                   dtype=torch.float64) / self.head_dim)
        if trained is None:
            return freqs / factor
        keep = ((trained * freqs / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        return freqs * (keep + (1 - keep) / factor)

    def _set_cos_sin_cache(self, seq_len):
        self.max_seq_len_cached = seq_len
        if self.scaling is not None:
            t = torch.arange(seq_len, dtype=torch.float64, device=self.freqs.device)
            thetas = torch.outer(t, self._scaled_freqs(self.freqs.device))
            size = 1.0
            if self.scaling.trained_positions is not None:
                size = 0.1 * math.log(self.scaling.factor) + 1.0
            self.register_buffer("cos_cached", (size * thetas.cos()).float(), persistent=False)
            self.register_buffer("sin_cached", (size * thetas.sin()).float(), persistent=False)
            return
        t = torch.arange(seq_len, dtype=torch.float32, device=self.freqs.device)
        thetas = torch.outer(t, self.freqs)
        self.register_buffer("cos_cached", thetas.cos().to(torch.float32), persistent=False)
        self.register_buffer("sin_cached", thetas.sin().to(torch.float32), persistent=False)

    def forward(self, x, seq_len=None):
        if seq_len is None:
            seq_len = x.shape[0]
        if seq_len > self.max_seq_len_cached:
            self._set_cos_sin_cache(seq_len)
        return (self.cos_cached[:seq_len, :].to(x.dtype),
                self.sin_cached[:seq_len, :].to(x.dtype))
