"""Queries and keys as attention reads them: normed per head and rotated.

The codecs and caches of this package take keys after a model's own norm and
position rotation (``k`` of smaq/score.py and smaq/capture.py are such keys).
``apply_norm_rotary`` makes them from a layer's projection in one pass over
queries and keys, without a cosine table: angles are formed from the positions
in 64 bits, so far positions lose nothing.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from smaq_amd import _native

SCALINGS = ("none", "linear", "ntk", "yarn")


class RotaryPositions:
    """Frequencies of a position rotation, kept on a device.

    Pair i of the first ``rotary_dim`` dims turns by ``position * freqs[i]``,
    ``freqs[i] = base^(-2 i / rotary_dim)``; pairs are (i, rotary_dim / 2 + i),
    or neighbours (2 i, 2 i + 1) when ``interleaved``.  ``scaling`` extends a
    model trained on ``original_length`` positions by ``factor``:

    * ``linear``: every frequency divided by the factor;
    * ``ntk``: the base times factor^(r / (r - 2)), which divides the slowest
      frequency by the factor and leaves the fastest;
    * ``yarn``: pairs that make more than ``beta_fast`` turns over the original
      length keep their frequency, those below ``beta_slow`` turns are divided,
      linearly in between; sines and cosines are multiplied by
      ``0.1 ln(factor) + 1`` (or ``attention_factor``).

    ``freqs`` (a sequence of rotary_dim / 2 numbers) replaces the formula for
    any other schedule.
    """

    def __init__(self, rotary_dim: int, base: float = 10000.0, interleaved: bool = False, scaling: str = "none",
                 factor: float = 1.0, original_length: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 attention_factor: Optional[float] = None, freqs=None, device="cuda"):
        if rotary_dim < 0 or rotary_dim % 2:
            raise ValueError(f"rotary_dim must be an even number of 0 or more, got {rotary_dim}")
        if scaling not in SCALINGS:
            raise ValueError(f"unknown scaling {scaling!r}; expected one of {SCALINGS}")
        if not (base > 1.0 and math.isfinite(base)):
            raise ValueError(f"base must be a number above 1, got {base}")
        if not (factor >= 1.0 and math.isfinite(factor)):
            raise ValueError(f"factor must be a number of 1 or more, got {factor}")
        self.rotary_dim = int(rotary_dim)
        self.interleaved = bool(interleaved)
        self.gain = 1.0
        half = self.rotary_dim // 2
        if freqs is not None:
            if scaling != "none":
                raise ValueError("freqs are final: scaling does not apply to them")
            table = torch.as_tensor(freqs, dtype=torch.float64).reshape(-1).cpu()
            if table.numel() != half:
                raise ValueError(f"freqs has {table.numel()} entries for {half} pairs")
        else:
            table = self._schedule(half, base, scaling, factor, original_length, beta_fast, beta_slow)
            if scaling == "yarn":
                self.gain = 0.1 * math.log(factor) + 1.0
        if attention_factor is not None:
            self.gain = float(attention_factor)
        if not bool(torch.isfinite(table).all()) or not abs(self.gain) < 1e38:
            raise ValueError("frequencies must be finite, attention_factor a number below 1e38")
        self.freqs = table.contiguous().to(device)

    def _schedule(self, half, base, scaling, factor, original_length, beta_fast, beta_slow) -> torch.Tensor:
        r = self.rotary_dim
        if scaling == "ntk" and r > 2:
            base = base * factor ** (r / (r - 2))
        f = torch.tensor([base ** (-2.0 * i / r) for i in range(half)], dtype=torch.float64)
        if scaling == "linear":
            return f / factor
        if scaling != "yarn":
            return f
        if original_length <= 0 or not beta_fast > beta_slow > 0:
            raise ValueError("yarn needs original_length above 0 and beta_fast above beta_slow above 0")

        def pair_of(turns):  # the (fractional) pair that makes so many turns over the original length
            return r * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        low = max(0, math.floor(pair_of(beta_fast)))
        high = min(r - 1, math.ceil(pair_of(beta_slow)))
        share = ((torch.arange(half, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        return f * (1.0 - share) + f / factor * share

    def to(self, device) -> "RotaryPositions":
        """The same rotation with its frequencies on another device."""
        new = object.__new__(RotaryPositions)
        new.__dict__.update(self.__dict__, freqs=self.freqs.to(device))
        return new


def _heads(what: str, x: torch.Tensor, lead, D: int, dtype) -> torch.Tensor:
    """x [*lead, H, D] as [T, H, D] (a view where its strides allow)."""
    shape = x.shape
    if len(shape) < 2 or shape[:-2] != lead or shape[-1] != D or x.dtype != dtype:
        raise ValueError(f"apply_norm_rotary: {what} {tuple(x.shape)} {x.dtype} do not match queries of tokens "
                         f"{tuple(lead)}, head_dim {D} and {dtype}")
    if len(shape) != 3:
        x = x.reshape(math.prod(lead), *shape[-2:])
    return x if x.stride(2) == 1 or D == 1 else x.contiguous()


def apply_norm_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary: RotaryPositions,
                      q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                      eps: float = 1e-6, weight_offset: float = 0.0):
    """RMS norm per head, then rotation, of queries [*lead, Hq, D] and keys
    [*lead, Hk, D] (None: queries alone) at ``positions`` [*lead] (integers).

    ``x * rsqrt(mean(x^2) + eps) * (weight + weight_offset)`` over the head dim
    where a weight [D] is given (queries and keys apart), then the rotation of
    the first ``rotary.rotary_dim`` dims.  fp32 between input and output, one
    rounding.  Views of a packed projection are read in place; the results are
    new contiguous tensors, (q, k), or (q, None).
    """
    freqs = rotary.freqs
    index = _native.require_inputs("apply_norm_rotary", q, k, positions, freqs, q_weight, k_weight)
    if q.dim() < 2:
        raise ValueError(f"apply_norm_rotary: queries must be [*lead, heads, head_dim], got {tuple(q.shape)}")
    shape, dtype = q.shape, q.dtype
    lead, D = shape[:-2], shape[-1]
    wide = positions.dtype == torch.int64
    if positions.shape != lead or not (wide or positions.dtype == torch.int32):
        raise ValueError(f"apply_norm_rotary: positions must be int32 or int64 {tuple(lead)}, got "
                         f"{tuple(positions.shape)} {positions.dtype}")
    weight_dtype = None
    for w in (q_weight, k_weight):
        if w is not None:
            weight_dtype = weight_dtype or w.dtype
            if w.dim() != 1 or w.shape[0] != D or w.dtype != weight_dtype:
                raise ValueError(f"apply_norm_rotary: weights must be [{D}] and of one dtype, got {tuple(w.shape)} "
                                 f"{w.dtype}")
    if not (0.0 <= eps < 1e38 and abs(weight_offset) < 1e38):
        raise ValueError("apply_norm_rotary: eps must be a number from 0 to 1e38, weight_offset one below 1e38")
    code = _native.dtype_code(dtype)
    weight_code = _native.F32 if weight_dtype is None else _native.dtype_code(weight_dtype)
    qf = _heads("queries", q, lead, D, dtype)
    pos = positions.reshape(-1) if len(lead) != 1 else positions
    pos = pos.contiguous()
    qw = q_weight if q_weight is None else q_weight.contiguous()
    kw = k_weight if k_weight is None else k_weight.contiguous()
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = None
    T, Hq, _ = qf.shape
    Hk = kp = ko = kst = ksh = 0
    if k is not None:
        kf = _heads("keys", k, lead, D, dtype)
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        Hk, kp, ko = kf.shape[1], kf.data_ptr(), k_out.data_ptr()
        kst, ksh, _ = kf.stride()
    qst, qsh, _ = qf.stride()
    p = _native.RotaryParams(
        code, Hq, Hk, D, rotary.rotary_dim, rotary.interleaved, T, qf.data_ptr(), qst, qsh, kp, kst, ksh,
        q_out.data_ptr(), ko, pos.data_ptr(), 8 if wide else 4, freqs.data_ptr(), rotary.gain,
        None if qw is None else qw.data_ptr(), None if kw is None else kw.data_ptr(), weight_code, eps, weight_offset)
    _native.launch_on(index, _native.lib().smaq_norm_rotary, "smaq_norm_rotary", ctypes.byref(p))
    return q_out, k_out
