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
        if not bool(torch.isfinite(table).all()) or not math.isfinite(self.gain):
            raise ValueError("frequencies and attention_factor must be finite")
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


def _side(what: str, x: Optional[torch.Tensor], like: torch.Tensor):
    """x [*lead, H, D] as [T, H, D] (a view where its strides allow)."""
    if x is None:
        return None
    if x.dim() < 2 or x.shape[:-2] != like.shape[:-2] or x.shape[-1] != like.shape[-1] or x.dtype != like.dtype:
        raise ValueError(f"apply_norm_rotary: {what} {tuple(x.shape)} {x.dtype} does not match queries "
                         f"{tuple(like.shape)} {like.dtype} in tokens, head_dim or dtype")
    flat = x.reshape(math.prod(x.shape[:-2]), *x.shape[-2:])
    return flat if flat.stride(-1) == 1 or flat.shape[-1] == 1 else flat.contiguous()


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
    dev = _native.require_gpu(q, k, positions, rotary.freqs, q_weight, k_weight)
    _native.require_plain("apply_norm_rotary", q, k, q_weight, k_weight)
    if q.dim() < 2:
        raise ValueError(f"apply_norm_rotary: queries must be [*lead, heads, head_dim], got {tuple(q.shape)}")
    if tuple(positions.shape) != tuple(q.shape[:-2]) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"apply_norm_rotary: positions must be int32 or int64 {tuple(q.shape[:-2])}, got "
                         f"{tuple(positions.shape)} {positions.dtype}")
    D = q.shape[-1]
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if tuple(w.shape) != (D,) or w.dtype != weights[0].dtype:
            raise ValueError(f"apply_norm_rotary: weights must be [{D}] and of one dtype, got {tuple(w.shape)} {w.dtype}")
    if not (eps >= 0.0 and math.isfinite(eps) and math.isfinite(weight_offset)):
        raise ValueError("apply_norm_rotary: eps must be a finite number of 0 or more, weight_offset finite")
    code = _native.dtype_code(q.dtype)
    qf, kf, pos = _side("queries", q, q), _side("keys", k, q), positions.reshape(-1).contiguous()
    qw, kw = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
    q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    k_out = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=dev)
    p = _native.RotaryParams()
    p.dtype, p.n_q_heads, p.head_dim, p.tokens = code, qf.shape[1], D, qf.shape[0]
    p.q, p.q_stride_t, p.q_stride_h, p.q_out = qf.data_ptr(), qf.stride(0), qf.stride(1), q_out.data_ptr()
    if kf is not None:
        p.n_k_heads, p.k, p.k_out = kf.shape[1], kf.data_ptr(), k_out.data_ptr()
        p.k_stride_t, p.k_stride_h = kf.stride(0), kf.stride(1)
    p.rotary_dim, p.interleaved, p.gain = rotary.rotary_dim, int(rotary.interleaved), rotary.gain
    p.freqs, p.positions, p.position_bytes = rotary.freqs.data_ptr(), pos.data_ptr(), pos.element_size()
    p.q_weight, p.k_weight = (None if w is None else w.data_ptr() for w in (qw, kw))
    p.weight_dtype = _native.dtype_code(weights[0].dtype) if weights else _native.F32
    p.eps, p.weight_offset = eps, weight_offset
    _native.launch_on(dev, _native.lib().smaq_norm_rotary, "smaq_norm_rotary", ctypes.byref(p))
    return q_out, k_out
