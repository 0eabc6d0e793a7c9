"""Attention over exact keys and values, next to the compressed history's.

``compute_hybrid_attention`` and the paged pools answer a decode step from
compressed tokens.  Around them a serving program attends exact ones: a
prefill over the step's own tokens, several requests back to back, and decode
over an exact paged cache (layers kept exact, contexts too short to compress).
Scores may be capped by a tanh and biased by distance; documents, prefixes and
windows mask them.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from smaq_amd import _native

_INTEGERS = (torch.int32, torch.int64)
_TYPES = {torch.float16: _native.F16, torch.bfloat16: _native.BF16}


def _scores(what: str, head_dim: int, scale: Optional[float], score_cap: float, window: int):
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    if not abs(scale) < 1e38:
        raise ValueError(f"{what}: scale must be a number below 1e38, got {scale}")
    if score_cap != 0.0 and not 1e-30 <= score_cap < 1e30:
        raise ValueError(f"{what}: score_cap must be 0 (none) or a number from 1e-30 to 1e30, got {score_cap}")
    if window < 0 or window > 0x7fffffff:
        raise ValueError(f"{what}: window must be 0 (none) or a number of tokens, got {window}")
    return scale, float(score_cap), int(window)


def _slopes(what: str, alibi_slopes: Optional[torch.Tensor], heads: int):
    if alibi_slopes is None:
        return None
    if alibi_slopes.dim() != 1 or alibi_slopes.shape[0] != heads or not alibi_slopes.dtype.is_floating_point:
        raise ValueError(f"{what}: alibi_slopes must be [{heads}] floating point, got {tuple(alibi_slopes.shape)} "
                         f"{alibi_slopes.dtype}")
    return (alibi_slopes if alibi_slopes.dtype == torch.float32 else alibi_slopes.float()).contiguous()


def _int32(t: torch.Tensor) -> torch.Tensor:
    """int32 or int64 as contiguous int32; numbers beyond it stay beyond any size."""
    if t.dtype != torch.int32:
        t = t.clamp(-(2 ** 31), 2 ** 31 - 1).to(torch.int32)
    return t.contiguous()


def _ints(what: str, name: str, t: torch.Tensor, n: int) -> torch.Tensor:
    """t [n] of integers as contiguous int32."""
    if t.dim() != 1 or t.shape[0] != n or t.dtype not in _INTEGERS:
        raise ValueError(f"{what}: {name} must be int32 or int64 [{n}], got {tuple(t.shape)} {t.dtype}")
    return _int32(t)


def _rows(t: torch.Tensor):
    """(t, its row strides), t copied where its rows are not dense or not on 16 bytes."""
    steps = _native.row_steps(t)
    if steps is None:
        t = t.clone(memory_format=torch.contiguous_format)
        steps = _native.row_steps(t)
    return t, steps


def _heads(what: str, q: torch.Tensor, hkv: int, D: int) -> None:
    if q.dtype not in _TYPES:
        raise ValueError(f"{what}: float16 or bfloat16 queries, keys and values, got {q.dtype}")
    if D % 8 or not 0 < D <= 256:
        raise ValueError(f"{what}: head_dim must be a multiple of 8 up to 256, got {D}")
    if hkv <= 0 or q.shape[1] <= 0 or q.shape[1] % hkv:
        raise ValueError(f"{what}: {q.shape[1]} query heads are not a multiple of {hkv} key-value heads")


def _out(what: str, out: Optional[torch.Tensor], q: torch.Tensor, *others: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous()
            or out.data_ptr() % 16):
        raise ValueError(f"{what}: out must be a contiguous, 16-byte aligned {tuple(q.shape)} {q.dtype} tensor on "
                         f"{q.device}")
    if any(_native.overlap(out, t) for t in (q, *others)):
        raise ValueError(f"{what}: out shares memory with an input")
    return out


def compute_packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, *,
                             scale: Optional[float] = None, causal: bool = True,
                             prefix_lens: Optional[torch.Tensor] = None, window: int = 0, score_cap: float = 0.0,
                             alibi_slopes: Optional[torch.Tensor] = None,
                             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of queries [T, Hq, D] over the same tokens' keys and values
    [T, Hkv, D], documents back to back: document b is tokens ``cu_seqlens[b]``
    to ``cu_seqlens[b + 1] - 1`` (integers, [documents + 1], ascending).

    Within a document, row i sees key j when ``not causal or j <= i`` and
    ``window == 0 or j > i - window``; the document's first ``prefix_lens[b]``
    keys are seen from all its rows.  Scores are ``scale q.k`` (scale None:
    1/sqrt(D)), then ``score_cap tanh(x / score_cap)`` if the cap is not 0, then
    minus ``alibi_slopes[head] |i - j|``.  Whatever stands in unseen places does
    not reach a row, NaN and infinities among it.

    fp16 or bf16, head_dim a multiple of 8 up to 256; views of a packed
    projection are read in place.  Rows of no document are zeros in a new
    result, and left as they are in ``out``.
    """
    what = "compute_packed_attention"
    index = _native.require_inputs(what, q, k, v, cu_seqlens, prefix_lens, alibi_slopes, out)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError(f"{what}: queries [T, Hq, D] and keys and values [T, Hkv, D] expected, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: one dtype for queries, keys and values, got {q.dtype}, {k.dtype}, {v.dtype}")
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    _heads(what, q, Hkv, D)
    scale, cap, window = _scores(what, D, scale, score_cap, window)
    docs = cu_seqlens.numel() - 1
    if docs < 0:
        raise ValueError(f"{what}: cu_seqlens must be int32 or int64 [documents + 1], got none")
    starts = _ints(what, "cu_seqlens", cu_seqlens, docs + 1)
    prefix = None if prefix_lens is None else _ints(what, "prefix_lens", prefix_lens, docs)
    slopes = _slopes(what, alibi_slopes, Hq)
    res = _out(what, out, q, k, v)
    q, (qt, qh) = _rows(q)
    k, (kt, kh) = _rows(k)
    v, (vt, vh) = _rows(v)
    p = _native.PackedParams(
        _TYPES[q.dtype], docs, Hq, Hkv, D, bool(causal), window, out is None, T, scale, cap, starts.data_ptr(),
        None if prefix is None else prefix.data_ptr(), None if slopes is None else slopes.data_ptr(), q.data_ptr(),
        k.data_ptr(), v.data_ptr(), res.data_ptr(), qt, qh, kt, kh, vt, vh, Hq * D, D)
    _native.launch_on(index, _native.lib().smaq_packed_attention, "smaq_packed_attention", ctypes.byref(p))
    return res


def compute_paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                            seq_lens: torch.Tensor, max_seq_len: int, *, scale: Optional[float] = None,
                            window: int = 0, score_cap: float = 0.0, alibi_slopes: Optional[torch.Tensor] = None,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence, queries [B, Hq, D], over a paged
    exact cache: keys and values [blocks, block_size, Hkv, D] (views such as
    ``kv_cache[0]`` and ``kv_cache[1]`` of a flash-layout cache), token t of
    sequence b in row ``t % block_size`` of block ``block_table[b, t // block_size]``.

    The query is the sequence's last token, number ``seq_lens[b] - 1``; its key
    and value are in the cache.  It sees the last ``window`` tokens (0: all),
    scored as in ``compute_packed_attention``.  ``max_seq_len`` bounds every
    length (longer sequences are cut to it) and sets how the length is split over
    the card.  Tokens whose table entry is no block of the cache are left out; a
    sequence without a token gives zeros.

    fp16 or bf16, head_dim a multiple of 8 up to 256, block_size a multiple of
    16, cache rows on 16 bytes.
    """
    what = "compute_paged_attention"
    index = _native.require_inputs(what, q, k_cache, v_cache, block_table, seq_lens, alibi_slopes, out)
    if q.dim() != 3 or k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.shape[3] != q.shape[2]:
        raise ValueError(f"{what}: queries [B, Hq, D] and caches [blocks, block_size, Hkv, D] expected, got "
                         f"{tuple(q.shape)}, {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError(f"{what}: one dtype for queries and caches, got {q.dtype}, {k_cache.dtype}, {v_cache.dtype}")
    B, Hq, D = q.shape
    blocks, bs, Hkv, _ = k_cache.shape
    _heads(what, q, Hkv, D)
    scale, cap, window = _scores(what, D, scale, score_cap, window)
    if bs <= 0 or bs % 16:
        raise ValueError(f"{what}: block_size must be a multiple of 16, got {bs}")
    k_steps, v_steps = _native.row_steps(k_cache), _native.row_steps(v_cache)
    if k_steps is None or v_steps is None:
        raise ValueError(f"{what}: cache rows must be dense and start on 16 bytes")
    if block_table.dim() != 2 or block_table.shape[0] < B or block_table.dtype not in _INTEGERS:
        raise ValueError(f"{what}: block_table must be an integer [>= {B}, max_blocks] tensor, got "
                         f"{tuple(block_table.shape)} {block_table.dtype}")
    if seq_lens.dim() != 1 or seq_lens.shape[0] < B or seq_lens.dtype not in _INTEGERS:
        raise ValueError(f"{what}: seq_lens must be int32 or int64 [>= {B}], got {tuple(seq_lens.shape)} "
                         f"{seq_lens.dtype}")
    if max_seq_len < 0:
        raise ValueError(f"{what}: max_seq_len must be 0 or more, got {max_seq_len}")
    slopes = _slopes(what, alibi_slopes, Hq)
    res = _out(what, out, q, k_cache, v_cache)
    q, (qb, qh) = _rows(q)
    table = _int32(block_table)
    lens = seq_lens.contiguous()
    p = _native.PagedParams(
        _TYPES[q.dtype], B, Hq, Hkv, D, bs, blocks, table.shape[1], window, lens.dtype == torch.int64,
        min(int(max_seq_len), 0x7fffffff),
        scale, cap, lens.data_ptr(), table.data_ptr(), None if slopes is None else slopes.data_ptr(), q.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), res.data_ptr(), qb, qh, Hq * D, D, *k_steps, *v_steps)
    lib, ref = _native.lib(), ctypes.byref(p)
    size = lib.smaq_paged_workspace_bytes(ref)
    if size:
        if size < 0:
            _native._check(-1, "smaq_paged_attention")
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), size
    _native.launch_on(index, lib.smaq_paged_attention, "smaq_paged_attention", ref)
    return res
