"""Block tables and slots of a scheduler step, built on the GPU.

The paged caches of this package (``PagedQuantizedKV``, the vLLM adapter's
pools) are addressed by a block table and written by a slot map; this builds
both from the requests' lengths without reading one back to the host.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from smaq_amd import _native


_LENGTHS = (torch.int32, torch.int64)


class PageStep(NamedTuple):
    slot_mapping: torch.Tensor     # int64 [num_tokens], -1: no slot
    positions: torch.Tensor        # int64 [num_tokens]
    query_start_loc: torch.Tensor  # int32 [requests + 1]
    seq_lens: torch.Tensor         # int32 [requests]
    status: torch.Tensor           # int32 [2]: pages taken, new tokens without a slot


def build_page_step(context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                    free_blocks: torch.Tensor, block_size: int, num_tokens: int) -> PageStep:
    """Pages for ``new_lens[b]`` new tokens behind the ``context_lens[b]`` that
    request b has in the cache, and the new tokens' slots and positions.

    Request b's missing pages are taken off the front of ``free_blocks`` (int32,
    ids of 0 or more), in request order, and written into its row of
    ``block_table`` (int32 [requests, max_blocks], contiguous, updated in place:
    nothing but the taken entries changes, so the same call again gives the same
    result).  ``num_tokens`` sizes the token outputs: at least the sum of
    ``new_lens``, more for a padded step; places behind the last token get slot
    -1 and position 0.  A token without a page (the free list or the row too
    short, the entry of a partly filled page negative) gets slot -1 and is
    counted in ``status[1]``; ``status[0]`` is the number of pages the step takes
    off the list, more than it holds when it was too short.
    """
    index = _native.require_inputs("build_page_step", context_lens, new_lens, block_table, free_blocks)
    n = context_lens.shape[0] if context_lens.dim() else -1
    for t, what in ((context_lens, "context_lens"), (new_lens, "new_lens")):
        if t.dim() != 1 or t.shape[0] != n or t.dtype not in _LENGTHS:
            raise ValueError(f"build_page_step: {what} must be int32 or int64 [requests], got {tuple(t.shape)} {t.dtype}")
    if (block_table.dim() != 2 or block_table.shape[0] < n or block_table.dtype != torch.int32
            or not block_table.is_contiguous()):
        raise ValueError(f"build_page_step: block_table must be a contiguous int32 [>= {n}, max_blocks] tensor, got "
                         f"{tuple(block_table.shape)} {block_table.dtype}")
    if free_blocks.dim() != 1 or free_blocks.dtype != torch.int32:
        raise ValueError(f"build_page_step: free_blocks must be a one-dimensional int32 tensor, got "
                         f"{tuple(free_blocks.shape)} {free_blocks.dtype}")
    ctx, new, free = context_lens.contiguous(), new_lens.contiguous(), free_blocks.contiguous()
    table, width = block_table.data_ptr(), block_table.shape[1]
    end = table + 4 * block_table.shape[0] * width
    for t, what in ((ctx, "context_lens"), (new, "new_lens"), (free, "free_blocks")):
        start = t.data_ptr()
        if start < end and start + t.shape[0] * t.element_size() > table:
            raise ValueError(f"build_page_step: block_table shares memory with {what}")
    num_tokens, block_size = int(num_tokens), int(block_size)
    if not (0 <= num_tokens <= 0x7fffffff and 1 <= block_size <= 65536):
        raise ValueError(f"build_page_step: num_tokens must be 0 or more, got {num_tokens}, and block_size 1..65536, got "
                         f"{block_size}")
    dev = block_table.device
    slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    positions = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    starts = torch.empty(n + 1, dtype=torch.int32, device=dev)
    seq_lens = torch.empty(n, dtype=torch.int32, device=dev)
    status = torch.empty(2, dtype=torch.int32, device=dev)
    _native.launch_on(index, _native.lib().smaq_page_step, "smaq_page_step", ctx.data_ptr(), ctx.element_size(),
                      new.data_ptr(), new.element_size(), n, table, width, free.data_ptr(), free.shape[0],
                      block_size, num_tokens, slots.data_ptr(), positions.data_ptr(), starts.data_ptr(),
                      seq_lens.data_ptr(), status.data_ptr())
    return PageStep(slots, positions, starts, seq_lens, status)
