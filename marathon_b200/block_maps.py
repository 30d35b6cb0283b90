"""Block tables and slot maps of one step, built on the GPU from request lengths.

The host-side :func:`marathon_b200.shift_store.slots` needs a request's length
and block table on the host; a step whose lengths live on the GPU (the previous
step's sampler wrote them) would wait for them there.  :func:`block_maps`
takes the lengths where they are and makes, in one launch, what the step's other
operators read: query offsets, whole lengths, slots, positions, and the new
blocks' entries in the block tables.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from ._serve import block_table_rows, cuda_on, int32_vector, launch

__all__ = ["BlockMaps", "block_maps"]


@dataclass(frozen=True)
class BlockMaps:
    """One step's maps.  Request ``r`` has rows ``query_start[r]:query_start[r + 1]``."""

    query_start: torch.Tensor  # int32 [requests + 1]
    seq_lens: torch.Tensor  # int32 [requests]: cached + new tokens
    slots: torch.Tensor  # int64 [tokens]: block * block_size + offset, -1 behind the last request
    positions: torch.Tensor  # int64 [tokens], 0 behind the last request
    free_head: torch.Tensor  # int32 [1]: the free list's next block


def block_maps(
    cached_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_tables: torch.Tensor,
    free_blocks: torch.Tensor,
    free_head: torch.Tensor,
    block_size: int,
    tokens: int,
    *,
    check: bool = False,
) -> BlockMaps:
    """Maps of a step in which request ``r`` gets ``new_lens[r]`` tokens behind its
    ``cached_lens[r]`` (int32, on the GPU).

    The blocks a request lacks are taken from ``free_blocks[free_head:]`` (int32) in
    request order and entered into ``block_tables`` (int32 ``[requests, width]``,
    changed in place); ``free_head`` (int32 ``[1]``) is read, and the new head is
    returned, so feeding it to the next step allocates on.  ``tokens`` is the
    number of rows to map, a host integer and at least the sum of ``new_lens``: a
    step padded to a fixed size maps its padding to slot -1.  The call waits for nothing on the
    host and can be captured into a graph.

    Flagged, with slot -1 (``check=True`` synchronises and raises, otherwise
    :func:`~marathon_b200.shift_kernels.take_errors` tells): a free list that runs out, a table too
    narrow, an old entry or a free block below 0, negative lengths (read as 0), whole lengths
    past int32 (cut there), more tokens than ``tokens`` (the surplus is dropped, from ``seq_lens`` too,
    and takes no blocks).
    """
    dev = cuda_on("cached_lens new_lens block_tables free_blocks free_head", cached_lens, new_lens,
                  block_tables, free_blocks, free_head)
    reqs = int32_vector(cached_lens, "cached_lens")
    int32_vector(new_lens, "new_lens", reqs)
    n_free = int32_vector(free_blocks, "free_blocks")
    int32_vector(free_head, "free_head", 1)
    n_tables, stride, width = block_table_rows(block_tables)
    if n_tables != reqs:
        raise _lib.ShiftError(f"{n_tables} block tables for {reqs} requests")
    if block_size <= 0 or not 0 <= tokens < 2**31:
        raise _lib.ShiftError(f"block_size {block_size} and tokens {tokens} must be positive int32s")
    read = (cached_lens.data_ptr(), new_lens.data_ptr(), free_blocks.data_ptr(), free_head.data_ptr())
    table = block_tables.data_ptr()
    end = table + 4 * ((reqs - 1) * stride + width)
    for at, n in zip(read, (reqs, reqs, n_free, 1), strict=True):
        if at < end and table < at + 4 * n:
            raise _lib.ShiftError("an argument shares memory with block_tables, which are written")
    query_start = cached_lens.new_empty(reqs + 1)
    seq_lens = torch.empty_like(cached_lens)
    head = torch.empty_like(free_head)
    slots = cached_lens.new_empty(tokens, dtype=torch.int64)
    positions = torch.empty_like(slots)
    launch(_lib.load().mshift_block_maps, "block_maps", dev, (
        read[0], read[1], reqs, table, stride, width, read[2], n_free, read[3], block_size, tokens,
        query_start.data_ptr(), seq_lens.data_ptr(), slots.data_ptr(), positions.data_ptr(),
        head.data_ptr()), check)
    return BlockMaps(query_start, seq_lens, slots, positions, head)
