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
from ._serve import Launch, block_table_rows, cuda_on, finish, int32_vector, overlap

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
    narrow, an old entry below 0, negative lengths (read as 0), more tokens than ``tokens``
    (the surplus is dropped, from ``seq_lens`` too).
    """
    dev = cuda_on(None, cached_lens=cached_lens, new_lens=new_lens, block_tables=block_tables,
                  free_blocks=free_blocks, free_head=free_head)
    int32_vector(cached_lens, "cached_lens")
    reqs = cached_lens.numel()
    int32_vector(new_lens, "new_lens", reqs)
    int32_vector(free_blocks, "free_blocks")
    int32_vector(free_head, "free_head", 1)
    stride, width = block_table_rows(block_tables)
    if block_tables.shape[0] != reqs:
        raise _lib.ShiftError(f"{block_tables.shape[0]} block tables for {reqs} requests")
    if block_size <= 0 or not 0 <= tokens < 2**31:
        raise _lib.ShiftError(f"block_size {block_size} and tokens {tokens} must be positive int32s")
    for name, t in (("cached_lens", cached_lens), ("new_lens", new_lens),
                    ("free_blocks", free_blocks), ("free_head", free_head)):
        if overlap(t, block_tables):
            raise _lib.ShiftError(f"{name} shares memory with block_tables, which are written")
    lib = _lib.load()
    with Launch(dev) as on:
        ints = [torch.empty(n, dtype=torch.int32, device=dev) for n in (reqs + 1, reqs, 1)]
        rows = [torch.empty(tokens, dtype=torch.int64, device=dev) for _ in range(2)]
        status = lib.mshift_block_maps(
            cached_lens.data_ptr(), new_lens.data_ptr(), reqs, block_tables.data_ptr(), stride,
            width, free_blocks.data_ptr(), free_blocks.numel(), free_head.data_ptr(), block_size,
            tokens, ints[0].data_ptr(), ints[1].data_ptr(), rows[0].data_ptr(), rows[1].data_ptr(),
            ints[2].data_ptr(), on.err, on.stream)
    finish(status, "block_maps", dev, check)
    return BlockMaps(ints[0], ints[1], rows[0], rows[1], ints[2])
