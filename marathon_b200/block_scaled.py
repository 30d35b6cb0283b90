"""A paged cache held in 8 bits with a scale for each block of tokens and head.

The shift path's e4m3 caches have one scale a layer, which the caller calibrates.
Here every block has its own scale for each head, kept beside the cache in two
fp32 tensors ``k_scale`` and ``v_scale`` of shape ``[blocks, heads]``: an
element is ``code * scale[block, head]``.  :func:`append_block_scaled` writes new tokens
and chooses the scales; :func:`attend_block_scaled` is the attention that reads the cache, for decoding,
chunks and whole prefills in one batch.  The codes lie in any of the paged
layouts of :mod:`marathon_b200.paged` (``nhd``, ``hnd``, ``split``, ``split_blocks``); head sizes 64, 128 and
256.  A cache that the shift path filled is read too: its layer's scale, expanded to ``[blocks, heads]``, is
every block's.

Both take a step as :func:`marathon_b200.block_maps.block_maps` describes it: request ``r`` owns the rows
``query_start[r]:query_start[r + 1]``, its last row stands at position ``seq_lens[r] - 1``,
and position ``p`` lies in block ``block_tables[r, p // block_size]``.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from ._serve import (
    block_table_rows, cuda_on, distinct, geometry, heads_rows, int32_vector, launch, overlap, refuse_grad,
    scale_strides, tangents, whole_rows,
)
from .paged import dtype_code

__all__ = ["append_block_scaled", "attend_block_scaled"]

HEAD_SIZES = (64, 128, 256)


def _step(kv, k_scale, v_scale, block_tables, query_start, seq_lens, block_size, layout):
    """Checks what both operators take; (geometry, its record, K base, V base, step arguments)."""
    geo, paged = geometry(kv, block_size, layout)
    if geo.head_size not in HEAD_SIZES:
        raise _lib.ShiftError(f"head_size {geo.head_size} is not one of {HEAD_SIZES}")
    k_base = kv.data_ptr()
    if k_base % 16:
        raise _lib.ShiftError("the cache must start on a 16-byte boundary")
    reqs, stride, width = block_table_rows(block_tables)
    int32_vector(query_start, "query_start", reqs + 1)
    int32_vector(seq_lens, "seq_lens", reqs)
    cache = (paged, k_base, k_base + geo.v_offset, k_scale.data_ptr(),
             *scale_strides(k_scale, geo, "k_scale"), v_scale.data_ptr(),
             *scale_strides(v_scale, geo, "v_scale"))
    step = (block_tables.data_ptr(), stride, width, query_start.data_ptr(), seq_lens.data_ptr(), reqs)
    return geo, cache, step


def append_block_scaled(
    k: torch.Tensor,
    v: torch.Tensor,
    kv: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,
    query_start: torch.Tensor,
    seq_lens: torch.Tensor,
    block_size: int,
    layout: str | None = None,
    *,
    check: bool = False,
) -> None:
    """Quantise the step's rows ``k``, ``v`` (``[tokens, heads, head_size]``, bf16, fp16 or fp32)
    into the cache ``kv`` at their requests' last positions, in place.

    A block's scale is the least power of two that brings its largest finite element to at
    most 448 (at least 2^-64).  A block that already holds earlier tokens of its request
    keeps them: its scale only grows, and their codes are requantised when it does
    (exact but for codes that become subnormal).  A block whose first token is among the
    rows starts afresh whatever its scale was.  Infinities become the largest code, NaN stays NaN.

    Rows behind the last request are not written.  No two requests of a call may write the same block
    (copy a shared block before appending to it).  Flagged and skipped: a block outside
    the cache, positions past the block table, rows before position 0.  Flagged: offsets past the rows
    (those there are keep their places), below zero or out of order (which of their rows are written is
    unspecified).
    """
    dev = cuda_on("k v kv k_scale v_scale block_tables query_start seq_lens", k, v, kv, k_scale, v_scale,
                  block_tables, query_start, seq_lens)
    if k.requires_grad or v.requires_grad or k_scale.requires_grad or v_scale.requires_grad or tangents():
        refuse_grad("append_block_scaled", "detach its arguments", k, v, k_scale, v_scale)
    geo, cache, step = _step(kv, k_scale, v_scale, block_tables, query_start, seq_lens, block_size,
                             layout)
    code = dtype_code(k.dtype)
    if code == _lib.E4M3 or v.dtype != k.dtype:
        raise _lib.ShiftError(f"k and v must both be bf16, fp16 or fp32, got {k.dtype} and {v.dtype}")
    n = k.shape[0]
    want = (n, geo.heads, geo.head_size)
    k_rows, v_rows = (k.data_ptr(), *heads_rows(k, "k")), (v.data_ptr(), *heads_rows(v, "v"))
    vec = 4 if code == _lib.F32 else 8
    for name, t in (("k", k), ("v", v)):
        if t.shape != want:
            raise _lib.ShiftError(f"{name} must be [tokens, {geo.heads}, {geo.head_size}], got "
                                  f"{tuple(t.shape)}")
    if k_rows[0] % 16 or k_rows[1] % vec or k_rows[2] % vec:
        k_rows = (k_rows[0], *whole_rows(k, "k", vec))
    if v_rows[0] % 16 or v_rows[1] % vec or v_rows[2] % vec:
        v_rows = (v_rows[0], *whole_rows(v, "v", vec))
    apart = 4 * geo.num_blocks * geo.heads  # bytes of a contiguous scale
    if not (kv.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
        apart = min(apart, 1)
        for name, t in (("kv", kv), ("k_scale", k_scale), ("v_scale", v_scale)):
            if not distinct(t):
                raise _lib.ShiftError(f"{name} is written and must not repeat or overlap its elements")
    if abs(cache[3] - cache[6]) < apart:
        raise _lib.ShiftError("k_scale and v_scale must be two tensors")
    launch(_lib.load().mshift_append_block_scaled, "append_block_scaled", dev,
           (code, *k_rows, *v_rows, n, *cache, *step), check)


_workspaces: dict[tuple, int] = {}  # shapes of a call -> bytes of workspace it needs


def attend_block_scaled(
    q: torch.Tensor,
    kv: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,
    query_start: torch.Tensor,
    seq_lens: torch.Tensor,
    block_size: int,
    layout: str | None = None,
    *,
    max_query_len: int,
    max_seq_len: int,
    scale: float | None = None,
    causal: bool = True,
    window: int = 0,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
    check: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of the step's rows ``q`` (``[tokens, query heads, head_size]``, bf16 or fp16) over the cache.

    Query head ``j`` reads KV head ``j // (query heads / heads)``.  The row at position
    ``p`` sees keys ``0..p`` of its request (``causal=False``: all of them), of those
    only the last ``window`` (positions above ``p - window``) if ``window > 0``.  ``scale`` multiplies the
    scores (default ``head_size ** -0.5``).  ``max_query_len`` and ``max_seq_len`` are host
    bounds of the requests' row counts and ``seq_lens``; they size the launch, so a graph is captured with the
    largest values its replays will meet.

    Returns ``out`` (``q``'s type and shape), and with ``return_lse`` the rows' natural-log sums of
    exponentials (fp32 ``[tokens, query heads]``).  A row that sees no key gets zeros and
    ``-inf``.  Rows behind the last request and rows past ``max_query_len`` are left as they were in a
    given ``out``, and zeros otherwise (lse ``-inf`` either way).  Keys at positions that no row of a tile of
    rows may see are not read, so stale codes there do no harm, NaN included; a NaN among the values of a
    token that later rows of the same request see can reach its earlier rows too.  A row whose scores are all
    NaN gets NaN, and so does one that sees a scale of NaN.  Queries and weights are rounded to f16 for the products, whose sums are fp32; a bf16 result
    does not show the weights' 2^-11, the error of an fp16 one grows by a fifth.  Value scales must be
    positive (below 2^-64 they are read as 2^-64) and those of a request within 2^96 of each other.

    Flagged: a needed block outside the cache (its keys count as unseen), lengths below zero or past
    the bounds (cut off there), positions past the block table (unseen), offsets past the rows of ``q``
    (those there are keep their places), below zero or out of order (results are unspecified).
    """
    dev = cuda_on("q kv k_scale v_scale block_tables query_start seq_lens out", q, kv, k_scale, v_scale,
                  block_tables, query_start, seq_lens, out)
    if q.requires_grad or k_scale.requires_grad or v_scale.requires_grad or tangents() or \
            (out is not None and out.requires_grad):
        refuse_grad("attend_block_scaled", "a cache of codes is not trained through", q, k_scale, v_scale, out)
    geo, cache, step = _step(kv, k_scale, v_scale, block_tables, query_start, seq_lens, block_size,
                             layout)
    if q.dtype is torch.bfloat16:
        code = _lib.BF16
    elif q.dtype is torch.float16:
        code = _lib.F16
    else:
        raise _lib.ShiftError(f"q must be bf16 or fp16, got {q.dtype}")
    q_tok, q_head = heads_rows(q, "q")
    rows, hq, head_size = q.shape
    if head_size != geo.head_size or hq == 0 or hq % geo.heads:
        raise _lib.ShiftError(f"q {tuple(q.shape)} does not fit {geo.heads} heads of {geo.head_size}")
    q_at = q.data_ptr()
    if q_at % 16 or q_tok % 8 or q_head % 8:
        q_tok, q_head = whole_rows(q, "q", 8)
    if not 0 <= max_query_len < 2**31 or not 0 <= max_seq_len <= 2**30 or not 0 <= window < 2**31:
        raise _lib.ShiftError("max_query_len and window must be non-negative int32s, max_seq_len at most "
                              "2^30 and non-negative")
    scale = head_size ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= 2.0**127:  # times log2 e it is an fp32
        raise _lib.ShiftError(f"scale must be finite and at most 2^127, got {scale}")
    reqs = step[-1]
    lse = None
    zero_tail = out is None
    if zero_tail:
        # the kernels write every row, unless there is no request and so no kernel
        if not reqs:
            out = q.new_zeros((rows, hq, head_size))
        else:
            out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((rows, hq, head_size))
        o_tok, o_head = hq * head_size, head_size
        if return_lse:
            lse = q.new_empty((rows, hq), dtype=torch.float32)
            if not reqs:
                lse.fill_(-math.inf)
    else:
        o_tok, o_head = heads_rows(out, "out", written=True)
        if out.shape != q.shape or out.dtype is not q.dtype:
            raise _lib.ShiftError(f"out must be {q.dtype} {tuple(q.shape)}, got {out.dtype} "
                                  f"{tuple(out.shape)}")
        if out.data_ptr() % 16 or o_tok % 8 or o_head % 8:
            o_tok, o_head = whole_rows(out, "out", 8)
        for name, t in (("q", q), ("kv", kv), ("k_scale", k_scale), ("v_scale", v_scale)):
            if overlap(out, t):
                raise _lib.ShiftError(f"out shares memory with {name}")
        if return_lse:  # rows behind the last request have -inf where out keeps what it held
            lse = q.new_full((rows, hq), -math.inf, dtype=torch.float32)
    lib = _lib.load()
    key = (rows, hq, geo.heads, head_size, reqs, max_query_len, max_seq_len)
    need = _workspaces.get(key)
    if need is None:
        if len(_workspaces) > 4096:
            _workspaces.clear()
        need = _workspaces[key] = max(lib.mshift_attend_workspace(*key), 0)
    # from the caching allocator, on this stream: calls and graphs do not share it
    work = q.new_empty(need, dtype=torch.uint8) if need else None
    launch(lib.mshift_attend_block_scaled, "attend_block_scaled", dev, (
        code, q_at, q_tok, q_head, rows, hq, *cache, *step, max_query_len, max_seq_len, scale,
        int(causal), window, out.data_ptr(), o_tok, o_head, None if lse is None else lse.data_ptr(),
        int(zero_tail), None if work is None else work.data_ptr(), need), check)
    return (out, lse) if return_lse else out
