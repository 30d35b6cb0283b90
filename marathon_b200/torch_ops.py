"""The shift path as PyTorch operators: ``torch.ops.marathon.*``.

Tensor-level entry points over the same native library, for callers that
want PyTorch's operator registry rather than the connector classes (an
operator shows up in profiles and traces under its own name, and
``torch.compile`` treats it as one opaque call that mutates its cache
arguments).  Each operator runs the CUDA kernels and nothing else; CPU tensors
raise.

* ``marathon::scatter_shifted(src, kv!, slots, block_size, hnd, table?)`` --
  the reference's ``scatter_shifted`` (``src/marathon/shift_kernels.py:162-210``)
  with the rotation given as a ``[2, rotary/2]`` cos/sin table (``RopeShift.table``)
  or None for a plain scatter.
* ``marathon::shift_load(stores, kv!, segments, block_tables, inv_freq,
  block_size, layout, k_scales?)`` -- every segment of every session through
  every layer in one launch: the connector's load step
  (``vllm_shift_connector.py:481-534``).
* ``marathon::shift_save(kv, stores!, segments, block_tables, block_size,
  layout)`` -- paged rows back into the store rows at the same positions
  (``vllm_shift_connector.py:539-553``), all layers in one launch.

* ``marathon::block_maps``, ``marathon::rotary_axes``, ``marathon::append_block_scaled`` and
  ``marathon::attend_block_scaled`` -- the serving operators over a block-scaled e4m3 cache,
  with the arguments of :mod:`marathon_b200.block_maps`, :mod:`~marathon_b200.rotary` and
  :mod:`~marathon_b200.block_scaled`.  ``rotary_axes`` records gradients of ``q`` and ``k``
  (the rotation by the negative angles).  Rotary, append and attention refuse to run under
  forward-mode differentiation.

``stores`` is flat, session-major: session ``s``'s layer ``l`` buffer is
``stores[s * n_layers + l]`` (``[capacity, heads, 2*head_size]``).
``segments`` is an int64 ``[n, 5]`` tensor of ``(session, src_start,
dst_start, length, delta)`` rows on the host; for a save ``src_start`` is
ignored and rows ``[dst_start, +length)`` are written.  ``block_tables[s]`` is
session ``s``'s int32 block table (its logical position ``p`` lives in block
``block_tables[s][p // block_size]``).
"""

from __future__ import annotations

import numpy as np
import torch

from ._serve import tangents
from .block_maps import block_maps
from .block_scaled import append_block_scaled, attend_block_scaled
from .paged import KVLayers
from .rotary import rotary_axes
from .shift_kernels import Launcher, RopeShift, RunSpec, ShiftError, StoreView, scatter_shifted

_launchers: dict = {}


def _launcher(kv: list[torch.Tensor], block_size: int, layout: str) -> Launcher:
    """One launcher per set of cache addresses and shapes (their pointers are staged once).

    The cached launcher keeps only the addresses, not the tensors: a cache the
    caller frees is freed, and a later cache at the same addresses with the
    same shape, strides and dtype is served by the same launcher.
    """
    key = (tuple((t.data_ptr(), tuple(t.shape), t.stride(), t.dtype) for t in kv), block_size,
           layout)
    la = _launchers.get(key)
    if la is None:
        if len(_launchers) > 16:
            for old in _launchers.values():
                old.drain()  # their pinned staging may still feed copies in flight
            _launchers.clear()
        fp8 = kv[0].dtype in (torch.float8_e4m3fn, torch.uint8)
        la = Launcher(KVLayers(list(kv), block_size, layout, fp8=fp8))
        la.layers.tensors = []  # the kernels need the staged addresses only
        _launchers[key] = la
    return la


def _view(stores: list[torch.Tensor], n_layers: int) -> StoreView:
    if not stores or len(stores) % n_layers:
        raise ShiftError(f"{len(stores)} store buffers for {n_layers} layers")
    n_sessions = len(stores) // n_layers
    ptrs = np.array([t.data_ptr() for t in stores], dtype=np.uint64).reshape(n_sessions, n_layers)
    caps = np.array([stores[s * n_layers].shape[0] for s in range(n_sessions)], dtype=np.int64)
    t = stores[0]
    for b in stores:
        if not b.is_cuda or b.stride() != t.stride() or b.dtype != t.dtype:
            raise ShiftError("store buffers must be CUDA tensors of one dtype and row layout")
    return StoreView(ptrs, caps, t.stride(0), t.stride(1), list(stores))


def _runs(segments: torch.Tensor, block_tables: list[torch.Tensor], load: bool) -> list[RunSpec]:
    seg = segments.to("cpu", torch.int64).numpy()
    if seg.ndim != 2 or seg.shape[1] != 5:
        raise ShiftError("segments must be [n, 5]: session, src_start, dst_start, length, delta")
    tables = [bt.to(torch.int32).contiguous() for bt in block_tables]
    runs = []
    for s, src, dst, n, delta in seg.tolist():
        if not 0 <= s < len(tables):
            raise ShiftError(f"segment names session {s} of {len(tables)}")
        bt = tables[s]
        if not bt.is_cuda:
            bt = bt.numpy()  # travels inside the batch's descriptor copy
        runs.append(RunSpec(s, src if load else dst, n, delta if load else 0,
                            block_table=bt, paged_start=dst))
    return runs


@torch.library.custom_op("marathon::scatter_shifted", mutates_args=("kv",))
def _scatter_shifted_op(src: torch.Tensor, kv: torch.Tensor, slots: torch.Tensor,
                        block_size: int, hnd: bool, table: torch.Tensor | None = None) -> None:
    shift = None
    if table is not None:
        tab = table.to(torch.float32).reshape(2, table.shape[-1]).contiguous()
        c, sn = tab[0], tab[1]
        # only `table` (and the rotary width) is read by the kernel path; the
        # delta is any non-zero marker: the table already encodes it
        shift = RopeShift(1, None, None, None, torch.cat((c, c)), torch.cat((sn, sn)), tab)
    scatter_shifted(src, kv, slots, block_size, hnd, shift)


@torch.library.custom_op("marathon::shift_load", mutates_args=("kv",))
def _shift_load_op(stores: list[torch.Tensor], kv: list[torch.Tensor], segments: torch.Tensor,
                   block_tables: list[torch.Tensor], inv_freq: torch.Tensor, block_size: int,
                   layout: str, k_scales: torch.Tensor | None = None) -> None:
    la = _launcher(kv, block_size, layout)
    runs = _runs(segments, block_tables, load=True)
    if runs:
        la.load(runs, _view(stores, len(kv)), inv_freq.to(la.device, torch.float32),
                k_scales=k_scales, check=True)


@torch.library.custom_op("marathon::shift_save", mutates_args=("stores",))
def _shift_save_op(kv: list[torch.Tensor], stores: list[torch.Tensor], segments: torch.Tensor,
                   block_tables: list[torch.Tensor], block_size: int, layout: str) -> None:
    la = _launcher(kv, block_size, layout)
    runs = _runs(segments, block_tables, load=False)
    if runs:
        la.save(runs, _view(stores, len(kv)), check=True)


@_scatter_shifted_op.register_fake
def _(src, kv, slots, block_size, hnd, table=None) -> None:
    return None


@_shift_load_op.register_fake
def _(stores, kv, segments, block_tables, inv_freq, block_size, layout, k_scales=None) -> None:
    return None


@_shift_save_op.register_fake
def _(kv, stores, segments, block_tables, block_size, layout) -> None:
    return None


# ------------------------------------------------------------ serving operators
def _no_tangents(what: str) -> None:
    """Tangents end at an operator without a word, and some are out of its sight (``torch.func.jvp``'s)."""
    if tangents():
        raise ShiftError(f"torch.ops.marathon.{what} has no forward-mode gradient")


@torch.library.custom_op("marathon::block_maps", mutates_args=("block_tables",))
def _block_maps_op(
    cached_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor,
    free_blocks: torch.Tensor, free_head: torch.Tensor, block_size: int, tokens: int,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    m = block_maps(cached_lens, new_lens, block_tables, free_blocks, free_head, block_size, tokens)
    return m.query_start, m.seq_lens, m.slots, m.positions, m.free_head


@_block_maps_op.register_fake
def _(cached_lens, new_lens, block_tables, free_blocks, free_head, block_size, tokens):
    reqs = cached_lens.shape[0]
    rows = [cached_lens.new_empty(tokens, dtype=torch.int64) for _ in range(2)]
    return (cached_lens.new_empty(reqs + 1), cached_lens.new_empty(reqs), *rows,
            cached_lens.new_empty(1))


@torch.library.custom_op("marathon::rotary_axes", mutates_args=())
def _rotary_axes_op(
    q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
    axes: torch.Tensor | None = None, inverse: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    _no_tangents("rotary_axes")
    # detached: gradients are recorded around the operator, not in it
    return rotary_axes(q.detach(), k.detach(), positions, inv_freq.detach(), axes, inverse=inverse)


@_rotary_axes_op.register_fake
def _(q, k, positions, inv_freq, axes=None, inverse=False):
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _rotary_axes_setup(ctx, inputs, output) -> None:
    _, _, *tables, ctx.inverse = inputs
    if tables[1].requires_grad:
        raise ShiftError("torch.ops.marathon.rotary_axes records no gradient of inv_freq")
    ctx.save_for_backward(*tables)  # a table changed before the backward pass is noticed there


def _rotary_axes_backward(ctx, dq, dk):
    # a sum's gradient comes as one element read many times: the kernel wants contiguous heads
    dq, dk = (d if d.stride(-1) == 1 else d.contiguous() for d in (dq, dk))
    return *torch.ops.marathon.rotary_axes(dq, dk, *ctx.saved_tensors, not ctx.inverse), None, None, None, None


_rotary_axes_op.register_autograd(_rotary_axes_backward, setup_context=_rotary_axes_setup)


@torch.library.custom_op("marathon::append_block_scaled", mutates_args=("kv", "k_scale", "v_scale"))
def _append_block_scaled_op(
    k: torch.Tensor, v: torch.Tensor, kv: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
    block_tables: torch.Tensor, query_start: torch.Tensor, seq_lens: torch.Tensor, block_size: int,
    layout: str,
) -> None:
    _no_tangents("append_block_scaled")
    append_block_scaled(k, v, kv, k_scale, v_scale, block_tables, query_start, seq_lens, block_size,
                        layout)


@_append_block_scaled_op.register_fake
def _(k, v, kv, k_scale, v_scale, block_tables, query_start, seq_lens, block_size, layout) -> None:
    return None


@torch.library.custom_op("marathon::attend_block_scaled", mutates_args=())
def _attend_block_scaled_op(
    q: torch.Tensor, kv: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
    block_tables: torch.Tensor, query_start: torch.Tensor, seq_lens: torch.Tensor, block_size: int,
    layout: str, max_query_len: int, max_seq_len: int, scale: float | None = None,
    causal: bool = True, window: int = 0,
) -> tuple[torch.Tensor, torch.Tensor]:
    _no_tangents("attend_block_scaled")
    return attend_block_scaled(
        q, kv, k_scale, v_scale, block_tables, query_start, seq_lens, block_size, layout,
        max_query_len=max_query_len, max_seq_len=max_seq_len, scale=scale, causal=causal,
        window=window, return_lse=True)


@_attend_block_scaled_op.register_fake
def _(q, kv, k_scale, v_scale, block_tables, query_start, seq_lens, block_size, layout,
      max_query_len, max_seq_len, scale=None, causal=True, window=0):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)
