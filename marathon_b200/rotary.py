"""Rotary positions with several axes (time, height, width), queries and keys in one launch.

The shift path rotates by one axis: a delta for each segment
(:func:`marathon_b200.shift_kernels.rope_tables`).  Models that see images or
video give a token one position for each axis, and each rotary frequency takes
its angle from one of them.  :func:`rotary_axes` applies that to queries and keys; with deltas in the place of
positions it re-rotates reused keys (R(p + d) = R(d) R(p) holds axis by axis),
and ``inverse`` undoes it, which is also its transpose: the gradient of the result
goes back to the inputs through ``inverse=True``.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from . import _lib
from ._serve import cuda_on, heads_rows, int32_vector, launch, overlap, refuse_grad, tangents
from .paged import dtype_code

__all__ = ["axis_map", "rotary_axes"]


def axis_map(sections: Sequence[int], interleaved: bool = False, device=None) -> torch.Tensor:
    """The axis of each rotary frequency (int32), from how many frequencies each axis has.

    Contiguous: ``sections[0]`` frequencies of axis 0, then axis 1, and so on.
    ``interleaved``: frequency ``i`` belongs to axis ``i % len(sections)`` as long as that
    axis has frequencies left in its turn (``i < sections[axis] * len(sections)``), and to axis 0 otherwise.
    """
    n, half = len(sections), sum(sections)
    if n == 0 or min(sections) < 0:
        raise _lib.ShiftError(f"sections must be counts of frequencies, got {tuple(sections)}")
    if interleaved:
        axes = [i % n if i < sections[i % n] * n else 0 for i in range(half)]
        if any(axes.count(a) != sections[a] for a in range(n)):
            raise _lib.ShiftError(f"sections {tuple(sections)} cannot be interleaved: an axis behind "
                                  "the first has more frequencies than turns")
    else:
        axes = [a for a, m in enumerate(sections) for _ in range(m)]
    return torch.tensor(axes, dtype=torch.int32, device=device)


def rotary_axes(
    q: torch.Tensor | None,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    axes: torch.Tensor | None = None,
    *,
    inverse: bool = False,
    inplace: bool = False,
    check: bool = False,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """``q`` and ``k`` (``[tokens, heads, head_size]``, either may be None) rotated by their positions.

    ``positions`` is int32 or int64, ``[tokens]`` or ``[n_axes, tokens]``, of any
    sign; ``inv_freq`` fp32 ``[rotary / 2]`` with ``rotary <= head_size`` (the tail
    passes through); ``axes`` int32 ``[rotary / 2]`` (:func:`axis_map`), or None where all
    frequencies take axis 0.  NeoX half-split pairs, bf16, fp16 or fp32, rotated in fp32 and
    rounded once.  Angles are exact modulo a turn to fp32 precision at any position (for
    frequencies up to 2^64).  Any token and head strides; ``inplace`` writes into ``q`` and ``k``
    themselves.  All tensors on one GPU.  An entry of ``axes`` that names no axis is flagged.
    """
    one = q if q is not None else k
    if one is None:
        raise _lib.ShiftError("rotary_axes needs q or k")
    dev = cuda_on("q k positions inv_freq axes", q, k, positions, inv_freq, axes)
    if one.requires_grad or (k is not None and k.requires_grad) or inv_freq.requires_grad or tangents():
        refuse_grad("rotary_axes", "its gradient is rotary_axes(..., inverse=True) of the result's, and "
                    "torch.ops.marathon.rotary_axes records that of q and k", q, k, inv_freq)
    code = dtype_code(one.dtype)
    if code == _lib.E4M3:
        raise _lib.ShiftError("rotary_axes takes bf16, fp16 or fp32")
    shape = one.shape
    if len(shape) != 3:
        raise _lib.ShiftError(f"q and k must be [tokens, heads, head_size], got {tuple(shape)}")
    n, _, head_size = shape
    hq = 0 if q is None else shape[1]
    hk = 0
    if k is not None:
        kshape = k.shape
        if k.dtype is not one.dtype or len(kshape) != 3 or kshape[0] != n or kshape[2] != head_size:
            raise _lib.ShiftError(f"q {one.dtype} {tuple(shape)} and k {k.dtype} {tuple(kshape)} differ "
                                  "in type, tokens or head size")
        hk = kshape[1]
    if inv_freq.dtype is not torch.float32 or inv_freq.dim() != 1:
        raise _lib.ShiftError("inv_freq must be an fp32 vector")
    half = inv_freq.numel()
    if 2 * half > head_size:
        raise _lib.ShiftError(f"rotary {2 * half} > head_size {head_size}")
    if half > 256 or head_size > 1024:
        raise _lib.ShiftError("rotary_axes takes head sizes up to 1024 and rotary up to 512")
    pshape = positions.shape
    if positions.dtype not in (torch.int32, torch.int64) or len(pshape) not in (1, 2) \
            or pshape[-1] != n:
        raise _lib.ShiftError(f"positions must be int32 or int64 [{n}] or [axes, {n}], got "
                              f"{positions.dtype} {tuple(pshape)}")
    n_axes = pshape[0] if len(pshape) == 2 else 1
    if n_axes == 0:
        raise _lib.ShiftError("positions have no axis")
    if axes is not None:
        int32_vector(axes, "axes", half)
    elif n_axes > 1:
        raise _lib.ShiftError(f"positions have {n_axes} axes: axes must say which each frequency takes")
    if n > 1 and positions.stride(-1) != 1:
        positions = positions.contiguous()
    if half > 1 and inv_freq.stride(0) != 1:
        inv_freq = inv_freq.contiguous()
    q_in = (None, 0, 0) if q is None else (q.data_ptr(), *heads_rows(q, "q", inplace))
    k_in = (None, 0, 0) if k is None else (k.data_ptr(), *heads_rows(k, "k", inplace))
    if inplace:
        if q is not None and k is not None and overlap(q, k) and _interleaved_clash(q, k):
            raise _lib.ShiftError("q and k share elements and cannot both be rotated in place")
        for t in (positions, inv_freq, axes):
            if t is not None and any(x is not None and overlap(t, x) for x in (q, k)):
                raise _lib.ShiftError("an argument shares memory with a tensor rotated in place")
        q_out, k_out, q_to, k_to = q, k, q_in, k_in
    else:
        q_out = q_to = k_out = k_to = None
        if q is not None:
            q_out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
            q_to = (q_out.data_ptr(), hq * head_size, head_size)
        if k is not None:
            k_out = torch.empty_like(k) if k.is_contiguous() else k.new_empty(k.shape)
            k_to = (k_out.data_ptr(), hk * head_size, head_size)
    launch(_lib.load().mshift_rotary_axes, "rotary_axes", dev, (
        code, *q_in, *(q_to or q_in), hq, *k_in, *(k_to or k_in), hk, n, head_size, 2 * half,
        positions.data_ptr(), positions.stride(0) if n_axes > 1 else n,
        int(positions.dtype is torch.int64), n_axes, inv_freq.data_ptr(),
        None if axes is None else axes.data_ptr(), int(inverse)), check)
    return q_out, k_out


def _interleaved_clash(q: torch.Tensor, k: torch.Tensor) -> bool:
    """Whether overlapping address ranges share elements.  Views of one fused projection
    ([tokens, (q heads + k heads) * head_size]) interleave by token without sharing any."""
    if q.stride(0) != k.stride(0) or q.shape[0] < 2:
        return True
    row = q.stride(0)
    width_q = (q.shape[1] - 1) * q.stride(1) + q.shape[2]
    width_k = (k.shape[1] - 1) * k.stride(1) + k.shape[2]
    gap = (k.data_ptr() - q.data_ptr()) // q.element_size()
    return not (0 <= gap - width_q and gap + width_k <= row) and \
        not (0 <= -gap - width_k and -gap + width_q <= row)
