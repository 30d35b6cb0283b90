"""Argument checks and launch context shared by the serving operators."""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import ShiftError
from .paged import PagedLayout, describe
from .shift_kernels import _ERR, _err_word, _raise_bits, take_errors


def cuda_on(names: str, *tensors: torch.Tensor | None) -> int:
    """Every tensor given (named in order by ``names``, None left out) is on one CUDA device,
    whose index is returned."""
    at = -1
    for t in tensors:
        if t is not None:
            i = t.get_device()
            if i < 0 or i != at >= 0:
                name = names.split()[next(j for j, x in enumerate(tensors) if x is t)]
                if i < 0:
                    raise ShiftError(f"{name} is on {t.device}: the kernels are CUDA-only and have no "
                                     "CPU path")
                raise ShiftError(f"{name} is on {t.device}, other arguments are on cuda:{at}")
            at = i
    return at


def tangents() -> bool:
    """Whether forward-mode differentiation is on, so that tensors may carry tangents."""
    return forward_ad._current_level >= 0


def refuse_grad(what: str, hint: str, *tensors: torch.Tensor | None) -> None:
    """These operators record no gradient and carry no tangent; a caller who would lose one is told."""
    given = [t for t in tensors if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        raise ShiftError(f"{what} records no gradient: {hint}")
    if tangents() and any(forward_ad.unpack_dual(t).tangent is not None for t in given):
        raise ShiftError(f"{what} has no forward-mode gradient: {hint}")


def int32_vector(t: torch.Tensor, name: str, numel: int | None = None) -> int:
    """Its length, which is ``numel`` if that is given."""
    shape = t.shape
    if t.dtype is not torch.int32 or len(shape) != 1 or (shape[0] > 1 and t.stride(0) != 1):
        raise ShiftError(f"{name} must be a contiguous int32 vector, got {t.dtype} {tuple(shape)}")
    n = shape[0]
    if numel is not None and n != numel:
        raise ShiftError(f"{name} has {n} entries, {numel} are wanted")
    return n


def block_table_rows(t: torch.Tensor) -> tuple[int, int, int]:
    """(rows, row stride, width) of an int32 ``[requests, width]`` block table."""
    shape = t.shape
    if t.dtype is not torch.int32 or len(shape) != 2 or (shape[1] > 1 and t.stride(1) != 1):
        raise ShiftError("block_tables must be int32 [requests, width] with contiguous rows, got "
                         f"{t.dtype} {tuple(shape)}")
    rows, width = shape
    if rows <= 1:
        return rows, width, width
    stride = t.stride(0)
    if stride < width:
        raise ShiftError("block_tables' rows overlap")
    return rows, stride, width


def span(t: torch.Tensor) -> tuple[int, int]:
    """Addresses [first, end) that a tensor's elements lie in."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride(), strict=True))
    at = t.data_ptr()
    return at, at + (last + 1) * t.element_size()


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def distinct(t: torch.Tensor) -> bool:
    """Whether the elements of a tensor that is written lie in different places: its dimensions
    nest in the order of their strides, each wider than what is inside it."""
    if t.is_contiguous():
        return True
    shape, reach = t.shape, 0
    for stride, n in sorted(zip(t.stride(), shape, strict=True)):
        if n > 1:
            if stride <= reach:
                return 0 in shape
            reach += (n - 1) * stride
    return True


def heads_rows(t: torch.Tensor, name: str, written: bool = False) -> tuple[int, int]:
    """(token, head) strides of a ``[tokens, heads, head_size]`` tensor with contiguous heads."""
    stride = t.stride()
    if len(stride) != 3:
        raise ShiftError(f"{name} must be [tokens, heads, head_size], got {tuple(t.shape)}")
    if stride[2] != 1 and t.shape[2] > 1:
        raise ShiftError(f"{name}'s head dimension must be contiguous")
    if written and not distinct(t):
        raise ShiftError(f"{name} is written and must not repeat or overlap its elements")
    return stride[0], stride[1]


def whole_rows(t: torch.Tensor, name: str, vec: int) -> tuple[int, int]:
    """``heads_rows`` of a tensor some of whose strides are no whole 16-byte vectors of ``vec`` elements:
    zeros for dimensions of one, whose strides say nothing; else rows do not start on 16-byte boundaries."""
    tok, head = (s if n > 1 else 0 for s, n in zip(t.stride()[:2], t.shape[:2], strict=True))
    if t.data_ptr() % 16 or tok % vec or head % vec:
        raise ShiftError(f"{name}'s rows must start on 16-byte boundaries")
    return tok, head


_geometries: dict = {}


def geometry(kv: torch.Tensor, block_size: int, layout: str | None) -> tuple[PagedLayout, object]:
    """Geometry of an e4m3 paged cache and its ``mshift_paged`` record, worked out
    once for each shape, stride and layout."""
    key = (kv.shape, kv.stride(), kv.dtype, block_size, layout)
    got = _geometries.get(key)
    if got is None:
        if kv.dtype not in (torch.float8_e4m3fn, torch.uint8):
            raise ShiftError(f"a block-scaled cache holds float8_e4m3fn codes, got {kv.dtype}")
        geo = describe(kv, block_size, layout, fp8=True)
        if (geo.blk_stride | geo.off_stride | geo.head_stride | geo.v_offset) % 16:
            raise ShiftError("the cache's strides must be whole 16-byte vectors")
        sizes = ((geo.num_blocks, geo.blk_stride), (geo.block_size, geo.off_stride),
                 (geo.heads, geo.head_stride))
        if any(n > 1 and s < geo.head_size for n, s in sizes):
            raise ShiftError("the cache's rows overlap")
        if len(_geometries) > 256:
            _geometries.clear()
        got = _geometries[key] = (geo, ctypes.byref(geo.struct()))
    return got


def scale_strides(scale: torch.Tensor, geo: PagedLayout, name: str) -> tuple[int, int]:
    if scale.dtype is not torch.float32 or scale.shape != (geo.num_blocks, geo.heads):
        raise ShiftError(f"{name} must be fp32 [{geo.num_blocks}, {geo.heads}] (blocks, heads), "
                         f"got {scale.dtype} {tuple(scale.shape)}")
    return scale.stride()


_status: dict[int, int] = {}  # device index -> address of its status word


def _status_word(index: int) -> int:
    """Address of the device's status word (``take_errors`` reads and clears it)."""
    if index not in _ERR and torch.cuda.is_current_stream_capturing():
        raise ShiftError("call the operator once on this device before capturing it: its "
                         "status word must not live in a graph's memory")
    with torch.cuda.device(index):
        at = _status[index] = _err_word(torch.device("cuda", index)).data_ptr()
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream().synchronize()  # other streams may use it from now on
    return at


def launch(fn, what: str, device: int, args: tuple, check: bool) -> None:
    """Call the entry point with the device's status word and current stream behind ``args``,
    that device being current."""
    if check and torch.cuda.is_current_stream_capturing():
        raise ShiftError(f"{what}: check=True waits for the device and cannot be captured")
    err = _status.get(device) or _status_word(device)
    stream = torch._C._cuda_getCurrentRawStream(device)
    if torch.cuda.current_device() == device:
        status = fn(*args, err, stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, err, stream)
    if status or check:
        finish(status, what, device, check)


def finish(status: int, what: str, device: int, check: bool) -> None:
    _lib.check(status, what)
    if check:
        _raise_bits(take_errors(torch.device("cuda", device)), what)
