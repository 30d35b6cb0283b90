"""Argument checks and launch context shared by the serving operators."""

from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib
from ._lib import ShiftError
from .paged import PagedLayout, describe
from .shift_kernels import _ERR, _err_word, _raise_bits, take_errors

_NO_GUARD = contextlib.nullcontext()


def cuda_on(device: torch.device | None, **tensors: torch.Tensor | None) -> torch.device:
    """Every tensor given is on one CUDA device (``device`` if not None), which is returned."""
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise ShiftError(f"{name} is on {t.device}: the kernels are CUDA-only and have no "
                             "CPU path")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ShiftError(f"{name} is on {t.device}, other arguments are on {device}")
    return device


def refuse_grad(what: str, hint: str, *tensors: torch.Tensor | None) -> None:
    """These operators record no gradient; a caller who would lose one is told."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ShiftError(f"{what} records no gradient: {hint}")


def int32_vector(t: torch.Tensor, name: str, numel: int | None = None) -> None:
    if t.dtype != torch.int32 or t.dim() != 1 or (t.numel() > 1 and t.stride(0) != 1):
        raise ShiftError(f"{name} must be a contiguous int32 vector, got {t.dtype} "
                         f"{tuple(t.shape)}")
    if numel is not None and t.numel() != numel:
        raise ShiftError(f"{name} has {t.numel()} entries, {numel} are wanted")


def block_table_rows(t: torch.Tensor) -> tuple[int, int]:
    """(row stride, width) of an int32 ``[requests, width]`` block table."""
    if t.dtype != torch.int32 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ShiftError("block_tables must be int32 [requests, width] with contiguous rows, got "
                         f"{t.dtype} {tuple(t.shape)}")
    width = t.shape[1]
    if t.shape[0] > 1 and t.stride(0) < width:
        raise ShiftError("block_tables' rows overlap")
    return (t.stride(0) if t.shape[0] > 1 else width), width


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


def heads_rows(t: torch.Tensor, name: str, written: bool = False) -> tuple[int, int]:
    """(token, head) strides of a ``[tokens, heads, head_size]`` tensor with contiguous heads."""
    if t.dim() != 3:
        raise ShiftError(f"{name} must be [tokens, heads, head_size], got {tuple(t.shape)}")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ShiftError(f"{name}'s head dimension must be contiguous")
    if written and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride(), strict=True)):
        raise ShiftError(f"{name} is written and must not repeat its elements")
    return t.stride(0), t.stride(1)


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
    if scale.dtype != torch.float32 or tuple(scale.shape) != (geo.num_blocks, geo.heads):
        raise ShiftError(f"{name} must be fp32 [{geo.num_blocks}, {geo.heads}] (blocks, heads), "
                         f"got {scale.dtype} {tuple(scale.shape)}")
    return scale.stride(0), scale.stride(1)


def status_word(device: torch.device) -> torch.Tensor:
    """The device's status word (``take_errors`` reads and clears it)."""
    if device.index not in _ERR:
        if torch.cuda.is_current_stream_capturing():
            raise ShiftError("call the operator once on this device before capturing it: its "
                             "status word must not live in a graph's memory")
        with torch.cuda.device(device):
            _err_word(device)
            torch.cuda.current_stream().synchronize()
    return _ERR[device.index]


class Launch:
    """The device's status word and current stream, with that device current inside ``with``."""

    __slots__ = ("device", "err", "guard", "stream")

    def __init__(self, device: torch.device) -> None:
        self.device = device
        self.err = status_word(device).data_ptr()
        self.guard = (_NO_GUARD if torch.cuda.current_device() == device.index
                      else torch.cuda.device(device))

    def __enter__(self) -> Launch:
        self.guard.__enter__()
        self.stream = torch.cuda.current_stream(self.device).cuda_stream
        return self

    def __exit__(self, *exc) -> None:
        self.guard.__exit__(*exc)


def finish(status: int, what: str, device: torch.device, check: bool) -> None:
    _lib.check(status, what)
    if check:
        _raise_bits(take_errors(device), what)
