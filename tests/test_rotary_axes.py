"""Rotary positions with several axes against the 64-bit formula.

Tolerance.  The kernel rounds the turns left modulo one to fp32 (an angle within
pi 2^-24), sincospif is within 2 ulp (2^-23 each), two products and a sum round three times:
below (3.2 + 4 + 3) 2^-24 < 2^-20 of |x| + |y| for a pair (x, y), then half a step of the type.
"""

from __future__ import annotations

import pytest
import torch

from marathon_b200 import _lib
from marathon_b200.rotary import axis_map, rotary_axes
from marathon_b200.shift_kernels import ShiftError, inv_freq, rope_shift, take_errors
from serving import rotary as plain


def _check(got, x, positions, inv, axes, inverse):
    want = plain(x.cpu(), positions.cpu(), inv.cpu(), axes.cpu(), inverse)
    half = inv.numel()
    pair = x.cpu().double().abs()
    both = pair.clone()
    both[..., :half] += pair[..., half:2 * half]
    both[..., half:2 * half] += pair[..., :half]
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + 2.0**-20 * both
    if x.dtype == torch.float16:
        tol += 2.0**-25  # subnormals
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())
    assert torch.equal(got[..., 2 * half:], x[..., 2 * half:])


def test_axis_map():
    assert axis_map((2, 1, 3)).tolist() == [0, 0, 1, 2, 2, 2]
    assert axis_map((4, 2, 2), interleaved=True).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert axis_map((24, 20, 20), interleaved=True).tolist().count(1) == 20
    with pytest.raises(ShiftError, match="interleaved"):
        axis_map((1, 5, 2), interleaved=True)
    with pytest.raises(ShiftError, match="counts"):
        axis_map(())


def test_refuses_cpu_tensors_and_bad_arguments():
    q = torch.zeros(2, 1, 64)
    with pytest.raises(ShiftError, match="CUDA"):
        rotary_axes(q, None, torch.arange(2), inv_freq(64, 1e4))
    with pytest.raises(ShiftError, match="needs q or k"):
        rotary_axes(None, None, torch.arange(2), inv_freq(64, 1e4))
    lib = _lib.load()

    def call(dtype=0, q=16, n=2, d=64, rot=64, pos=16, n_axes=1, inv=16, err=16, hq=1):
        return lib.mshift_rotary_axes(dtype, q, 64, 64, q, 64, 64, hq, None, 0, 0, None, 0, 0, 0, n, d, rot,
                                      pos, 2, 1, n_axes, inv, None, 0, err, None)

    for bad in (dict(q=None), dict(n=-1), dict(d=0), dict(rot=66), dict(rot=7), dict(pos=None),
                dict(n_axes=0), dict(inv=None), dict(err=None), dict(hq=-1), dict(n=1 << 40)):
        assert call(**bad) == _lib.EINVAL, bad
    assert call(dtype=3) == _lib.EUNSUPPORTED
    assert call(d=1024, rot=1024) == _lib.EUNSUPPORTED
    assert call(n=0) == _lib.OK


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,hq,hk,d,rot,sections,inter", [
    (1, 8, 1, 128, 128, (16, 24, 24), False),
    (7, 5, 5, 64, 64, (32,), False),
    (333, 40, 8, 128, 128, (24, 20, 20), True),
    (4099, 4, 2, 128, 64, (8, 12, 12), False),
    (65, 3, 0, 256, 256, (43, 43, 42), True),
    (33, 2, 1, 80, 20, (4, 3, 3), False),
    (9, 2, 2, 30, 14, (3, 2, 2), True),
    (3, 1, 1, 512, 512, (256,), False),
    (2, 2, 1, 16, 0, (0,), False),
])
def test_matches_the_formula(cuda, dtype, n, hq, hk, d, rot, sections, inter):
    g = torch.Generator().manual_seed(n + d)
    q = torch.randn(n, hq, d, generator=g).to(dtype).to(cuda)
    k = torch.randn(n, hk, d, generator=g).to(dtype).to(cuda) if hk else None
    axes = axis_map(sections, inter, cuda)
    inv = inv_freq(rot, 1e6).to(cuda) if rot else torch.empty(0, device=cuda)
    pos = torch.randint(-5000, 40000, (len(sections), n), generator=g).to(cuda)
    for inverse in (False, True):
        a, b = rotary_axes(q, k, pos, inv, axes, inverse=inverse, check=True)
        _check(a, q, pos, inv, axes, inverse)
        if k is None:
            assert b is None
        else:
            _check(b, k, pos, inv, axes, inverse)


@pytest.mark.gpu
def test_far_positions_and_int32(cuda):
    pos = torch.tensor([[0, 1, 2**20 + 1, 2**31 - 1, -(2**31) + 1, 10**6 + 3]], device=cuda)
    q = torch.randn(6, 2, 128, device=cuda)
    inv, axes = inv_freq(128, 1e6).to(cuda), axis_map((64,), device=cuda)
    a, _ = rotary_axes(q, None, pos, inv, axes, check=True)
    # 2^31 * 2^-53 turns more at the far end, far below the fp32 rounding
    _check(a, q, pos, inv, axes, False)
    b, _ = rotary_axes(q, None, pos[0].int(), inv, check=True)
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_strides_alignment_and_in_place(cuda):
    n, hq, hk, d = 37, 6, 2, 128
    inv, axes = inv_freq(d, 1e6).to(cuda), axis_map((16, 24, 24), device=cuda)
    pos = torch.randint(0, 9000, (3, n), device=cuda)
    base = torch.randn(n, (hq + 2 * hk) * d + 8, device=cuda).bfloat16()
    for shift in (0, 8, 3):  # aligned, aligned to 16 bytes, not aligned
        fused = base.clone()
        q = fused[:, shift: shift + hq * d].view(n, hq, d) if shift != 3 else \
            fused.as_strided((n, hq, d), (fused.stride(0), d, 1), 3)
        k = fused.as_strided((n, hk, d), (fused.stride(0), d, 1), shift + hq * d)
        want_q, want_k = q.clone(), k.clone()
        a, b = rotary_axes(q, k, pos, inv, axes, check=True)
        _check(a, want_q, pos, inv, axes, False)
        _check(b, want_k, pos, inv, axes, False)
        keep = fused[:, shift + (hq + hk) * d:].clone()
        c, e = rotary_axes(q, k, pos, inv, axes, inplace=True, check=True)
        assert c.data_ptr() == q.data_ptr() and torch.equal(q, a) and torch.equal(k, b)
        assert torch.equal(fused[:, shift + (hq + hk) * d:], keep) and e.data_ptr() == k.data_ptr()
    # head-major q, one row for all tokens, positions with a stride
    q = torch.randn(hq, n, d, device=cuda).transpose(0, 1)
    a, _ = rotary_axes(q, None, pos, inv, axes)
    _check(a, q, pos, inv, axes, False)
    one = torch.randn(1, 2, d, device=cuda).expand(n, 2, d)
    a, _ = rotary_axes(one, None, pos.repeat_interleave(2, 1)[:, ::2], inv, axes)
    _check(a, one, pos, inv, axes, False)


@pytest.mark.gpu
def test_deltas_re_rotate_like_the_shift_tables(cuda):
    """With one delta as every token's position, the shift path's rotation: its tables round the
    angle to fp32 first, up to |delta| 2^-24 rad away."""
    n, d, delta = 50, 128, -566
    inv = inv_freq(d, 1e6).to(cuda)
    k = torch.randn(n, 4, d, device=cuda)
    _, got = rotary_axes(None, k, torch.full((n,), delta, device=cuda), inv)
    sh = rope_shift(delta, d, inv, cuda)
    a, b = k[..., :64], k[..., 64:]
    c, s = sh.table[0], sh.table[1]
    want = torch.cat((a * c - b * s, b * c + a * s), -1)
    tol = (abs(delta) * 2.0**-24 + 2.0**-20) * (a.abs() + b.abs())
    assert bool(((got - want).abs() <= torch.cat((tol, tol), -1)).all())


@pytest.mark.gpu
def test_gradient_is_the_inverse(cuda):
    """d(sum w y)/dx by central differences of the fp64 formula, against inverse=True of w."""
    n, d = 5, 64
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(n, 2, d, generator=g), torch.randn(n, 2, d, generator=g)
    pos = torch.randint(0, 3000, (3, n), generator=g)
    inv, axes = inv_freq(d, 1e4), axis_map((10, 11, 11))
    got, _ = rotary_axes(w.to(cuda), None, pos.to(cuda), inv.to(cuda), axes.to(cuda), inverse=True)
    e = 2.0**-10
    for at in ((0, 0, 0), (1, 1, 5), (4, 0, 40), (2, 1, 63), (3, 0, 31)):
        hi, lo = x.double().clone(), x.double().clone()
        hi[at] += e
        lo[at] -= e
        f = [(plain(t, pos, inv, axes, False) * w.double()).sum() for t in (hi, lo)]
        # the function is linear: the difference is exact but for fp64 rounding
        assert abs(float(got[at]) - float(f[0] - f[1]) / (2 * e)) < 2.0**-18


@pytest.mark.gpu
def test_capture_other_stream_and_flags(cuda):
    n, d = 12, 128
    q = torch.randn(n, 4, d, device=cuda).half()
    pos = torch.arange(3 * n, device=cuda).view(3, n)
    inv, axes = inv_freq(d, 1e6).to(cuda), axis_map((16, 24, 24), device=cuda)
    want, _ = rotary_axes(q, None, pos, inv, axes, check=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got, _ = rotary_axes(q, None, pos, inv, axes)
    g.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, _ = rotary_axes(q, None, pos, inv, axes)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(other, want)
    axes[5] = 3
    take_errors(cuda)
    rotary_axes(q, None, pos, inv, axes)
    assert take_errors(cuda) == _lib.EBIT_TABLE


@pytest.mark.gpu
def test_refusals(cuda):
    q = torch.zeros(4, 2, 64, device=cuda)
    pos, inv = torch.zeros(4, dtype=torch.long, device=cuda), inv_freq(64, 1e4).to(cuda)
    for bad, match in (
        (lambda: rotary_axes(q, q.half(), pos, inv), "differ"),
        (lambda: rotary_axes(q, q[:3], pos, inv), "differ"),
        (lambda: rotary_axes(q[..., :32], None, pos, inv), "rotary"),
        (lambda: rotary_axes(q, None, pos[:3], inv), "positions"),
        (lambda: rotary_axes(q, None, pos.float(), inv), "positions"),
        (lambda: rotary_axes(q, None, pos.expand(2, 4), inv), "axes must say"),
        (lambda: rotary_axes(q, None, pos, inv.double()), "fp32"),
        (lambda: rotary_axes(q, None, pos, inv, torch.zeros(3, dtype=torch.int32, device=cuda)), "entries"),
        (lambda: rotary_axes(torch.zeros(4, 64, 2, device=cuda).transpose(1, 2), None, pos, inv), "contiguous"),
        (lambda: rotary_axes(q[0], None, pos, inv), "heads"),
        (lambda: rotary_axes(q.double(), None, pos, inv), "unsupported"),
        (lambda: rotary_axes(q.clone().requires_grad_(), None, pos, inv), "gradient"),
        (lambda: rotary_axes(q[:1].expand(4, 2, 64), None, pos, inv, inplace=True), "repeat"),
        (lambda: rotary_axes(q, q, pos, inv, inplace=True), "share"),
        (lambda: rotary_axes(q, None, pos.cpu(), inv), "CUDA"),
    ):
        with pytest.raises(ShiftError, match=match):
            bad()
