"""Appending to a block-scaled e4m3 cache and the attention over it, against 64-bit forms.

Append is defined bit for bit (powers of two, one rounding), so codes and scales are equal.

Attention's tolerance, with A = sum p|v| / sum p of the element and eps / 2 half a step:
  out   eps_t/2 |o|  (its own rounding)
      + 2^-11 A      (P to f16)
      + 2^-20 A      (P below f16's normal range, 2^-25 each over at most 2^5 kept terms a unit of P;
                      ex2.approx within 2^-22; fp32 sums)
      + d A          with d = 2^-20 * max_j sum|q||k| scale: a score is a sum of exact products in
                      fp32, within 2^-24 of its magnitude a rounding over some 2^3 levels, and e^d - 1 ~ d
  lse   d + 2^-20 + 2^-22 |lse|.
"""

from __future__ import annotations

import random

import pytest
import torch

from marathon_b200 import _lib
from marathon_b200.block_scaled import append_block_scaled, attend_block_scaled
from marathon_b200.shift_kernels import ShiftError, take_errors
import serving

F8 = torch.float8_e4m3fn
NAN_CODE = 0x7F


def _i32(cuda, x):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def _cum(x):
    out = [0]
    for v in x:
        out.append(out[-1] + v)
    return out


class Case:
    """A batch: lens are whole lengths, new the rows of each request (its last ones)."""

    def __init__(self, cuda, lens, new, hq, hk, d, bs, layout="nhd", dtype=torch.bfloat16, seed=0,
                 pow2=False, pad=0, loud=1.0):
        g = torch.Generator().manual_seed(seed)
        r = random.Random(seed)
        self.lens, self.new, self.qs = lens, new, _cum(new)
        self.bs, self.layout, self.hk, self.d = bs, layout, hk, d
        need = [-(-n // bs) for n in lens]
        blocks = sum(need) + 3
        ids = list(range(blocks))
        r.shuffle(ids)
        it = iter(ids)
        width = max(need + [0]) + 2
        self.tables = [[next(it) if b < m else -1 for b in range(width)] for m in need]
        shape = serving.cache_shape(layout, blocks, bs, hk, d)
        codes = (torch.randn(shape, generator=g) * 90 * loud).clamp(-448, 448).to(F8)
        # what belongs to no request holds NaN codes and NaN scales
        raw = codes.view(torch.uint8)
        used = torch.zeros(blocks, bs, dtype=torch.bool)
        for n, t in zip(lens, self.tables, strict=True):
            for p in range(n):
                used[t[p // bs], p % bs] = True
        for side in serving.sides(raw, layout):
            side[~used] = NAN_CODE
        self.kv = codes
        if pow2:
            self.ks, self.vs = (2.0 ** torch.randint(-9, -4, (blocks, hk), generator=g).float()
                                for _ in range(2))
        else:
            self.ks, self.vs = (torch.rand(blocks, hk, generator=g) * 0.02 + 0.003 for _ in range(2))
        free = ~used.any(1)
        self.ks[free] = self.vs[free] = float("nan")
        self.q = torch.randn(sum(new) + pad, hq, d, generator=g).to(dtype)
        self.dev = [x.to(cuda) for x in (self.q, self.kv, self.ks, self.vs)]
        self.step = [_i32(cuda, self.tables) if self.tables else torch.zeros(0, 2, dtype=torch.int32, device=cuda),
                     _i32(cuda, self.qs), _i32(cuda, lens)]
        self.bounds = dict(max_query_len=max(new + [0]), max_seq_len=max(lens + [0]))

    def run(self, **kw):
        return attend_block_scaled(*self.dev, *self.step, self.bs, self.layout, return_lse=True,
                                   check=True, **{**self.bounds, **kw})

    def check(self, got, **kw):
        out, lse = (x.cpu().double() for x in got)
        scale = kw.get("scale") or self.d**-0.5
        want, wlse, mag, big = serving.attend(
            self.q, self.kv, self.ks, self.vs, self.tables, self.qs, self.lens, self.bs, self.layout,
            scale, kw.get("causal", True), kw.get("window", 0))
        d = 2.0**-20 * big
        tol = torch.finfo(self.q.dtype).eps / 2 * want.abs() + (2.0**-11 + 2.0**-20 + d[..., None]) * mag
        assert bool(out.isfinite().all())
        bad = (out - want).abs() > tol
        assert not bool(bad.any()), (int(bad.sum()), float(((out - want).abs() / tol.clamp(min=1e-30)).max()))
        none = wlse == float("-inf")
        assert torch.equal(none, lse == float("-inf"))
        assert bool((out[none] == 0).all())
        off = torch.where(none, 0.0, (lse - wlse).abs())
        assert bool((off <= d + 2.0**-20 + 2.0**-22 * wlse.abs().nan_to_num(posinf=0)).all()), float(off.max())


# --------------------------------------------------------------- without a GPU
def test_refuse_cpu_tensors():
    kv = torch.zeros(2, 16, 1, 128, dtype=torch.uint8)
    s = torch.ones(2, 1)
    t = torch.zeros(1, 2, dtype=torch.int32)
    k = torch.zeros(1, 1, 64)
    one = torch.ones(2, dtype=torch.int32)
    with pytest.raises(ShiftError, match="CUDA"):
        append_block_scaled(k, k, kv, s, s, t, one, one[:1], 16)
    with pytest.raises(ShiftError, match="CUDA"):
        attend_block_scaled(k.half(), kv, s, s, t, one, one[:1], 16, max_query_len=1, max_seq_len=1)


def test_entry_points_validate_before_any_launch():
    lib = _lib.load()
    paged = lambda **kw: _lib.Paged(**{**dict(  # noqa: E731
        blk_stride=4096, off_stride=256, head_stride=128, num_blocks=4, block_size=16, heads=2,
        head_size=64, dtype=_lib.E4M3), **kw})

    def app(dtype=0, k=16, tok=128, head=64, rows=1, p=None, kb=16, ks=16, bt=16, stride=2, width=2,
            qs=16, lens=16, reqs=1, err=16):
        return lib.mshift_append_block_scaled(dtype, k, tok, head, 16, 128, 64, rows, p or paged(), kb, 16,
                                              ks, 2, 1, 16, 2, 1, bt, stride, width, qs, lens, reqs, err, None)

    def att(dtype=0, q=16, tok=256, rows=1, hq=4, p=None, kb=16, bt=16, stride=2, width=2, reqs=1,
            maxq=1, maxs=16, window=0, out=16, ws=None, wsb=0, err=16):
        return lib.mshift_attend_block_scaled(dtype, q, tok, 64, rows, hq, p or paged(), kb, 16, 16, 2, 1, 16,
                                              2, 1, bt, stride, width, 16, 16, reqs, maxq, maxs, 0.1, 1,
                                              window, out, 256, 64, None, 0, ws, wsb, err, None)

    for call in (app, att):
        for bad in (dict(rows=-1), dict(reqs=-1), dict(stride=1), dict(width=-1), dict(kb=None),
                    dict(kb=24), dict(bt=None), dict(err=None), dict(tok=129),
                    dict(p=paged(heads=0)), dict(p=paged(block_size=0)), dict(p=paged(off_stride=250))):
            assert call(**bad) == _lib.EINVAL, bad
        assert call(p=paged(dtype=_lib.BF16)) == _lib.EUNSUPPORTED
        assert call(rows=0) == _lib.OK
        assert call(reqs=0) == _lib.OK
    assert app(dtype=3) == _lib.EUNSUPPORTED
    assert app(p=paged(head_size=96)) == _lib.EUNSUPPORTED
    for bad in (dict(k=None), dict(k=24), dict(ks=None), dict(qs=None), dict(lens=None)):
        assert app(**bad) == _lib.EINVAL, bad
    assert att(dtype=2) == _lib.EUNSUPPORTED
    for bad in (dict(q=None), dict(q=24), dict(hq=3), dict(hq=0), dict(out=None), dict(maxq=-1),
                dict(maxs=-1), dict(window=-1), dict(maxs=100000)):  # the last needs a workspace
        assert att(**bad) == _lib.EINVAL, bad
    assert lib.mshift_attend_workspace(1, 4, 2, 64, 1, 1, 16) == 0
    assert lib.mshift_attend_workspace(1, 4, 3, 64, 1, 1, 16) == -1
    assert lib.mshift_attend_workspace(1, 4, 2, 64, 1, 1, 100000) > 0
    assert lib.mshift_attend_workspace(0, 4, 2, 64, 1, 1, 100000) == 0


# ----------------------------------------------------------------------- append
def _append(cuda, cached, new, heads, d, bs, layout, dtype, seed=0, fill=None, pad=0):
    lens = [c + n for c, n in zip(cached, new, strict=True)]
    case = Case(cuda, lens, new, heads, heads, d, bs, layout, seed=seed, pow2=seed % 2 == 0)
    g = torch.Generator().manual_seed(seed + 1)
    n = sum(new) + pad
    k = (torch.randn(n, heads, d, generator=g) * 10.0 ** (torch.rand(n, 1, 1, generator=g) * 4 - 2)).to(dtype)
    v = torch.randn(n, heads, d, generator=g).to(dtype)
    if fill is not None:
        fill(k, v)
    kv, ks, vs = (x.clone() for x in case.dev[1:])
    append_block_scaled(k.to(cuda), v.to(cuda), kv, ks, vs, *case.step, bs, layout, check=True)
    wkv, wks, wvs = case.kv.double(), case.ks.double(), case.vs.double()
    serving.append(k, v, wkv, wks, wvs, case.tables, case.qs, lens, bs, layout)
    torch.testing.assert_close(ks.cpu().double(), wks, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(vs.cpu().double(), wvs, rtol=0, atol=0, equal_nan=True)
    if seed % 2 == 0:
        torch.testing.assert_close(kv.cpu().double(), wkv, rtol=0, atol=0, equal_nan=True)
        return
    # an old scale that is no power of two: code * (old / new) and x / new round in fp32
    # before they round to e4m3, which can move a value next to a border by one step
    got = kv.cpu().double()
    assert torch.equal(got.isnan(), wkv.isnan())
    off = (got - wkv).abs().nan_to_num()
    step = torch.exp2(torch.floor(torch.log2(wkv.abs().nan_to_num().clamp(min=2.0**-6))) - 3)
    assert bool((off <= step).all()) and float((off > 0).double().mean()) < 1e-3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("cached,new,heads,d,bs,layout", [
    ([0], [1], 1, 64, 16, "nhd"),
    ([5, 16, 0, 31], [1, 1, 1, 1], 8, 128, 16, "nhd"),
    ([3, 0, 100, 17], [40, 0, 5, 16], 2, 128, 16, "hnd"),
    ([7, 0], [90, 33], 3, 64, 24, "split"),
    ([1, 130], [300, 2], 2, 256, 128, "split_blocks"),
    ([2] * 40, [3] * 40, 1, 128, 1, "nhd"),
    ([9], [200], 2, 256, 16, "hnd"),
])
@pytest.mark.parametrize("seed", [0, 1])
def test_append_is_the_definition(cuda, dtype, cached, new, heads, d, bs, layout, seed):
    _append(cuda, cached, new, heads, d, bs, layout, dtype, seed, pad=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_extremes(cuda, dtype):
    """Zeros, infinities, NaN, the type's largest and smallest values, exact powers of two."""
    top = torch.finfo(dtype).max

    def fill(k, v):
        k[0] = 0
        k[1, :, 3] = float("inf")
        k[2, :, 5] = float("nan")
        k[3] = float("-inf")
        k[20] = top
        k[40] = 1e-38
        v[0] = 448.0
        v[16:40] = 0
        v[18, 0, 0] = 2.0**-64
        v[41] = 449.0

    _append(cuda, [4], [60], 2, 128, 16, "nhd", dtype, 0, fill)


@pytest.mark.gpu
def test_append_strided_rows_and_steps_in_turn(cuda):
    """k and v as views of a fused projection, one token at a time: the same blocks as a 64-bit
    cache that takes the same steps."""
    heads, d, bs, n = 2, 128, 16, 40
    case = Case(cuda, [n, n], [n, n], heads, heads, d, bs, pow2=True)
    fused = torch.randn(2 * n, 3 * heads * d, device=cuda).bfloat16()
    k, v = (fused[:, i * heads * d: (i + 1) * heads * d].view(2 * n, heads, d) for i in (1, 2))
    kv, ks, vs = (x.clone() for x in case.dev[1:])
    wkv, wks, wvs = case.kv.double(), case.ks.double(), case.vs.double()
    for at in range(n):
        rows = torch.tensor([at, n + at], device=cuda)
        lens = [at + 1, at + 1]
        step = (case.step[0], _i32(cuda, [0, 1, 2]), _i32(cuda, lens))
        append_block_scaled(k[rows], v[at::n], kv, ks, vs, *step, bs, check=True)
        serving.append(k[rows].cpu(), v[at::n].cpu(), wkv, wks, wvs, case.tables, [0, 1, 2], lens, bs, "nhd")
    torch.testing.assert_close(ks.cpu().double(), wks, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(kv.cpu().double(), wkv, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(vs.cpu().double(), wvs, rtol=0, atol=0, equal_nan=True)


@pytest.mark.gpu
def test_append_bad_blocks_and_lengths_are_flagged_and_skipped(cuda):
    heads, d, bs = 2, 64, 16
    take_errors(cuda)
    case = Case(cuda, [20, 20], [20, 20], heads, heads, d, bs, pow2=True)
    k = torch.randn(40, heads, d, device=cuda).half()
    for col, value, flag in ((1, -1, _lib.EBIT_SLOT), (1, 1 << 30, _lib.EBIT_SLOT)):
        kv, ks, vs = (x.clone() for x in case.dev[1:])
        t = case.step[0].clone()
        t[1, col] = value
        append_block_scaled(k, k, kv, ks, vs, t, *case.step[1:], bs)
        assert take_errors(cuda) == flag
        bad = case.tables[1][1]
        assert torch.equal(kv.view(torch.uint8)[bad], case.dev[1].view(torch.uint8)[bad])
        assert not torch.equal(kv.view(torch.uint8)[case.tables[0][1]],
                               case.dev[1].view(torch.uint8)[case.tables[0][1]])
    kv, ks, vs = (x.clone() for x in case.dev[1:])
    append_block_scaled(k, k, kv, ks, vs, case.step[0][:, :1], *case.step[1:], bs)
    assert take_errors(cuda) == _lib.ERR_POOL
    append_block_scaled(k, k, kv, ks, vs, case.step[0], case.step[1], _i32(cuda, [20, 7]), bs)
    assert take_errors(cuda) == _lib.ERR_LENGTHS
    with pytest.raises(ShiftError, match="past the call's bound"):
        append_block_scaled(k, k, kv, ks, vs, case.step[0], case.step[1], _i32(cuda, [20, 7]), bs, check=True)


# -------------------------------------------------------------------- attention
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,new,hq,hk,d,bs,layout", [
    ([1], [1], 1, 1, 64, 16, "nhd"),
    ([1, 17, 0, 300], [1, 1, 0, 1], 8, 2, 128, 16, "nhd"),
    ([33, 64, 5000], [1, 1, 1], 5, 1, 128, 16, "hnd"),
    ([700, 3, 81], [1, 2, 4], 8, 2, 64, 24, "split"),
    ([257, 40], [1, 3], 6, 3, 256, 32, "split_blocks"),
    ([50, 129, 400], [50, 1, 37], 4, 2, 128, 16, "nhd"),
    ([130, 200], [130, 129], 8, 8, 64, 16, "hnd"),
    ([301, 64], [80, 64], 10, 2, 128, 8, "nhd"),
    ([90], [41], 4, 1, 256, 16, "nhd"),
    ([37, 2], [1, 1], 32, 1, 128, 1, "nhd"),
    ([600, 45, 9], [600, 45, 9], 5, 1, 128, 64, "split"),
    ([20, 0, 7], [0, 0, 7], 2, 2, 64, 16, "nhd"),
])
def test_attention_matches_the_formula(cuda, dtype, lens, new, hq, hk, d, bs, layout):
    c = Case(cuda, lens, new, hq, hk, d, bs, layout, dtype, seed=len(lens) + hq)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 5, 16, 100])
@pytest.mark.parametrize("lens,new,hq,hk,d,bs", [
    ([300, 77, 18], [1, 1, 1], 4, 1, 128, 16),
    ([300, 77, 18], [140, 3, 18], 4, 2, 64, 16),
    ([200, 31], [9, 31], 3, 1, 128, 24),
])
def test_windows_and_full_attention(cuda, causal, window, lens, new, hq, hk, d, bs):
    c = Case(cuda, lens, new, hq, hk, d, bs, seed=window)
    c.check(c.run(causal=causal, window=window), causal=causal, window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("scale,loud", [(1.0, 1.0), (0.02, 1.0), (-0.05, 1.0), (0.3, 5.0)])
def test_sharp_and_flat_scores(cuda, scale, loud):
    """From near-uniform weights to a single key, with growing maxima along the keys."""
    c = Case(cuda, [900, 64], [1, 64], 4, 2, 128, 16, seed=3, loud=loud)
    c.check(c.run(scale=scale), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_scales_far_apart(cuda, d):
    """Block scales over many binades: large values with small weights and the reverse."""
    c = Case(cuda, [200, 170], [1, 40], 4, 2, d, 16, seed=9)
    g = torch.Generator().manual_seed(1)
    c.vs = torch.where(c.vs.isnan(), c.vs, 2.0 ** torch.randint(-30, 30, c.vs.shape, generator=g).float())
    c.ks = torch.where(c.ks.isnan(), c.ks, c.ks * 4.0 ** torch.randint(-4, 2, c.ks.shape, generator=g))
    c.dev[2], c.dev[3] = c.ks.to(cuda), c.vs.to(cuda)
    c.check(c.run())


@pytest.mark.gpu
def test_small_and_large_queries(cuda):
    """bf16 rows from 1e-30 to 1e30 against keys that bring the scores back to order one."""
    c = Case(cuda, [100, 100, 100], [1, 1, 1], 4, 2, 64, 16, seed=2)
    c.q[0] *= 1e-30
    c.q[2] *= 1e18
    for r, by in ((0, 1e30), (2, 1e-18)):
        ids = torch.tensor([b for b in c.tables[r] if b >= 0])
        c.ks[ids] *= by
    c.dev = [x.to(cuda) for x in (c.q, c.kv, c.ks, c.vs)]
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("bound", [1000, 20000, 300000])
def test_splits_and_loose_bounds(cuda, bound):
    """Bounds far above the lengths: empty splits join to the same result."""
    c = Case(cuda, [1000, 16, 1, 0, 700], [1, 1, 1, 0, 2], 5, 1, 128, 16, seed=4)
    c.check(c.run(max_seq_len=bound, max_query_len=7))
    c.check(c.run(max_seq_len=bound, window=33), window=33)


@pytest.mark.gpu
def test_rows_behind_the_last_request(cuda):
    c = Case(cuda, [40, 300], [1, 60], 4, 2, 128, 16, pad=9)
    for bound in (300, 40000):
        out, lse = c.run(max_seq_len=bound)
        assert bool((out[61:] == 0).all()) and bool((lse[61:] == float("-inf")).all())
        c.check((out, lse))
        mine = torch.full_like(out, 7.0)
        got, lse2 = c.run(max_seq_len=bound, out=mine)
        assert got.data_ptr() == mine.data_ptr() and bool((mine[61:] == 7).all())
        assert torch.equal(mine[:61], out[:61]) and torch.equal(lse, lse2)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new,hq,hk,d,bs,layout,window", [
    ([2500], [300], 4, 1, 128, 16, "nhd", 0),
    ([3300, 700, 20], [90, 513, 1], 10, 2, 64, 32, "split", 0),
    ([1900], [1900], 1, 1, 128, 16, "hnd", 300),
    ([1500, 40], [77, 40], 6, 2, 128, 24, "nhd", 0),
    ([2048, 2049], [64, 65], 2, 1, 64, 128, "split_blocks", 0),
    ([1100], [130], 5, 1, 256, 16, "nhd", 0),
])
def test_many_rows_over_many_key_tiles(cuda, lens, new, hq, hk, d, bs, layout, window):
    """Longer than every ring of stages, with and without splits of the keys."""
    c = Case(cuda, lens, new, hq, hk, d, bs, layout, seed=len(lens))
    c.check(c.run(window=window), window=window)
    c.check(c.run(window=window, max_seq_len=60000), window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 60])
def test_nan_keys_reach_the_rows_that_see_them_and_no_others(cuda, new):
    """Every place of a step in turn, so that each way an exponential is worked out meets one."""
    at = 130
    c = Case(cuda, [200, 150], [new, new], 4, 2, 128, 16, seed=5)
    good = c.run()
    for key in range(at, at + 18):
        kv = c.dev[1].clone()
        block = c.tables[0][key // 16]
        kv.view(torch.uint8)[block, key % 16, 1, 7] = NAN_CODE
        out, lse = attend_block_scaled(c.dev[0], kv, *c.dev[2:], *c.step, 16, "nhd", return_lse=True,
                                       check=True, **c.bounds)
        row = torch.arange(2 * new, device=cuda)
        hit = (row < new) & (200 - new + row >= key)
        assert bool(lse[hit][:, 2:].isnan().all()) and bool(out[hit][:, 2:].isnan().all())
        assert torch.equal(out[~hit], good[0][~hit]) and torch.equal(lse[~hit], good[1][~hit])
        assert torch.equal(out[:, :2], good[0][:, :2])


@pytest.mark.gpu
def test_empty_steps_and_rows_before_the_first_request(cuda):
    c = Case(cuda, [40, 9], [0, 0], 4, 2, 128, 16, pad=5)
    for bound in (40, 40000):
        out, lse = c.run(max_query_len=0, max_seq_len=bound)
        assert bool((out == 0).all()) and bool((lse == float("-inf")).all())
    c = Case(cuda, [40], [3], 4, 2, 128, 16, pad=5)
    want, _ = c.run()
    c.step[1] = _i32(cuda, [2, 5])
    c.dev[0] = c.dev[0].roll(2, 0)
    out, lse = c.run()
    assert torch.equal(out[2:5], want[:3]) and bool((out[:2] == 0).all()) and bool((out[5:] == 0).all())
    assert bool((lse[:2] == float("-inf")).all())


@pytest.mark.gpu
def test_check_cannot_be_captured(cuda):
    c = Case(cuda, [40], [1], 4, 2, 128, 16)
    c.run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = attend_block_scaled(*c.dev, *c.step, 16, "nhd", **c.bounds)
        with pytest.raises(ShiftError, match="captured"):
            c.run()
    g.replay()
    assert torch.equal(out, c.run()[0])


@pytest.mark.gpu
def test_strided_queries_outputs_and_scales(cuda):
    c = Case(cuda, [60, 200], [3, 70], 4, 2, 128, 16, seed=6)
    want, wl = c.run()
    n = c.q.shape[0]
    fused = torch.zeros(n, 12, 128, dtype=c.q.dtype, device=cuda)
    fused[:, 4:8] = c.dev[0]
    wide = torch.zeros(n, 4, 256, dtype=c.q.dtype, device=cuda)
    q, ks = c.dev[0], c.dev[2]
    c.dev[0] = fused[:, 4:8]
    c.dev[2] = torch.stack((ks, ks)).permute(1, 2, 0)[..., 0]
    got, gl = c.run(out=wide[..., 64:192])
    assert torch.equal(got, want) and torch.equal(gl, wl)
    assert bool((wide[..., :64] == 0).all()) and bool((wide[..., 192:] == 0).all())
    c.dev[0] = q.transpose(0, 1).contiguous().transpose(0, 1)
    got, _ = c.run()
    assert torch.equal(got, want)
    one = Case(cuda, [60], [5], 4, 2, 64, 16)  # one row for every token
    one.q = one.q[:1].expand(5, 4, 64)
    one.dev[0] = one.q[:1].to(cuda).expand(5, 4, 64)
    one.check(one.run())


@pytest.mark.gpu
def test_cache_with_gaps_between_blocks_and_past_32_bits(cuda):
    """A cache whose strides leave room between rows, and blocks 5 GB apart."""
    heads, d, bs = 2, 64, 16
    c = Case(cuda, [50, 90], [1, 30], 4, heads, d, bs, seed=8)
    blocks = c.kv.shape[0]
    far = 5 * 2**30
    buf = torch.empty(far + blocks * bs * heads * 256, dtype=torch.uint8, device=cuda)
    gap = buf.as_strided((blocks, bs, heads, 2 * d), (bs * heads * 256, heads * 256, 256, 1))
    gap.copy_(c.dev[1].view(torch.uint8))
    c.dev[1] = gap.view(F8)
    c.check(c.run())
    # three blocks of a cache with a block stride of 2.5 GB, the last past 2^32 bytes
    three = buf.as_strided((3, bs, heads, 2 * d), (far // 2, heads * 2 * d, 2 * d, 1))
    c = Case(cuda, [20], [1], 4, heads, d, bs, seed=8)
    if c.kv.shape[0] > 3:
        c.kv, c.ks, c.vs = c.kv[[c.tables[0][0], 4, c.tables[0][1]]], c.ks[:3], c.vs[:3]
        c.ks, c.vs = torch.full((3, heads), 0.01), torch.full((3, heads), 0.02)
        c.tables = [[0, 2]]
    three.copy_(c.kv.view(torch.uint8))
    c.dev = [c.q.to(cuda), three.view(F8), c.ks.to(cuda), c.vs.to(cuda)]
    c.step[0] = _i32(cuda, c.tables)
    c.check(c.run())


@pytest.mark.gpu
def test_append_and_many_rows_in_blocks_past_32_bits(cuda):
    """Blocks 2.5 GB apart, so that the third starts past 2^32 bytes."""
    heads, d, bs, stride = 2, 64, 16, 5 * 2**29
    buf = torch.zeros(2 * stride + bs * heads * 2 * d, dtype=torch.uint8, device=cuda)
    kv = buf.as_strided((3, bs, heads, 2 * d), (stride, heads * 2 * d, 2 * d, 1)).view(F8)
    ks, vs = (torch.ones(3, heads, device=cuda) for _ in range(2))
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(30, heads, d, generator=g).bfloat16() for _ in range(2))
    step = [_i32(cuda, [[0, 2]]), _i32(cuda, [0, 30]), _i32(cuda, [30])]
    append_block_scaled(k.to(cuda), v.to(cuda), kv, ks, vs, *step, bs, check=True)
    want = torch.zeros(3, bs, heads, 2 * d, dtype=torch.float64)
    wks, wvs = (torch.ones(3, heads, dtype=torch.float64) for _ in range(2))
    serving.append(k, v, want, wks, wvs, [[0, 2]], [0, 30], [30], bs, "nhd")
    for b in range(3):
        assert torch.equal(kv[b].cpu().double(), want[b])
    assert torch.equal(ks.cpu().double(), wks) and torch.equal(vs.cpu().double(), wvs)
    c = Case(cuda, [30], [30], 4, heads, d, bs)
    c.kv, c.ks, c.vs, c.tables = torch.stack([kv[b].cpu() for b in range(3)]), wks, wvs, [[0, 2]]
    c.dev, c.step = [c.dev[0], kv, ks, vs], step
    c.check(c.run())


@pytest.mark.gpu
def test_bad_blocks_lengths_and_bounds_are_flagged(cuda):
    take_errors(cuda)
    c = Case(cuda, [64, 64], [1, 20], 4, 2, 128, 16, seed=1)
    good = c.run()

    def run(**kw):
        return attend_block_scaled(*c.dev, *c.step, c.bs, c.layout, return_lse=True, **{**c.bounds, **kw})

    for value in (-1, 1 << 29):
        t = c.step[0].clone()
        t[1, 1] = value
        was, c.step[0] = c.step[0], t
        out, lse = run()
        assert take_errors(cuda) == _lib.EBIT_SLOT
        assert torch.equal(out[0], good[0][0]) and bool(out.isfinite().all())
        c.step[0] = was
    # the tokens of the bad block are left out, the others are not
    c2 = Case(cuda, [64], [1], 4, 2, 128, 16, seed=1)
    t = c2.step[0].clone()
    t[0, :] = -1
    out, lse = attend_block_scaled(*c2.dev, t, *c2.step[1:], 16, return_lse=True, **c2.bounds)
    assert take_errors(cuda) == _lib.EBIT_SLOT
    assert bool((out == 0).all()) and bool((lse == float("-inf")).all())
    run(max_seq_len=63)
    assert take_errors(cuda) == _lib.ERR_LENGTHS
    run(max_query_len=19)
    assert take_errors(cuda) == _lib.ERR_LENGTHS
    was, c.step[0] = c.step[0], c.step[0][:, :3]
    out, _ = run()
    assert take_errors(cuda) == _lib.ERR_POOL and bool(out.isfinite().all())
    c.step[0] = was
    c.step[2] = _i32(cuda, [64, 7])  # more rows than tokens: those before position 0 see nothing
    out, lse = run()
    assert take_errors(cuda) == _lib.ERR_LENGTHS
    assert bool((out[1:14] == 0).all()) and bool((lse[1:14] == float("-inf")).all())
    assert bool(out.isfinite().all()) and bool((out[14:] != 0).any())
    c.step[2] = _i32(cuda, [64, -5])
    out, lse = run()
    assert take_errors(cuda) == _lib.ERR_LENGTHS and bool((out[1:] == 0).all())
    c.step[2] = _i32(cuda, [64, 64])
    c.step[1] = _i32(cuda, [0, 50, 3])  # offsets out of order and past the rows stay inside them
    run()
    assert take_errors(cuda) & _lib.ERR_LENGTHS
    with pytest.raises(ShiftError, match="past the call's bound"):
        c.run(max_seq_len=63)


@pytest.mark.gpu
def test_two_graphs_other_streams_and_repeats(cuda):
    """Two captured calls replayed in turn with an eager one between them; the same bits each time."""
    a = Case(cuda, [2000, 300], [1, 1], 8, 2, 128, 16, seed=1)
    b = Case(cuda, [900, 1500, 40], [1, 2, 40], 8, 2, 128, 16, seed=2)
    want = [c.run() for c in (a, b)]
    graphs, got = [], []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(attend_block_scaled(*c.dev, *c.step, c.bs, c.layout, return_lse=True, **c.bounds))
        graphs.append(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(side):
            other = b.run()
        graphs[1].replay()
    torch.cuda.synchronize()
    for x, y in zip([*got, other], [*want, want[1]], strict=True):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


@pytest.mark.gpu
def test_refusals(cuda):
    c = Case(cuda, [40], [2], 4, 2, 128, 16)
    q, kv, ks, vs = c.dev
    bad = [
        (dict(q=q.float()), "bf16 or fp16"),
        (dict(q=q[:, :3]), "does not fit"),
        (dict(q=q[..., :64]), "does not fit"),
        (dict(q=q.transpose(1, 2)), "contiguous"),
        (dict(q=q.clone().requires_grad_()), "gradient"),
        (dict(q=torch.zeros(2, 4, 132, dtype=q.dtype, device=cuda)[..., :128]), "16-byte"),
        (dict(kv=kv.to(torch.bfloat16)), "float8"),
        (dict(kv=kv[..., :192]), "head_size"),
        (dict(ks=ks[:, :1]), "k_scale"),
        (dict(vs=vs.double()), "v_scale"),
        (dict(q=q.cpu()), "CUDA"),
        (dict(scale=float("inf")), "finite"),
        (dict(window=-1), "non-negative"),
        (dict(max_seq_len=-1), "non-negative"),
        (dict(out=torch.empty_like(q)[:1]), "out must be"),
        (dict(out=q), "shares memory"),
        (dict(out=torch.empty_like(q)[:1].expand(2, 4, 128)), "repeat"),
        (dict(tables=c.step[0].long()), "int32"),
        (dict(qs=c.step[1][:1]), "entries"),
        (dict(lens=c.step[2].repeat(2)), "entries"),
    ]
    for kw, match in bad:
        kw = dict(kw)
        args = [kw.pop("q", q), kw.pop("kv", kv), kw.pop("ks", ks), kw.pop("vs", vs),
                kw.pop("tables", c.step[0]), kw.pop("qs", c.step[1]), kw.pop("lens", c.step[2])]
        with pytest.raises(ShiftError, match=match):
            attend_block_scaled(*args, 16, "nhd", **{**c.bounds, **kw})
    with pytest.raises(ShiftError, match="block size"):
        attend_block_scaled(q, kv, ks, vs, *c.step, 32, "nhd", **c.bounds)
    k = torch.zeros(2, 2, 128, dtype=torch.bfloat16, device=cuda)
    for args, match in (
        ((k, k.half(), kv, ks, vs), "both be"), ((k[:, :1], k, kv, ks, vs), "must be"),
        ((k, k[:1], kv, ks, vs), "must be"), ((k, k, kv, ks, ks), "two tensors"),
        ((k, k, kv, ks[:1].expand_as(ks), vs), "repeat"),
        ((k.clone().requires_grad_(), k, kv, ks, vs), "gradient"),
        ((torch.zeros(2, 2, 130, dtype=k.dtype, device=cuda)[..., :128], k, kv, ks, vs), "16-byte"),
        ((k, k, kv[:1].expand_as(kv), ks, vs), "overlap"),
    ):
        with pytest.raises(ShiftError, match=match):
            append_block_scaled(*args, *c.step, 16, "nhd")


def test_workspaces_stay_small_whatever_the_bounds():
    """Partial results go by the caller's bounds: a loose one must not ask for more than a few GB."""
    lib = _lib.load()
    r = random.Random(0)
    for _ in range(5000):
        hk, group = r.choice([1, 2, 4, 8]), r.choice([1, 2, 5, 16])
        args = (r.randint(1, 20000), hk * group, hk, r.choice([64, 128, 256]), r.randint(1, 256),
                r.choice([1, 4, r.randint(1, 20000)]), r.choice([1, 100, 40000, 1 << 20, 1 << 30]))
        assert 0 <= lib.mshift_attend_workspace(*args) <= 3 << 30, args
    assert lib.mshift_attend_workspace(256, 32, 8, 128, 256, 1, 1 << 20) < 200 << 20
    assert lib.mshift_attend_workspace(1, 4, 2, 64, 1, 1, (1 << 30) + 1) == -1
