"""Edges of the serving operators: bounds that a request passes, NaN, flagged lengths, what is refused."""

from __future__ import annotations

import math

import pytest
import torch
from torch.autograd import forward_ad

import marathon_b200  # noqa: F401  (registers the operators)
import serving
from marathon_b200 import _lib
from marathon_b200._serve import geometry
from marathon_b200.block_maps import block_maps
from marathon_b200.block_scaled import append_block_scaled, attend_block_scaled
from marathon_b200.rotary import axis_map, rotary_axes
from marathon_b200.shift_kernels import ShiftError, inv_freq, rope_shift, scatter_shifted, take_errors
from test_block_scaled import NAN_CODE, Case, _cum, _i32


def _attend(c, **kw):
    """The call without ``check``, so that what it flags is left for the test."""
    return attend_block_scaled(*c.dev, *c.step, c.bs, c.layout, return_lse=True, **{**c.bounds, **kw})


def _check_rows(c, got, rows, **kw):
    """The listed rows against the formula, within the tolerances of test_block_scaled.py."""
    out, lse = (x.cpu().double()[rows] for x in got)
    want, wlse, mag, big = (x[rows] for x in serving.attend(
        c.q, c.kv, c.ks, c.vs, c.tables, c.qs, c.lens, c.bs, c.layout, c.d**-0.5, **kw))
    d = 2.0**-20 * big
    tol = torch.finfo(c.q.dtype).eps / 2 * want.abs() + (2.0**-11 + 2.0**-20 + d[..., None]) * mag
    assert bool(((out - want).abs() <= tol).all())
    none = wlse == -math.inf
    assert torch.equal(none, lse == -math.inf) and bool((out[none] == 0).all())
    off = torch.where(none, 0.0, (lse - wlse).abs())
    assert bool((off <= d + 2.0**-20 + 2.0**-22 * torch.where(none, 0.0, wlse).abs()).all())


# ------------------------------------------------------ rows past max_query_len
PAST = [  # rows of the requests, bound, query heads, KV heads, head size: few rows, several tiles, many rows
    ([1, 2, 1, 3], 1, 10, 2, 128),
    ([2, 1, 9], 1, 4, 4, 64),
    ([2, 9, 1], 2, 8, 2, 256),
    ([7, 3, 40], 3, 10, 2, 128),
    ([90, 30, 200], 60, 4, 2, 64),
]


def _past(cuda, new, hq, hk, d):
    lens = [700 + 311 * i + n for i, n in enumerate(new)]
    return Case(cuda, lens, new, hq, hk, d, 16, seed=len(new) + d, pad=2)


@pytest.mark.gpu
@pytest.mark.parametrize("most", [2000, 30720])
@pytest.mark.parametrize("new,bound,hq,hk,d", PAST)
def test_rows_past_the_query_bound_are_left_and_the_others_right(cuda, new, bound, hq, hk, d, most):
    """One request or more has more rows than the caller's bound, with splits of the keys."""
    take_errors(cuda)
    c = _past(cuda, new, hq, hk, d)
    out = torch.full((c.q.shape[0], hq, d), 7.0, dtype=c.q.dtype, device=cuda)
    got = _attend(c, max_query_len=bound, max_seq_len=most, out=out)
    assert take_errors(cuda) == _lib.ERR_LENGTHS
    rows = [q + i for q, n in zip(c.qs, new, strict=False) for i in range(min(n, bound))]
    _check_rows(c, got, rows)
    rest = [i for i in range(c.q.shape[0]) if i not in set(rows)]
    assert bool((out[rest] == 7).all()) and bool((got[1][rest] == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new,bound,hq,hk,d", PAST)
def test_rows_past_the_query_bound_leave_what_is_behind_the_workspace(cuda, new, bound, hq, hk, d):
    take_errors(cuda)
    c = _past(cuda, new, hq, hk, d)
    lib, rows, most = _lib.load(), c.q.shape[0], 30720
    geo, paged = geometry(c.dev[1], c.bs, c.layout)
    need = lib.mshift_attend_workspace(rows, hq, hk, d, len(new), bound, most)
    assert need > 0
    work = torch.full((need + (1 << 20),), 0x5A, dtype=torch.uint8, device=cuda)
    out = torch.zeros_like(c.dev[0])
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    kv, ks, vs = c.dev[1:]
    tables, qs, lens = c.step
    status = lib.mshift_attend_block_scaled(
        _lib.BF16, c.dev[0].data_ptr(), hq * d, d, rows, hq, paged, kv.data_ptr(),
        kv.data_ptr() + geo.v_offset, ks.data_ptr(), *ks.stride(), vs.data_ptr(), *vs.stride(),
        tables.data_ptr(), tables.stride(0), tables.shape[1], qs.data_ptr(), lens.data_ptr(), len(new),
        bound, most, d**-0.5, 1, 0, out.data_ptr(), hq * d, d, None, 0, work.data_ptr(), need,
        err.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert status == _lib.OK
    assert int(err.item()) == _lib.ERR_LENGTHS
    assert bool((work[need:] == 0x5A).all())


@pytest.mark.gpu
def test_a_graph_captured_for_one_token_and_replayed_with_two(cuda):
    """The bound a graph was captured with is passed by its replay's lengths: flagged, the others right."""
    c = _past(cuda, [1, 1, 1], 8, 2, 128)
    want = c.run(max_query_len=1, max_seq_len=30720)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = _attend(c, max_query_len=1, max_seq_len=30720)
    g.replay()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and take_errors(cuda) == 0
    c.step[1].copy_(_i32(cuda, _cum([2, 1, 1])))  # one of the rows of padding becomes a token
    c.new, c.qs = [2, 1, 1], _cum([2, 1, 1])
    g.replay()
    assert take_errors(cuda) == _lib.ERR_LENGTHS
    _check_rows(c, (out, lse), [0, 2, 3])


@pytest.mark.gpu
@pytest.mark.parametrize("most", [2000, 30720])
@pytest.mark.parametrize("new,bound,hq,hk,d", PAST)
def test_rows_past_the_query_bound_are_zeros_in_a_new_result(cuda, new, bound, hq, hk, d, most):
    take_errors(cuda)
    c = _past(cuda, new, hq, hk, d)
    junk = [torch.full((c.q.shape[0], hq, w), 7.0, dtype=t, device=cuda)
            for w, t in ((d, c.q.dtype), (1, torch.float32))]
    del junk  # what a result's memory may hold before
    out, lse = _attend(c, max_query_len=bound, max_seq_len=most)
    assert take_errors(cuda) == _lib.ERR_LENGTHS
    rows = [q + i for q, n in zip(c.qs, new, strict=False) for i in range(min(n, bound))]
    _check_rows(c, (out, lse), rows)
    rest = [i for i in range(c.q.shape[0]) if i not in set(rows)]
    assert bool((out[rest] == 0).all()) and bool((lse[rest] == -math.inf).all())


# ------------------------------------------------------------------------ NaN
@pytest.mark.gpu
@pytest.mark.parametrize("most", [700, 40000])
@pytest.mark.parametrize("new,d,bs", [(1, 128, 16), (2, 64, 24), (60, 128, 16), (60, 64, 24), (40, 256, 16)])
def test_nan_queries_give_nan_and_no_empty_rows(cuda, new, d, bs, most):
    c = Case(cuda, [700, 90], [new, new], 4, 2, d, bs, seed=3)
    good = c.run(max_seq_len=most)
    for at, head in ((0, 1), (new - 1, 2), (new, 3), (2 * new - 1, 0)):
        was = c.dev[0]
        c.dev[0] = was.clone()
        c.dev[0][at, head, 5] = float("nan")
        out, lse = c.run(max_seq_len=most)
        c.dev[0] = was
        hit = torch.zeros(2 * new, 4, dtype=torch.bool, device=cuda)
        hit[at, head] = True
        assert bool(out[hit].isnan().all()) and bool(lse[hit].isnan().all())
        assert torch.equal(out[~hit], good[0][~hit]) and torch.equal(lse[~hit], good[1][~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("most", [60, 40000])
@pytest.mark.parametrize("new,d", [(1, 128), (60, 128), (60, 64), (7, 256)])
def test_rows_whose_only_keys_are_nan(cuda, new, d, most):
    take_errors(cuda)
    c = Case(cuda, [new, 5], [new, 5], 4, 2, d, 16, seed=4)
    good = c.run(max_seq_len=most)
    c.dev[1] = c.dev[1].clone()
    serving.sides(c.dev[1].view(torch.uint8), "nhd")[0][c.tables[0][0], 0, 1, 7] = NAN_CODE  # the first key, KV head 1
    out, lse = c.run(max_seq_len=most)
    assert bool(out[:new, 2:].isnan().all()) and bool(lse[:new, 2:].isnan().all())
    assert torch.equal(out[:, :2], good[0][:, :2]) and torch.equal(lse[:, :2], good[1][:, :2])
    assert torch.equal(out[new:], good[0][new:])
    c = Case(cuda, [9, 5], [9, 1], 4, 2, d, 16, seed=4)
    c.dev[2] = c.dev[2].clone()
    c.dev[2][c.tables[0][0], 0] = float("nan")
    out, lse = c.run(max_seq_len=most)
    assert bool(out[:9, :2].isnan().all()) and bool(lse[:9, :2].isnan().all())
    assert bool(out[:9, 2:].isfinite().all()) and bool(out[9:].isfinite().all())
    # keys in bad blocks count as unseen, to a row of NaN too
    c.dev[0] = torch.full_like(c.dev[0], float("nan"))
    c.step[0] = torch.full_like(c.step[0], -1)
    out, lse = _attend(c, max_seq_len=most)
    assert take_errors(cuda) == _lib.EBIT_SLOT
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("most", [200, 40000])
@pytest.mark.parametrize("new,d,bs", [(1, 128, 16), (3, 64, 24), (60, 128, 16), (60, 64, 24), (20, 256, 16)])
def test_value_scales_that_are_nan_or_negative(cuda, new, d, bs, most):
    """NaN reaches the rows that see a key of its block and no others; below 2^-64 reads as 2^-64."""
    c = Case(cuda, [200, 90], [new, new], 4, 2, d, bs, seed=8)
    good = c.run(max_seq_len=most)
    col = (200 - new // 2 - 1) // bs
    was = c.dev[3]
    c.dev[3] = was.clone()
    c.dev[3][c.tables[0][col], 1] = float("nan")
    out, lse = c.run(max_seq_len=most)
    row = torch.arange(2 * new, device=cuda)
    hit = (row < new) & (200 - new + row >= col * bs)
    assert bool(hit.any()) and bool(out[hit][:, 2:].isnan().all()) and bool(lse[hit][:, 2:].isnan().all())
    assert torch.equal(out[~hit], good[0][~hit]) and torch.equal(lse[~hit], good[1][~hit])
    assert torch.equal(out[:, :2], good[0][:, :2])
    got = []
    for scale in (-3.0, 0.0, 2.0**-64):
        c.dev[3] = was.clone()
        c.dev[3][c.tables[0][col], 1] = scale
        got.append(c.run(max_seq_len=most))
    for out, lse in got[:2]:
        assert torch.equal(out, got[2][0]) and torch.equal(lse, got[2][1])


@pytest.mark.gpu
@pytest.mark.parametrize("most", [64, 40000])
@pytest.mark.parametrize("new,d", [(1, 128), (40, 128), (40, 64), (4, 256)])
def test_scores_far_below_zero_are_scores(cuda, new, d, most):
    c = Case(cuda, [40], [new], 4, 2, d, 16, seed=5, pow2=True)
    k, v = serving.sides(c.kv.view(torch.uint8), "nhd")
    for p in range(40):  # key p's codes are all alike, larger for later keys
        k[c.tables[0][p // 16], p % 16] = 8 + p
    c.q = torch.full_like(c.q, -(2.0**110))
    c.ks = torch.ones_like(c.ks)
    c.dev = [x.to(cuda) for x in (c.q, c.kv, c.ks, c.vs)]
    out, lse = c.run(max_seq_len=most)
    # the first key's score is 2^100 above the next one's: all the weight
    first = v[c.tables[0][0], 0].view(torch.float8_e4m3fn).double() * c.vs[c.tables[0][0]].double()[:, None]
    want = first.repeat_interleave(2, 0).expand(new, 4, d)
    assert bool(((out.cpu().double() - want).abs() <= 2.0**-8 * want.abs()).all())
    score = -(2.0**110) * d * 2.0**-6 * d**-0.5
    assert bool(((lse.cpu().double() / score - 1).abs() <= 2.0**-20).all())


# ------------------------------------------------------- windows and cut lengths
def _formula(c, at, key_end, window, group):
    """Rows at positions `at` of request 0: keys below key_end, causal, windowed."""
    kc, vc = serving.sides(c.kv, c.layout)
    ids = torch.tensor(c.tables[0][: -(-key_end // c.bs)])
    kk = (kc[ids].double() * c.ks[ids].double()[:, None, :, None]).reshape(-1, c.hk, c.d)
    vv = (vc[ids].double() * c.vs[ids].double()[:, None, :, None]).reshape(-1, c.hk, c.d)
    out = torch.zeros(len(at), c.q.shape[1], c.d, dtype=torch.float64)
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64)
    for i, x in enumerate(at):
        lo, hi = max(x - window + 1, 0), min(x + 1, key_end)
        for h in range(c.q.shape[1]) if lo < hi else ():
            s = kk[lo:hi, h // group] @ c.q[i, h].double() * c.d**-0.5
            lse[i, h] = torch.logsumexp(s, 0)
            out[i, h] = torch.softmax(s, 0) @ vv[lo:hi, h // group]
    return out, lse


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hk,d", [(2, 2, 128), (8, 2, 128), (8, 2, 64), (2, 1, 256)])
@pytest.mark.parametrize("cut", ["bound", "table"])
@pytest.mark.parametrize("long", [0, 5120])
def test_windows_of_requests_cut_at_a_bound(cuda, hq, hk, d, cut, long):
    """Rows behind a cut length whose window still reaches a key see it, the others nothing; with and
    without splits."""
    take_errors(cuda)
    c = Case(cuda, [long + 100], [20], hq, hk, d, 16, seed=6)
    if cut == "bound":
        got, flag, end = _attend(c, max_seq_len=long + 90, window=5), _lib.ERR_LENGTHS, long + 90
    else:
        c.step[0] = c.step[0][:, : (long + 80) // 16]
        got, flag, end = _attend(c, max_seq_len=2 * long + 100, window=5), _lib.ERR_POOL, long + 80
    assert take_errors(cuda) == flag
    want, wlse = _formula(c, range(long + 80, long + 100), end, 5, hq // hk)
    out, lse = (x.cpu().double() for x in got)
    none = wlse == -math.inf
    assert torch.equal(none, lse == -math.inf) and bool((out[none] == 0).all())
    # the tolerances of test_block_scaled.py with what bounds their terms here: |o| <= A <= 448 * 0.023 and
    # sum |q||k| scale < 2^8 * 448 * 0.023 * 5 / 8 < 2^11
    assert bool((torch.where(none, 0.0, lse - wlse).abs() <= 2.0**-9).all())
    assert bool(((out - want).abs() <= 2.0**-8 * want.abs() + (2.0**-11 + 2.0**-20 + 2.0**-9) * 10.4).all())
    assert not bool(none[:4].any()) and bool(none[-4:].all())


# ----------------------------------------------------------------- block maps
@pytest.mark.gpu
def test_dropped_tokens_take_no_blocks(cuda):
    take_errors(cuda)
    c, n, f, h = (_i32(cuda, x) for x in ([0, 0, 3], [20, 20, 40], [1, 2, 3, 4, 5, 6, 7, 8], [1]))
    for tokens, head, lens in ((25, 4, [20, 5, 3]), (20, 3, [20, 0, 3]), (0, 1, [0, 0, 3]), (37, 5, [20, 17, 3]),
                               (45, 5, [20, 20, 8]), (79, 7, [20, 20, 42])):
        t = torch.full((3, 4), -1, dtype=torch.int32, device=cuda)
        t[2, 0] = 99
        got = block_maps(c, n, t, f, h, 16, tokens)
        assert take_errors(cuda) == _lib.ERR_LENGTHS
        assert got.seq_lens.tolist() == lens and got.free_head.tolist() == [head], tokens
        named = [b for row in t.tolist() for b in row if b >= 0 and b != 99]
        assert named == list(range(2, head + 1)), tokens
    # too few free blocks for the lengths, enough for the rows
    t = torch.full((3, 4), -1, dtype=torch.int32, device=cuda)
    got = block_maps(c, n, t, f[:4], h, 16, 25)
    assert take_errors(cuda) == _lib.ERR_LENGTHS and got.free_head.tolist() == [4]


@pytest.mark.gpu
def test_a_free_block_below_zero_is_flagged(cuda):
    take_errors(cuda)
    c, n, f, h = (_i32(cuda, x) for x in ([0], [20], [4, -1], [0]))
    t = torch.full((1, 2), -1, dtype=torch.int32, device=cuda)
    got = block_maps(c, n, t, f, h, 16, 20)
    assert take_errors(cuda) == _lib.EBIT_SLOT
    assert got.slots.tolist() == [64 + i for i in range(16)] + [-1] * 4


@pytest.mark.gpu
def test_lengths_past_32_bits_are_flagged(cuda):
    take_errors(cuda)
    c, n, f, h = (_i32(cuda, x) for x in ([2**31 - 2, 5], [4, 1], [0, 1, 2], [0]))
    t = torch.zeros((2, 2), dtype=torch.int32, device=cuda)
    got = block_maps(c, n, t, f, h, 2**30, 5)
    assert take_errors(cuda) & _lib.ERR_LENGTHS
    assert got.seq_lens.tolist() == [2**31 - 1, 6]


# -------------------------------------------------------------------- rotary
@pytest.mark.gpu
def test_changed_positions_stop_a_rotary_backward(cuda):
    q, k = (torch.randn(6, 2, 64, device=cuda, requires_grad=True) for _ in range(2))
    pos = torch.arange(6, device=cuda).expand(3, 6).clone()
    inv, axes = inv_freq(64, 1e4).to(cuda), axis_map((10, 11, 11), device=cuda)
    op = torch.ops.marathon.rotary_axes
    for changed in (pos, inv, axes):
        a, _ = op(q, k, pos, inv, axes)
        changed.add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            a.sum().backward()
    a, b = op(q, k, pos[0], inv)  # without a table of axes
    (a.sum() + b.sum()).backward()
    want, _ = rotary_axes(torch.ones_like(q), None, pos[0], inv, inverse=True)
    assert torch.equal(q.grad, want)

@pytest.mark.gpu
def test_a_rotary_step_with_its_backward_replays_from_a_graph(cuda):
    q = torch.randn(6, 3, 64, device=cuda, requires_grad=True)
    k = torch.randn(6, 2, 64, device=cuda, requires_grad=True)
    w = torch.randn(6, 3, 64, device=cuda)
    pos = torch.randint(0, 900, (3, 6), device=cuda)
    inv, axes = inv_freq(64, 1e4).to(cuda), axis_map((10, 11, 11), device=cuda)

    def step():
        a, b = torch.ops.marathon.rotary_axes(q, k, pos, inv, axes)
        return a.detach(), b.detach(), *torch.autograd.grad((a * w).sum() + b.square().sum(), (q, k))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in (1, 2):
        torch.manual_seed(seed)
        with torch.no_grad():
            q.normal_()
            k.normal_()
            w.normal_()
        pos.random_(0, 900)
        g.replay()
        for x, y in zip(got, step(), strict=True):
            assert torch.equal(x, y)



def _turns(inv, pos, bits=320):
    """pos * inv / 2 pi modulo one, in integers (pi by Machin's formula)."""
    one = 1 << bits

    def atan(n):
        total, term, k = 0, one // n, 1
        while term:
            total += term // k if k % 4 == 1 else -(term // k)
            term //= n * n
            k += 2
        return total

    pi = 4 * (4 * atan(5) - atan(239))
    num, den = float(inv).as_integer_ratio()
    return (num * pos * one * one // (den * 2 * pi)) % one / one


@pytest.mark.gpu
def test_positions_to_the_ends_of_64_bits(cuda):
    inv = torch.tensor([1.0, 0.1, 1e-3, 1e-6, 3e-9, 1e-20, 2.0**-126, 1e-42, 1e4, -1e-6, 1e18, 0.0], device=cuda)
    pos = [1, 2**31 + 3, 2**40 + 1, -(2**48) - 5, 2**55 + 12345, 2**62 + 1, 2**63 - 1, -(2**63), -1]
    q = torch.zeros(len(pos), 2, 24, device=cuda)
    q[..., :12] = 1  # a pair (1, 0) turns into (cos, sin)
    out, _ = rotary_axes(q, None, torch.tensor(pos, device=cuda), inv, check=True)
    for i, p in enumerate(pos):
        for j, f in enumerate(inv.tolist()):
            a = 2 * math.pi * _turns(f, p)
            for got, want in ((out[i, 0, j], math.cos(a)), (out[i, 0, 12 + j], math.sin(a))):
                # test_rotary_axes.py's tolerance
                assert abs(float(got) - want) <= 2.0**-20, (p, f, float(got), want)


@pytest.mark.gpu
def test_frequencies_that_are_no_numbers(cuda):
    inv = torch.tensor([1.0, math.inf, math.nan, -math.inf, 0.5], device=cuda)
    q = torch.randn(3, 2, 12, device=cuda)
    out, _ = rotary_axes(q, None, torch.tensor([0, 7, -3], device=cuda), inv)
    bad = torch.tensor([False, True, True, True, False], device=cuda)
    assert bool(out[..., :5][..., bad].isnan().all()) and bool(out[..., 5:10][..., bad].isnan().all())
    assert bool(out[..., :5][..., ~bad].isfinite().all()) and torch.equal(out[..., 10:], q[..., 10:])


# ------------------------------------------------- offsets that the rows do not hold
@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1, 3, 2], [40, 3, 50]])
def test_offsets_past_the_rows_are_flagged_and_rows_keep_their_places(cuda, new):
    take_errors(cuda)
    c = Case(cuda, [300, 200, 400], new, 4, 2, 128, 16, seed=7)
    keep = sum(new) - 1
    for most in (400, 40000):
        whole, c.dev[0] = c.dev[0], c.dev[0][:keep]
        got = _attend(c, max_seq_len=most)
        c.dev[0] = whole
        assert take_errors(cuda) == _lib.ERR_LENGTHS
        _check_rows(c, got, list(range(keep)))
    for qs in ([0, 2, 1, 3], [-1, 0, 0, 1]):
        c.step[1] = _i32(cuda, qs)
        _attend(c)
        assert take_errors(cuda) == _lib.ERR_LENGTHS, qs


@pytest.mark.gpu
def test_append_with_offsets_past_the_rows(cuda):
    take_errors(cuda)
    c = Case(cuda, [40, 37], [9, 12], 2, 2, 64, 16, seed=2, pow2=True)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(21, 2, 64, generator=g).half().to(cuda) for _ in range(2))
    kv, ks, vs = (x.clone() for x in c.dev[1:])
    append_block_scaled(k[:18], v[:18], kv, ks, vs, *c.step, 16)
    assert take_errors(cuda) == _lib.ERR_LENGTHS
    want = [x.clone() for x in c.dev[1:]]  # the second request's last three rows are not there
    lens, qs = _i32(cuda, [40, 34]), _i32(cuda, [0, 9, 18])
    append_block_scaled(k[:18], v[:18], *want, c.step[0], qs, lens, 16, check=True)
    for a, b in zip((kv, ks, vs), want, strict=True):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for qs in ([0, 9, 4], [-2, 9, 21]):
        append_block_scaled(k, v, kv, ks, vs, c.step[0], _i32(cuda, qs), c.step[2], 16)
        assert take_errors(cuda) == _lib.ERR_LENGTHS


@pytest.mark.gpu
@pytest.mark.parametrize("most", [200, 40000])
def test_offsets_and_lengths_at_the_ends_of_int32(cuda, most):
    """Nothing is read or written outside the rows, whatever the arrays hold."""
    low, high = -(2**31), 2**31 - 1
    c = Case(cuda, [120, 90, 200], [3, 2, 40], 4, 2, 128, 16, seed=9)
    good = c.run(max_seq_len=most)
    n = c.q.shape[0]
    kv, ks, vs = c.dev[1:]
    k = torch.randn(n, 2, 128, device=cuda).half()
    wide = torch.full((n + 200, 4, 128), 7.0, dtype=c.q.dtype, device=cuda)
    for qs in ([0, 3, low, high], [low, 3, 5, high], [0, 3, 5, low], [high, high, low, low], [0, 3, high, 5],
               [low, low, low, low], [0, 3, 5, -1], [0, 3, 5, high]):
        for lens in ([120, 90, 200], [120, low, high], [high, high, low]):
            take_errors(cuda)
            step = [c.step[0], _i32(cuda, qs), _i32(cuda, lens)]
            out, lse = attend_block_scaled(*c.dev, *step, 16, return_lse=True, max_query_len=40, max_seq_len=most,
                                           out=wide[100: 100 + n])
            assert take_errors(cuda) & _lib.ERR_LENGTHS
            assert bool((wide[:100] == 7).all()) and bool((wide[100 + n:] == 7).all())
            if qs == [0, 3, 5, high] and lens[0] == 120:  # in order, only past the rows
                assert torch.equal(out[:3], good[0][:3]) and torch.equal(lse[:3], good[1][:3])
            cache = [x.clone() for x in (kv, ks, vs)]
            append_block_scaled(k, k, *cache, *step, 16)
            assert take_errors(cuda) & _lib.ERR_LENGTHS
            free = [b for b in range(ks.shape[0]) if all(b not in t for t in c.tables)]
            assert torch.equal(cache[0].view(torch.uint8)[free], kv.view(torch.uint8)[free])
            wide.fill_(7.0)


# ------------------------------------------------------ gradients that would be lost
def _dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.gpu
def test_forward_mode_is_refused(cuda):
    c = Case(cuda, [40], [2], 4, 2, 128, 16)
    q, kv, ks, vs = c.dev
    k = torch.zeros(2, 2, 128, dtype=torch.bfloat16, device=cuda)
    pos, inv = torch.arange(2, device=cuda), inv_freq(128, 1e4).to(cuda)
    with forward_ad.dual_level():
        for call in (lambda: rotary_axes(_dual(q), None, pos, inv),
                     lambda: rotary_axes(None, _dual(q), pos, inv),
                     lambda: rotary_axes(q, None, pos, _dual(inv)),
                     lambda: torch.ops.marathon.rotary_axes(_dual(q), k, pos, inv),
                     lambda: append_block_scaled(_dual(k), k, kv, ks, vs, *c.step, 16),
                     lambda: append_block_scaled(k, _dual(k), kv, ks, vs, *c.step, 16),
                     lambda: attend_block_scaled(_dual(q), kv, ks, vs, *c.step, 16, **c.bounds),
                     lambda: attend_block_scaled(q, kv, _dual(ks), vs, *c.step, 16, **c.bounds)):
            with pytest.raises(ShiftError, match="gradient"):
                call()
        rotary_axes(q, None, pos, inv)  # nothing to lose
    for f in (lambda x: torch.ops.marathon.rotary_axes(x, k, pos, inv)[0],
              lambda x: torch.ops.marathon.attend_block_scaled(x, kv, ks, vs, *c.step, 16, "nhd", 2, 40)[0]):
        with pytest.raises(ShiftError, match="gradient"):
            torch.func.jvp(f, (q,), (q,))


def _leaf(t):
    return t.clone().requires_grad_()


@pytest.mark.gpu
def test_gradients_of_frequencies_and_scales_are_refused(cuda):
    c = Case(cuda, [40], [2], 4, 2, 128, 16)
    q, kv, ks, vs = c.dev
    k = torch.zeros(2, 2, 128, dtype=torch.bfloat16, device=cuda)
    pos, inv = torch.arange(2, device=cuda), inv_freq(128, 1e4).to(cuda)
    for call in (lambda: rotary_axes(q, None, pos, _leaf(inv)),
                 lambda: torch.ops.marathon.rotary_axes(q, k, pos, _leaf(inv)),
                 lambda: append_block_scaled(k, k, kv, _leaf(ks), vs, *c.step, 16),
                 lambda: attend_block_scaled(q, kv, ks, _leaf(vs), *c.step, 16, **c.bounds)):
        with pytest.raises(ShiftError, match="gradient"):
            call()
        with torch.no_grad():
            call()


# ------------------------------------------------------------ results in one another
@pytest.mark.gpu
def test_results_that_overlap_themselves_are_refused(cuda):
    c = Case(cuda, [40], [3], 4, 2, 128, 16)
    q, kv, ks, vs = c.dev
    buf = torch.zeros(1 << 16, dtype=q.dtype, device=cuda)
    pos, inv = torch.arange(3, device=cuda), inv_freq(128, 1e4).to(cuda)
    for strides in ((512, 64, 1), (128, 128, 1), (384, 128, 1), (64, 1024, 1)):
        o = buf.as_strided((3, 4, 128), strides)
        with pytest.raises(ShiftError, match="overlap|repeat"):
            attend_block_scaled(q, kv, ks, vs, *c.step, 16, out=o, **c.bounds)
        with pytest.raises(ShiftError, match="overlap|repeat"):
            rotary_axes(o, None, pos, inv, inplace=True)
    k = torch.zeros(3, 2, 128, dtype=q.dtype, device=cuda)
    scales = torch.ones(4096, device=cuda)
    for strides in ((1, 1), (2, 2), (0, 1)):
        with pytest.raises(ShiftError, match="overlap|repeat"):
            append_block_scaled(k, k, kv, scales.as_strided(ks.shape, strides), vs, *c.step, 16)
    n = ks.numel()
    with pytest.raises(ShiftError, match="two tensors"):
        append_block_scaled(k, k, kv, scales[:n].view_as(ks), scales[2: n + 2].view_as(ks), *c.step, 16)
    append_block_scaled(k, k, kv, scales[:n].view_as(ks), scales[n: 2 * n].view_as(ks), *c.step, 16)
    b8 = torch.zeros(1 << 20, dtype=torch.uint8, device=cuda)
    for strides in ((512, 512, 256, 1), (8192, 512, 128, 1), (4096, 512, 256, 1)):
        with pytest.raises(ShiftError, match="overlap"):
            append_block_scaled(k, k, b8.as_strided(kv.shape, strides), ks, vs, *c.step, 16)
    for strides in ((512, 128, 1), (128, 512, 1), (4096, 256, 1)):
        attend_block_scaled(q, kv, ks, vs, *c.step, 16, out=buf.as_strided((3, 4, 128), strides), **c.bounds)


@pytest.mark.gpu
def test_scales_past_fp32_are_refused(cuda):
    c = Case(cuda, [40], [2], 4, 2, 128, 16)
    for scale in (1e39, -1e300, 3.4e38):
        with pytest.raises(ShiftError, match="scale"):
            c.run(scale=scale)


@pytest.mark.gpu
def test_strides_of_single_rows_and_heads_say_nothing(cuda):
    """One token out of rows of an odd width, one head of an odd stride: 16-byte boundaries all the same."""
    c = Case(cuda, [40], [1], 4, 1, 128, 16)
    q, kv, ks, vs = c.dev
    want = c.run()
    odd = torch.zeros(1024, dtype=q.dtype, device=cuda)
    for shape, strides in (((1, 4, 128), (4 * 128 + 3, 128, 1)), ((1, 4, 128), (7, 128, 1))):
        c.dev[0] = odd.as_strided(shape, strides).copy_(q)
        got = c.run(out=torch.zeros(1024, dtype=q.dtype, device=cuda).as_strided(shape, strides))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    pos, inv = torch.tensor([7], device=cuda), inv_freq(128, 1e4).to(cuda)
    assert torch.equal(rotary_axes(c.dev[0], None, pos, inv)[0], rotary_axes(q, None, pos, inv)[0])
    k = torch.randn(1, 1, 128, device=cuda).to(q.dtype)
    caches = []
    for strides in ((128, 128, 1), (5, 3, 1)):
        cache = [x.clone() for x in (kv, ks, vs)]
        x = odd.as_strided((1, 1, 128), strides).copy_(k)
        append_block_scaled(x, x, *cache, *c.step, 16, check=True)
        caches.append(cache)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*caches, strict=True))


# --------------------------------------------------------------- beside the shift path
@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_a_session_loaded_by_the_shift_path_is_attended(cuda, layout):
    """Stored rows re-rotated into a paged e4m3 cache with one scale a layer, and a decode step and a chunk over
    it: the layer's scale is every block's and head's, by strides of zero."""
    c = Case(cuda, [150, 70], [1, 60], 4, 2, 128, 16, layout=layout, seed=11)
    c.kv.view(torch.uint8).fill_(NAN_CODE)
    kv = c.kv.to(cuda)
    g = torch.Generator().manual_seed(2)
    rows = (torch.randn(220, 2, 256, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).to(cuda)
    cached = _i32(cuda, [0, 0])
    m = block_maps(cached, _i32(cuda, c.lens), c.step[0].clone(),
                   _i32(cuda, [b for t in c.tables for b in t if b >= 0]), _i32(cuda, [0]), 16, 220, check=True)
    shift = rope_shift(37, 128, inv_freq(128, 1e6), cuda)
    scatter_shifted(rows, kv, m.slots, 16, layout == "hnd", shift, fp8=True, check=True)
    k, v = (x.cpu().double() for x in serving.sides(kv, layout))
    stored = rows[:150].cpu().double()
    place = [(c.tables[0][p // 16], p % 16) for p in range(150)]
    turned = serving.rotary(stored[..., :128], torch.full((1, 150), 37), inv_freq(128, 1e6),
                            torch.zeros(64, dtype=torch.int32), False)
    for p, (b, o) in enumerate(place):  # the values as they were, the keys turned (within a step of e4m3)
        assert torch.equal(v[b, o], stored[p, :, 128:])
        assert bool(((k[b, o] - turned[p].clamp(-448, 448)).abs() <= 2.0**-4 * turned[p].abs() + 2.0**-9).all())
    ks, vs = torch.tensor(0.021), torch.tensor(0.013)
    blocks = c.kv.shape[0]
    c.kv, c.ks, c.vs = kv.cpu(), ks.expand(blocks, 2), vs.expand(blocks, 2)
    c.dev[1:] = [kv, ks.to(cuda).expand(blocks, 2), vs.to(cuda).expand(blocks, 2)]
    c.check(c.run())
    c.check(c.run(max_seq_len=20000))
