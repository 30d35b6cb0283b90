"""Block tables and slot maps from request lengths on the GPU, against a plain loop."""

from __future__ import annotations

import random

import pytest
import torch

from marathon_b200 import _lib
from marathon_b200.block_maps import block_maps
from marathon_b200.shift_kernels import ShiftError, take_errors
from serving import block_maps as plain


def _case(reqs, hi_cached, hi_new, bs, seed, lo_new=0):
    r = random.Random(seed)
    cached = [r.randint(0, hi_cached) for _ in range(reqs)]
    new = [r.randint(lo_new, hi_new) for _ in range(reqs)]
    width = max([-(-(c + n) // bs) for c, n in zip(cached, new, strict=True)] + [0]) + 2
    held = sum(-(-c // bs) for c in cached)
    need = sum(-(-(c + n) // bs) for c, n in zip(cached, new, strict=True))
    ids = list(range(need + 7))
    r.shuffle(ids)
    it = iter(ids)
    tables = [[next(it) if b < -(-c // bs) else -1 for b in range(width)] for c in cached]
    return cached, new, tables, ids[held:], width


def _dev(cuda, *lists):
    return [torch.tensor(x, dtype=torch.int32, device=cuda) for x in lists]


def _same(got, tables, want):
    qs, seq, slots, pos, head, tab = want
    assert got.query_start.tolist() == qs
    assert got.seq_lens.tolist() == seq
    assert got.slots.tolist() == slots
    assert got.positions.tolist() == pos
    assert got.free_head.tolist() == [head]
    assert tables.tolist() == tab


def test_refuses_cpu_tensors_and_bad_arguments():
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ShiftError, match="CUDA"):
        block_maps(i(1), i(1), i(0)[None], i(1), i(0), 16, 1)
    lib = _lib.load()
    ok = dict(reqs=1, stride=4, width=4, free=1, bs=16, tokens=1, head=64, head_out=128)

    def call(**kw):
        a = {**ok, **kw}
        return lib.mshift_block_maps(16, 16, a["reqs"], 16, a["stride"], a["width"], 16, a["free"],
                                     a["head"], a["bs"], a["tokens"], 16, 16, 16, 16, a["head_out"],
                                     16, None)

    for bad in (dict(reqs=-1), dict(stride=3), dict(width=-1), dict(free=-1), dict(bs=0),
                dict(tokens=-1), dict(head=None), dict(head_out=None), dict(head_out=64)):
        assert call(**bad) == _lib.EINVAL, bad


@pytest.mark.gpu
@pytest.mark.parametrize("reqs,hi_cached,hi_new,bs,pad", [
    (1, 0, 1, 16, 0), (1, 40, 1, 16, 3), (3, 100, 40, 16, 1), (64, 3000, 1, 16, 0),
    (65, 300, 65, 24, 500), (1023, 50, 3, 1, 2), (1025, 200, 9, 16, 0), (2500, 40, 2, 8, 1),
    (2, 10, 5000, 128, 77),
])
def test_matches_the_plain_loop(cuda, reqs, hi_cached, hi_new, bs, pad):
    cached, new, tables, free, _ = _case(reqs, hi_cached, hi_new, bs, seed=reqs + bs)
    tokens = sum(new) + pad
    c, n, t, f, h = _dev(cuda, cached, new, tables, free, [0])
    got = block_maps(c, n, t, f, h, bs, tokens, check=True)
    _same(got, t, plain(cached, new, tables, free, 0, bs, tokens))


@pytest.mark.gpu
def test_steps_chain_through_the_free_head_and_strided_tables(cuda):
    cached, new, tables, free, width = _case(9, 70, 20, 16, seed=5, lo_new=1)
    free = free + list(range(10_000, 10_100))
    c, n, f, head = _dev(cuda, cached, new, free, [0])
    whole = torch.full((9, width + 40), -7, dtype=torch.int32, device=cuda)
    t = whole[:, : width + 30]
    t.fill_(-1)
    t[:, :width] = torch.tensor(tables, dtype=torch.int32, device=cuda)
    rows = [r + [-1] * 30 for r in tables]
    at = 0
    for step in range(4):
        got = block_maps(c, n, t, f, head, 16, sum(new) + step, check=True)
        want = plain(cached, new, rows, free, at, 16, sum(new) + step)
        _same(got, t, want)
        c, head, cached, at, rows = got.seq_lens, got.free_head, want[1], want[4], want[5]
    assert bool((whole[:, width + 30:] == -7).all())


@pytest.mark.gpu
def test_no_requests_and_no_tokens(cuda):
    e = torch.empty(0, dtype=torch.int32, device=cuda)
    h = torch.tensor([3], dtype=torch.int32, device=cuda)
    got = block_maps(e, e, e.reshape(0, 4), torch.arange(9, dtype=torch.int32, device=cuda), h, 16, 5,
                     check=True)
    assert got.query_start.tolist() == [0] and got.slots.tolist() == [-1] * 5
    assert got.free_head.tolist() == [3]
    got = block_maps(h, h * 0, torch.zeros(1, 2, dtype=torch.int32, device=cuda), e, h * 0, 16, 0,
                     check=True)
    assert got.query_start.tolist() == [0, 0] and got.seq_lens.tolist() == [3]


@pytest.mark.gpu
def test_bad_lengths_pools_and_tables_are_flagged(cuda):
    take_errors(cuda)
    t = torch.full((2, 2), -1, dtype=torch.int32, device=cuda)
    c, n, f, h = _dev(cuda, [0, 0], [20, 20], [5, 6, 7], [0])
    got = block_maps(c, n, t, f, h, 16, 40)  # four blocks wanted, three there
    assert take_errors(cuda) == _lib.ERR_POOL
    assert t.tolist() == [[5, 6], [7, -1]]
    assert got.slots.tolist()[36:] == [-1] * 4 and got.slots.tolist()[35] == 7 * 16 + 15
    assert got.free_head.tolist() == [3]
    t.fill_(-1)
    n2, f2 = _dev(cuda, [40, 1], list(range(8)))  # three blocks in a table of two
    got = block_maps(c, n2, t, f2, h, 16, 41)
    assert take_errors(cuda) == _lib.ERR_POOL
    assert got.slots.tolist()[32:40] == [-1] * 8 and got.slots.tolist()[40] == 3 * 16
    t.fill_(-1)
    got = block_maps(c, n, t, _dev(cuda, [1, 2, 3, 4])[0], h, 16, 25)  # fewer rows than new tokens
    assert take_errors(cuda) == _lib.ERR_LENGTHS
    assert got.query_start.tolist() == [0, 20, 25] and got.seq_lens.tolist() == [20, 5]
    bad = _dev(cuda, [-3, 4])[0]
    t.fill_(2)
    got = block_maps(bad, n * 0 + 1, t, f, h, 16, 2)
    assert take_errors(cuda) == _lib.ERR_LENGTHS
    assert got.seq_lens.tolist() == [1, 5]
    t.fill_(-1)
    got = block_maps(n, n * 0 + 1, t, f, h, 16, 2)  # held blocks that the table does not name
    assert take_errors(cuda) == _lib.EBIT_SLOT
    assert got.slots.tolist() == [-1, -1]
    with pytest.raises(ShiftError, match="free blocks"):
        block_maps(c, n, t, f, h + 2, 16, 40, check=True)
    assert take_errors(cuda) == 0


@pytest.mark.gpu
def test_captured_step_replays_with_new_lengths(cuda):
    cached, new, tables, free, width = _case(33, 200, 30, 16, seed=8)
    c, n, t, f, h = _dev(cuda, cached, new, tables, free, [0])
    block_maps(c, n, t.clone(), f, h, 16, 1200)  # the status word exists before the capture
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = block_maps(c, n, t, f, h, 16, 1200)
    for seed in (21, 22):
        r = random.Random(seed)
        new = [r.randint(0, x) for x in new]
        n.copy_(torch.tensor(new, dtype=torch.int32))
        t.copy_(torch.tensor(tables, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        _same(got, t, plain(cached, new, tables, free, 0, 16, 1200))


@pytest.mark.gpu
def test_refusals(cuda):
    c, n, t, f, h = _dev(cuda, [1, 1], [1, 1], [[0], [1]], [2], [0])
    with pytest.raises(ShiftError, match="int32"):
        block_maps(c.long(), n, t, f, h, 16, 2)
    with pytest.raises(ShiftError, match="entries"):
        block_maps(c, n[:1], t, f, h, 16, 2)
    with pytest.raises(ShiftError, match="block tables for"):
        block_maps(c, n, t[:1], f, h, 16, 2)
    with pytest.raises(ShiftError, match="positive"):
        block_maps(c, n, t, f, h, 0, 2)
    with pytest.raises(ShiftError, match="overlap"):
        block_maps(c, n, c.new_zeros(4).as_strided((2, 2), (1, 1)), f, h, 16, 2)
    with pytest.raises(ShiftError, match="shares memory"):
        block_maps(c, n, t, t[1], h, 16, 2)
    with pytest.raises(ShiftError, match="CUDA"):
        block_maps(c, n, t, f, h.cpu(), 16, 2)
