"""The serving operators in a run, as a step uses them, and their operator-registry face.

A prefill, chunked continuations and decode steps of ragged requests go through block maps,
rotary, append and attention; every step's answers are compared with 64-bit attention
over the 64-bit cache that the same steps build.
"""

from __future__ import annotations

import pytest
import torch

import marathon_b200  # noqa: F401  (registers the operators)
import serving
from marathon_b200.block_maps import block_maps
from marathon_b200.block_scaled import append_block_scaled, attend_block_scaled
from marathon_b200.rotary import axis_map, rotary_axes
from marathon_b200.shift_kernels import ShiftError, inv_freq

HQ, HK, D, BS = 8, 2, 128, 16


def test_operators_are_registered_and_refuse_cpu_tensors():
    ops = torch.ops.marathon
    assert "Tensor(a2!) block_tables" in str(ops.block_maps.default._schema)
    for name in ("kv", "k_scale", "v_scale"):
        assert f"!) {name}" in str(ops.append_block_scaled.default._schema)
    i = torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 64)
    with pytest.raises(ShiftError, match="CUDA"):
        ops.block_maps(i, i, i[None], i, i, 16, 1)
    with pytest.raises(ShiftError, match="CUDA"):
        ops.rotary_axes(q, q, torch.zeros(1, dtype=torch.long), inv_freq(64, 1e4))
    kv = torch.zeros(2, 16, 2, 128, dtype=torch.uint8)
    s = torch.ones(2, 2)
    with pytest.raises(ShiftError, match="CUDA"):
        ops.append_block_scaled(q, q, kv, s, s, i[None], torch.zeros(2, dtype=torch.int32), i, 16, "nhd")
    with pytest.raises(ShiftError, match="CUDA"):
        ops.attend_block_scaled(q.half(), kv, s, s, i[None], torch.zeros(2, dtype=torch.int32), i, 16,
                                "nhd", 1, 1)


class _Pool:
    def __init__(self, cuda, layout, blocks=120, reqs=3, width=30):
        self.layout = layout
        shape = serving.cache_shape(layout, blocks, BS, HK, D)
        self.kv = torch.full(shape, 0x7F, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
        self.ks = torch.full((blocks, HK), float("nan"), device=cuda)
        self.vs = self.ks.clone()
        self.tables = torch.full((reqs, width), -1, dtype=torch.int32, device=cuda)
        self.free = torch.randperm(blocks, device=cuda).int()
        self.head = torch.zeros(1, dtype=torch.int32, device=cuda)
        self.lens = torch.zeros(reqs, dtype=torch.int32, device=cuda)
        self.ref = [t.double().cpu() for t in (self.kv, self.ks, self.vs)]


def _inputs(n, cuda, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(n, HQ, D, generator=g).bfloat16().to(cuda)
    k = (torch.randn(n, HK, D, generator=g) * 2).bfloat16().to(cuda)
    v = torch.randn(n, HK, D, generator=g).bfloat16().to(cuda)
    return q, k, v


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["nhd", "split"])
def test_prefill_chunks_and_decode_steps(cuda, layout):
    p = _Pool(cuda, layout)
    inv, axes = inv_freq(D, 1e6).to(cuda), axis_map((16, 24, 24), device=cuda)
    steps = [([37, 200, 0], 3), ([60, 1, 16], 0), ([1, 130, 1], 5), ([1, 1, 1], 0), ([1, 0, 1], 1)]
    for at, (new, pad) in enumerate(steps):
        n = sum(new) + pad
        q, k, v = _inputs(n, cuda, at)
        m = block_maps(p.lens, torch.tensor(new, dtype=torch.int32, device=cuda), p.tables, p.free,
                       p.head, BS, n, check=True)
        pos = torch.stack((m.positions, m.positions // 3, m.positions % 7))
        q, k = rotary_axes(q, k, pos, inv, axes, inplace=True, check=True)
        append_block_scaled(k, v, p.kv, p.ks, p.vs, p.tables, m.query_start, m.seq_lens, BS, layout,
                            check=True)
        out, lse = attend_block_scaled(q, p.kv, p.ks, p.vs, p.tables, m.query_start, m.seq_lens, BS,
                                       layout, max_query_len=max(new), max_seq_len=480,
                                       return_lse=True, check=True)
        p.lens, p.head = m.seq_lens, m.free_head
        qs, lens, tables = m.query_start.tolist(), m.seq_lens.tolist(), p.tables.tolist()
        serving.append(k.cpu(), v.cpu(), *p.ref, tables, qs, lens, BS, layout)
        for got, want in zip((p.kv, p.ks, p.vs), p.ref, strict=True):
            torch.testing.assert_close(got.double().cpu(), want, rtol=0, atol=0, equal_nan=True)
        want, wlse, mag, big = serving.attend(q.cpu(), *p.ref, tables, qs, lens, BS, layout, D**-0.5)
        # the tolerances of test_block_scaled.py
        d = 2.0**-20 * big
        tol = 2.0**-8 * want.abs() + (2.0**-11 + 2.0**-20 + d[..., None]) * mag
        assert bool(((out.double().cpu() - want).abs() <= tol).all()), at
        live = slice(0, sum(new))
        assert bool(((lse.double().cpu() - wlse)[live].abs()
                     <= (d + 2.0**-20 + 2.0**-22 * wlse.abs())[live]).all()), at
        assert bool((out[sum(new):] == 0).all())
        assert m.slots[sum(new):].tolist() == [-1] * pad


@pytest.mark.gpu
def test_a_decode_step_replays_from_a_graph(cuda):
    """Lengths, tables and the free head stay on the GPU and move on inside the graph."""
    eager, graph = _Pool(cuda, "nhd"), _Pool(cuda, "nhd")
    graph.free.copy_(eager.free)
    inv = inv_freq(D, 1e6).to(cuda)
    one = torch.ones(3, dtype=torch.int32, device=cuda)
    q, k, v = _inputs(3, cuda, 0)

    def step(p):
        m = block_maps(p.lens, one, p.tables, p.free, p.head, BS, 3)
        qr, kr = rotary_axes(q, k, m.positions, inv)
        append_block_scaled(kr, v, p.kv, p.ks, p.vs, p.tables, m.query_start, m.seq_lens, BS, "nhd")
        out = attend_block_scaled(qr, p.kv, p.ks, p.vs, p.tables, m.query_start, m.seq_lens, BS, "nhd",
                                  max_query_len=1, max_seq_len=480)
        p.lens.copy_(m.seq_lens)
        p.head.copy_(m.free_head)
        return out

    step(_Pool(cuda, "nhd"))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(graph)
    for at in range(40):
        for x, y in zip((q, k, v), _inputs(3, cuda, at), strict=True):
            x.copy_(y)
        want = step(eager)
        g.replay()
        assert torch.equal(out, want), at
    assert eager.lens.tolist() == graph.lens.tolist() == [40, 40, 40]
    assert eager.head.tolist() == graph.head.tolist() == [9]


@pytest.mark.gpu
def test_operators_match_the_functions_and_trace(cuda):
    p, o = _Pool(cuda, "nhd"), _Pool(cuda, "nhd")
    o.free.copy_(p.free)
    new = torch.tensor([20, 1, 40], dtype=torch.int32, device=cuda)
    q, k, v = _inputs(61, cuda, 1)
    inv, axes = inv_freq(D, 1e6).to(cuda), axis_map((16, 24, 24), device=cuda)
    pos = torch.randint(0, 500, (3, 61), device=cuda)
    ops = torch.ops.marathon

    def by_ops(x):
        qs, lens, slots, _, head = ops.block_maps(x.lens, new, x.tables, x.free, x.head, BS, 61)
        qr, kr = ops.rotary_axes(q, k, pos, inv, axes)
        ops.append_block_scaled(kr, v, x.kv, x.ks, x.vs, x.tables, qs, lens, BS, "nhd")
        out, lse = ops.attend_block_scaled(qr, x.kv, x.ks, x.vs, x.tables, qs, lens, BS, "nhd", 40, 480)
        return out, lse, slots, head

    m = block_maps(p.lens, new, p.tables, p.free, p.head, BS, 61)
    qr, kr = rotary_axes(q, k, pos, inv, axes)
    append_block_scaled(kr, v, p.kv, p.ks, p.vs, p.tables, m.query_start, m.seq_lens, BS, "nhd")
    out, lse = attend_block_scaled(qr, p.kv, p.ks, p.vs, p.tables, m.query_start, m.seq_lens, BS, "nhd",
                                   max_query_len=40, max_seq_len=480, return_lse=True)
    want = (out, lse, m.slots, m.free_head)
    for got in (by_ops(o), torch.compile(by_ops, backend="eager", fullgraph=True)(o)):
        for x, y in zip(got, want, strict=True):
            assert torch.equal(x, y)
    assert torch.equal(o.kv.view(torch.uint8), p.kv.view(torch.uint8))


@pytest.mark.gpu
def test_rotary_operator_gradients(cuda):
    """Against torch's own gradient of the formula, with shared heads and a broadcast input."""
    inv, axes = inv_freq(64, 1e4).to(cuda), axis_map((10, 11, 11), device=cuda)
    pos = torch.randint(0, 900, (3, 6), device=cuda)
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 1, 64, generator=g).to(cuda).requires_grad_()
    k = torch.randn(6, 2, 64, generator=g).to(cuda).requires_grad_()
    w = torch.randn(6, 3, 64, generator=g).to(cuda)
    a, b = torch.ops.marathon.rotary_axes(x.expand(6, 3, 64), k, pos, inv, axes)
    ((a * w).sum() + b.sum()).backward()
    ang = pos.double()[axes.long()].T * inv.double()
    c, s = ang.cos()[:, None], ang.sin()[:, None]

    def plain(t):
        p, r = t[..., :32], t[..., 32:]
        return torch.cat((p * c - r * s, r * c + p * s), -1)

    x2, k2 = (t.detach().double().requires_grad_() for t in (x, k))
    ((plain(x2.expand(6, 3, 64)) * w.double()).sum() + plain(k2).sum()).backward()
    # 2^-20 of a pair's magnitudes an element (test_rotary_axes.py), summed over three heads
    for got, want, most in ((x.grad, x2.grad, 2 * w.abs().sum(1).max()), (k.grad, k2.grad, 2.0)):
        assert float((got.double() - want).abs().max()) <= 2.0**-20 * float(most) + 2.0**-22 * float(most)
    # one output unused: the rotation keeps lengths, so the gradient of |y|^2 is 2 x
    q2 = torch.randn(6, 3, 64, device=cuda, requires_grad=True)
    torch.ops.marathon.rotary_axes(q2, k, pos, inv, axes)[0].square().sum().backward()
    torch.testing.assert_close(q2.grad, 2 * q2.detach(), rtol=0, atol=2.0**-17)
    with pytest.raises(ShiftError, match="gradient"):
        rotary_axes(q2, k, pos, inv, axes)
