"""Plain 64-bit forms of the serving operators, on the CPU (a test helper)."""

from __future__ import annotations

import math

import torch

FMAX = 448.0
F8 = torch.float8_e4m3fn


def sides(kv: torch.Tensor, layout: str):
    """K and V of a paged cache as views [blocks, block_size, heads, head_size]."""
    if layout == "split":
        return kv[0], kv[1]
    if layout == "split_blocks":
        return kv[:, 0], kv[:, 1]
    if layout == "hnd":
        kv = kv.transpose(1, 2)
    d = kv.shape[-1] // 2
    return kv[..., :d], kv[..., d:]


def cache_shape(layout: str, blocks: int, bs: int, heads: int, d: int):
    return {"nhd": (blocks, bs, heads, 2 * d), "hnd": (blocks, heads, bs, 2 * d),
            "split": (2, blocks, bs, heads, d), "split_blocks": (blocks, 2, bs, heads, d)}[layout]


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value of an fp64 tensor, ties to even, saturated; NaN stays."""
    a = x.abs().clamp(max=FMAX)
    e = torch.floor(torch.log2(a.clamp(min=2.0**-6)))
    step = torch.exp2(e - 3)
    return torch.copysign((a / step).round() * step, x)


def block_maps(cached, new, tables, free, head, bs, tokens):
    """Loops over requests; python lists and a [requests, width] list of lists."""
    tables = [list(t) for t in tables]
    qs, seq, slots, pos = [0], [], [], []
    for r, (c, n) in enumerate(zip(cached, new, strict=True)):
        for b in range(-(-c // bs), -(-(c + n) // bs)):
            tables[r][b] = free[head]
            head += 1
        for p in range(c, c + n):
            slots.append(tables[r][p // bs] * bs + p % bs)
            pos.append(p)
        qs.append(qs[-1] + n)
        seq.append(c + n)
    pad = tokens - len(slots)
    return qs, seq, slots + [-1] * pad, pos + [0] * pad, head, tables


def rotary(x, positions, inv_freq, axes, inverse):
    """fp64; x [n, heads, d], positions [axes, n]."""
    half = inv_freq.numel()
    angle = positions.double()[axes.long()].T * inv_freq.double()
    c, s = angle.cos()[:, None], angle.sin()[:, None] * (-1 if inverse else 1)
    y = x.double().clone()
    a, b = x.double()[..., :half], x.double()[..., half:2 * half]
    y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    return y


def append(k, v, kv, ks, vs, tables, qs, lens, bs, layout):
    """In place on fp64 copies: kv holds code values, ks/vs scales."""
    for x, cache, scale in ((k, sides(kv, layout)[0], ks), (v, sides(kv, layout)[1], vs)):
        x = x.double()
        for r in range(len(lens)):
            n, seq = qs[r + 1] - qs[r], lens[r]
            start = seq - n
            for col in range(start // bs, -(-seq // bs) if n else 0):
                lo, hi = max(start, col * bs), min(seq, (col + 1) * bs)
                b = tables[r][col]
                rows = x[qs[r] + lo - start: qs[r] + hi - start]
                for h in range(x.shape[1]):
                    y = rows[:, h]
                    finite = y[y.isfinite()].abs()
                    top = float(finite.max()) if finite.numel() else 0.0
                    want = 2.0**-64
                    if top > 0:
                        m, e = math.frexp(top)
                        want = max(want, 2.0 ** (e - 9 if m <= 0.875 else e - 8))
                    old = float(scale[b, h])
                    if lo > col * bs:
                        want = max(want, old)
                        if want != old:
                            kept = cache[b, : lo - col * bs, h]
                            cache[b, : lo - col * bs, h] = e4m3(kept * (old / want))
                    scale[b, h] = want
                    cache[b, lo - col * bs: hi - col * bs, h] = e4m3(y / want)


def attend(q, kv, ks, vs, tables, qs, lens, bs, layout, scale, causal=True, window=0):
    """(out, lse, mean |v| under the weights, largest sum |q||k| scale) in fp64, loops over
    requests and heads.  Rows of no request are zeros and -inf."""
    n, hq, d = q.shape
    kc, vc = sides(kv, layout)
    hk = kc.shape[2]
    out = torch.zeros(n, hq, d, dtype=torch.float64)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    mag = torch.zeros(n, hq, d, dtype=torch.float64)
    big = torch.zeros(n, hq, dtype=torch.float64)
    for r in range(len(lens)):
        m, seq = qs[r + 1] - qs[r], lens[r]
        if m == 0 or seq == 0:
            continue
        ids = torch.tensor([max(b, 0) for b in tables[r][: -(-seq // bs)]])
        kk = (kc[ids].double() * ks[ids].double()[:, None, :, None]).reshape(-1, hk, d)[:seq]
        vv = (vc[ids].double() * vs[ids].double()[:, None, :, None]).reshape(-1, hk, d)[:seq]
        at = torch.arange(seq - m, seq)[:, None]
        key = torch.arange(seq)[None]
        see = (key <= at) if causal else torch.ones(m, seq, dtype=torch.bool)
        see = see & (at >= 0)
        if window:
            see = see & (key > at - window)
        rows = slice(qs[r], qs[r + 1])
        for h in range(hq):
            x = q[rows, h].double()
            sc = x @ kk[:, h // (hq // hk)].T * scale
            big[rows, h] = (x.abs() @ kk[:, h // (hq // hk)].abs().T * abs(scale)).amax(-1)
            sc = sc.masked_fill(~see, -math.inf)
            some = see.any(-1)
            top = torch.where(some, sc.amax(-1), 0)
            p = (sc - top[:, None]).exp()
            tot = p.sum(-1)
            w = p / torch.where(some, tot, 1)[:, None]
            out[rows, h] = w @ vv[:, h // (hq // hk)]
            mag[rows, h] = w @ vv[:, h // (hq // hk)].abs()
            lse[rows, h] = top + tot.log()
    return out, lse, mag, big
