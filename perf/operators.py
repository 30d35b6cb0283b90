"""The serving operators over a block-scaled e4m3 paged cache, as cases to measure.

Four operators make one serving step: ``maps`` (block tables and slot maps from
request lengths), ``rotary`` (rotary positions with several axes), ``append``
(new keys and values quantised into the paged cache, one scale for each block
and head) and ``attend`` (attention over that cache).  ``run`` computes them in
their plain form, or with the framework's kernels where ``own`` is true.
"""

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
F8 = torch.float8_e4m3fn
FMAX = 448.0  # largest finite e4m3 value
FLOOR = 2.0 ** -64  # smallest scale of a block
THETA = 1e6


# ------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of 64 sessions with 2k-32k tokens each: one new token a session
        {"name": "maps_decode_64", "op": "maps", "reqs": 64, "cached_lo": 2048, "cached_hi": 32768, "new_lo": 1,
         "new_hi": 1, "bs": 16, "pad": 0, "mix": 1},
        # a chunked-prefill step of 512 requests, some of them decoding, padded to a graph's size
        {"name": "maps_chunked_512", "op": "maps", "reqs": 512, "cached_lo": 0, "cached_hi": 8192, "new_lo": 1,
         "new_hi": 128, "bs": 16, "pad": 37, "mix": 2},
        # a decode step's queries and keys, Qwen3-8B heads, positions of three axes
        {"name": "rotary_decode_64", "op": "rotary", "tokens": 64, "hq": 32, "hk": 8, "dim": 128, "rotary": 128,
         "axes": 3, "inter": False, "inverse": False, "dtype": "bf16", "far": 32768},
        # a whole 30,720-token prefill at Qwen3-14B heads
        {"name": "rotary_prefill_30720", "op": "rotary", "tokens": 30720, "hq": 40, "hk": 8, "dim": 128,
         "rotary": 128, "axes": 3, "inter": False, "inverse": False, "dtype": "bf16", "far": 32768},
        # the transpose (un-rotation, also the gradient) in fp32 with a partial rotary and interleaved axes
        {"name": "rotary_inverse_4099", "op": "rotary", "tokens": 4099, "hq": 16, "hk": 8, "dim": 128, "rotary": 64,
         "axes": 3, "inter": True, "inverse": True, "dtype": "fp32", "far": 1000000},
        # a decode step's append: one token into a partly filled block of each of 64 sessions
        {"name": "append_decode_64", "op": "append", "reqs": 64, "cached_lo": 2048, "cached_hi": 8192, "new_lo": 1,
         "new_hi": 1, "heads": 8, "dim": 128, "bs": 16, "dtype": "bf16", "layout": "nhd", "mix": 3},
        # the 28,608 tokens behind an edit, written from position 2,292 (inside a block)
        {"name": "append_turn_28608", "op": "append", "reqs": 1, "cached_lo": 2292, "cached_hi": 2292,
         "new_lo": 28608, "new_hi": 28608, "heads": 8, "dim": 128, "bs": 16, "dtype": "bf16", "layout": "nhd",
         "mix": 4},
        # the first answers of a short session: one token over 160 cached, Qwen3-0.6B heads
        {"name": "attend_decode_short", "op": "attend", "reqs": 1, "len_lo": 161, "len_hi": 161, "new_lo": 1,
         "new_hi": 1, "hq": 16, "hk": 8, "dim": 128, "bs": 16, "dtype": "bf16", "layout": "nhd", "window": 0,
         "pow2": True, "mix": 5},
        # one token of the 30,720-token Qwen3-14B session: few rows over a long cache
        {"name": "attend_decode_30720", "op": "attend", "reqs": 1, "len_lo": 30720, "len_hi": 30720, "new_lo": 1,
         "new_hi": 1, "hq": 40, "hk": 8, "dim": 128, "bs": 16, "dtype": "bf16", "layout": "nhd", "window": 0,
         "pow2": True, "mix": 6},
        # one token of each of 64 sessions of 2k-32k tokens, Qwen3-8B heads
        {"name": "attend_decode_64", "op": "attend", "reqs": 64, "len_lo": 2048, "len_hi": 32768, "new_lo": 1,
         "new_hi": 1, "hq": 32, "hk": 8, "dim": 128, "bs": 16, "dtype": "bf16", "layout": "hnd", "window": 0,
         "pow2": True, "mix": 7},
        # an edit's replacement text (244 tokens, and fewer) computed over the history of eight sessions
        {"name": "attend_chunk_8", "op": "attend", "reqs": 8, "len_lo": 2048, "len_hi": 30720, "new_lo": 64,
         "new_hi": 244, "hq": 40, "hk": 8, "dim": 128, "bs": 16, "dtype": "fp16", "layout": "nhd", "window": 0,
         "pow2": False, "mix": 8},
        # the prefill of 8,192 tokens, Qwen3-8B heads
        {"name": "attend_prefill_8192", "op": "attend", "reqs": 1, "len_lo": 8192, "len_hi": 8192, "new_lo": 8192,
         "new_hi": 8192, "hq": 32, "hk": 8, "dim": 128, "bs": 16, "dtype": "bf16", "layout": "nhd", "window": 0,
         "pow2": True, "mix": 9},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["maps", "rotary", "append", "attend", "attend"])
    mix, bs = rng.randrange(1 << 20), rng.choice([16, 16, 32, 64, 24])
    layout = rng.choice(["nhd", "hnd", "split", "split_blocks"])
    if op == "maps":
        reqs = _log(rng, 1, 512)
        lo = _log(rng, 1, 16000)
        return {"op": op, "reqs": reqs, "cached_lo": 0, "cached_hi": lo, "new_lo": rng.choice([0, 1]),
                "new_hi": _log(rng, 1, 128), "bs": bs, "pad": rng.choice([0, rng.randrange(1, 300)]), "mix": mix}
    dim = rng.choice([64, 128, 128, 256])
    if op == "rotary":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        hq, hk = rng.choice([(16, 8), (32, 8), (40, 8), (8, 1), (5, 5)])
        most = 30720 * 48 * 128 * 2 // ((hq + hk) * dim * (4 if dtype == "fp32" else 2))
        return {"op": op, "tokens": min(most, _log(rng, 1, 30720)), "hq": hq, "hk": hk, "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2]), "axes": rng.choice([1, 3, 3]),
                "inter": rng.choice([False, True]), "inverse": rng.choice([False, True]), "dtype": dtype,
                "far": _log(rng, 100, 1000000)}
    if op == "append":
        reqs, heads = _log(rng, 1, 64), rng.choice([1, 2, 4, 8])
        most = max(1, 28608 * 8 * 128 // (reqs * heads * dim))
        new = _log(rng, 1, min(most, 28608))
        return {"op": op, "reqs": reqs, "cached_lo": 0, "cached_hi": _log(rng, 1, 4000), "new_lo": max(1, new // 2),
                "new_hi": new, "heads": heads, "dim": dim, "bs": bs, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "layout": layout, "mix": mix}
    hq, hk = rng.choice([(16, 8), (32, 8), (40, 8), (4, 1), (8, 8), (16, 1)])
    dtype, pow2 = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([False, True])
    if rng.random() < 0.6:  # decoding, now and then with a few tokens at once
        reqs = _log(rng, 1, 64)
        new, length = rng.choice([1, 1, 1, 2, 4]), _log(rng, 4, min(30720, max(8, 1000000 // reqs)))
    else:  # chunks and prefills; the plain form's scores stay below the largest listed case's
        reqs, new = _log(rng, 1, 8), _log(rng, 5, 4096)
        length = min(30720, new + _log(rng, 1, 20000))
        while reqs * new * length * hq * dim > 8192 * 8192 * 32 * 64:
            reqs, new, length = max(1, reqs // 2), max(5, new * 2 // 3), max(8, length * 3 // 4)
        length = max(length, new)
    return {"op": op, "reqs": reqs, "len_lo": max(new, length // 3), "len_hi": length, "new_lo": max(1, new // 2),
            "new_hi": new, "hq": hq, "hk": hk, "dim": dim, "bs": bs, "dtype": dtype, "layout": layout,
            "window": rng.choice([0, 0, _log(rng, 16, 4096)]), "pow2": pow2, "mix": mix}


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """(cached or whole lengths, new lengths) of the case's requests: part of the case, not of the seed."""
    r = random.Random(case["mix"])
    lo, hi = (case["len_lo"], case["len_hi"]) if case["op"] == "attend" else (case["cached_lo"], case["cached_hi"])
    first = [r.randint(lo, hi) for _ in range(case["reqs"])]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["reqs"])]
    return first, new


def _cum(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cache(layout, blocks, bs, heads, dim):
    shape = {"nhd": (blocks, bs, heads, 2 * dim), "hnd": (blocks, heads, bs, 2 * dim),
             "split": (2, blocks, bs, heads, dim), "split_blocks": (blocks, 2, bs, heads, dim)}[layout]
    return shape


def _sides(kv, layout):
    """K and V of a paged cache as views [blocks, bs, heads, dim]."""
    if layout == "split":
        return kv[0], kv[1]
    if layout == "split_blocks":
        return kv[:, 0], kv[:, 1]
    if layout == "hnd":
        kv = kv.transpose(1, 2)
    dim = kv.shape[-1] // 2
    return kv[..., :dim], kv[..., dim:]


def _axes(case):
    """Which axis each frequency takes its position from: contiguous sections, or in turn."""
    half, n = case["rotary"] // 2, case["axes"]
    if case["inter"]:
        return [i % n for i in range(half)]
    return [min(n - 1, i * n // half) for i in range(half)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, bs = case["op"], case.get("bs", 16)
    s = {"case": case}
    if op == "rotary":
        n, dt = case["tokens"], DTYPES[case["dtype"]]
        s["q"] = torch.randn(n, case["hq"], case["dim"], device=DEV, generator=g).to(dt)
        s["k"] = torch.randn(n, case["hk"], case["dim"], device=DEV, generator=g).to(dt)
        s["positions"] = torch.randint(0, case["far"], (case["axes"], n), device=DEV, generator=g)
        e = torch.arange(0, case["rotary"], 2, dtype=torch.float32, device=DEV) / case["rotary"]
        s["inv_freq"] = 1.0 / (THETA ** e)
        s["axes"] = _i32(_axes(case))
        return s
    first, new = _lengths(case)
    total = [a + b for a, b in zip(first, new)] if op != "attend" else first
    need = [-(-t // bs) for t in total]
    blocks, width = sum(need) + 5, max(need) + 3
    perm = torch.randperm(blocks, device=DEV, generator=g).to(torch.int32)
    if op == "maps":
        have = [-(-c // bs) for c in first]
        tables = torch.full((len(first), width), -1, dtype=torch.int32, device=DEV)
        held = torch.arange(width, device=DEV)[None, :] < _i32(have)[:, None]
        tables[held] = perm[: sum(have)]
        s["tables"], s["free"], s["head"] = tables, perm[sum(have):].contiguous(), _i32([0])
        s["cached"], s["new"] = _i32(first), _i32(new)
        s["tokens"] = sum(new) + case["pad"]
        return s
    held = torch.arange(width, device=DEV)[None, :] < _i32(need)[:, None]
    tables = torch.full((len(first), width), -1, dtype=torch.int32, device=DEV)
    tables[held] = perm[: sum(need)]
    s["tables"], s["query_start"], s["seq_lens"] = tables, _i32(_cum(new)), _i32(total)
    s["max_new"], s["max_len"] = max(new), max(total)
    heads, dim = case.get("heads", case.get("hk")), case["dim"]
    shape = _cache(case["layout"], blocks, bs, heads, dim)
    n, dt = sum(new), DTYPES[case["dtype"]]
    loud = 10.0 ** (torch.rand(heads, dim, device=DEV, generator=g) * 2 - 1)  # a scale for each channel
    if op == "append":
        s["kv"] = (torch.randn(shape, device=DEV, generator=g, dtype=torch.bfloat16) * 60).clamp(-FMAX, FMAX).to(F8)
        # what the blocks held before: some scales will grow
        s["k_scale"] = 2.0 ** torch.randint(-7, -2, (blocks, heads), device=DEV, generator=g).float()
        s["v_scale"] = 2.0 ** torch.randint(-7, -2, (blocks, heads), device=DEV, generator=g).float()
        s["k"] = (torch.randn(n, heads, dim, device=DEV, generator=g) * loud).to(dt)
        s["v"] = torch.randn(n, heads, dim, device=DEV, generator=g).to(dt)
        return s
    s["kv"] = (torch.randn(shape, device=DEV, generator=g, dtype=torch.bfloat16) * 100).clamp(-FMAX, FMAX).to(F8)
    for name in ("k_scale", "v_scale"):
        if case["pow2"]:  # what append writes
            s[name] = 2.0 ** torch.randint(-8, -4, (blocks, heads), device=DEV, generator=g).float()
        else:  # scales of another origin
            s[name] = torch.rand(blocks, heads, device=DEV, generator=g) * 0.03 + 0.005
    s["q"] = torch.randn(n, case["hq"], dim, device=DEV, generator=g).to(dt)
    return s


# -------------------------------------------------------------- plain forms
def _rows(query_start, tokens, reqs):
    """The request of each token row and the row's place in it; rows behind the last request get `reqs`."""
    t = torch.arange(tokens, device=DEV)
    r = torch.searchsorted(query_start[1:].long(), t, right=True)
    return r, t - query_start.long()[r.clamp(max=reqs)]


def _plain_maps(s):
    bs, n = s["case"]["bs"], s["tokens"]
    cached, new, tables = s["cached"].long(), s["new"].long(), s["tables"]
    reqs = cached.numel()
    zero = torch.zeros(1, dtype=torch.long, device=DEV)
    query_start = torch.cat((zero, new.cumsum(0)))
    have, need = (cached + bs - 1) // bs, (cached + new + bs - 1) // bs
    first = torch.cat((zero, (need - have).cumsum(0)))
    col = torch.arange(tables.shape[1], device=DEV)[None, :]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    at = s["head"].long() + first[:-1, None] + col - have[:, None]
    tables.copy_(torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], tables))
    r, i = _rows(query_start, n, reqs)
    live, r = r < reqs, r.clamp(max=reqs - 1)
    pos = torch.where(live, cached[r] + i, 0)
    slots = torch.where(live, tables[r, pos // bs].long() * bs + pos % bs, -1)
    return [query_start.int(), (cached + new).int(), slots, pos, (s["head"].long() + first[-1:]).int(), tables]


def _rotate(x, cos, sin, rotary):
    half = rotary // 2
    x = x.to(cos.dtype)
    a, b = x[..., :half], x[..., half:rotary]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rotary:]), -1)


def _plain_rotary(s):
    case = s["case"]
    angle = s["positions"][s["axes"].long()].T.double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    sin = -sin if case["inverse"] else sin
    return [_rotate(x, cos, sin, case["rotary"]).to(x.dtype) for x in (s["q"], s["k"])]


def _pow2_scale(amax):
    """The least power of two s with amax <= 448 s, and at least FLOOR."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), FLOOR).clamp(min=FLOOR)


def _plain_append_side(x, cache, scale, blk, off, fresh, start_of_block):
    """One side (K or V): cache is a view [blocks, bs, heads, dim], blk/off the place of each row."""
    x = x.float()
    amax = torch.where(x.isfinite(), x.abs(), 0).amax(-1)
    want = torch.zeros_like(scale).scatter_reduce_(0, blk[:, None].expand_as(amax), amax, "amax")
    touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=DEV).index_fill_(0, blk, True)
    new = torch.where(fresh[:, None], _pow2_scale(want), torch.maximum(scale, _pow2_scale(want)))
    new = torch.where(touched[:, None], new, scale)
    grown = torch.nonzero(touched & ~fresh).squeeze(1)
    bs = cache.shape[1]
    old = cache[grown].float() * (scale[grown] / new[grown])[:, None, :, None]
    keep = torch.arange(bs, device=DEV)[None, :] < start_of_block[grown][:, None]
    was = cache[grown].view(torch.uint8)
    cache.view(torch.uint8)[grown] = torch.where(keep[..., None, None], old.to(F8).view(torch.uint8), was)
    rows = (x / new[blk][..., None]).clamp(-FMAX, FMAX).to(F8)
    cache.view(torch.uint8)[blk, off] = rows.view(torch.uint8)
    scale.copy_(new)


def _plain_append(s):
    bs, tables = s["case"]["bs"], s["tables"]
    new = s["query_start"].long().diff()
    reqs = new.numel()
    r, i = _rows(s["query_start"], s["k"].shape[0], reqs)
    start = s["seq_lens"].long() - new
    pos = start[r] + i
    blk, off = tables[r, pos // bs].long(), pos % bs
    blocks = s["k_scale"].shape[0]
    # where each touched block's first new row stands: 0 means that it held nothing of the request before
    begin = torch.full((blocks,), bs, dtype=torch.long, device=DEV).scatter_reduce_(0, blk, off, "amin")
    k, v = _sides(s["kv"], s["case"]["layout"])
    _plain_append_side(s["k"], k, s["k_scale"], blk, off, begin == 0, begin)
    _plain_append_side(s["v"], v, s["v_scale"], blk, off, begin == 0, begin)
    return [s["kv"], s["k_scale"], s["v_scale"]]


def _plain_attend(s):
    case, bs, tables = s["case"], s["case"]["bs"], s["tables"]
    reqs, hq, hk, dim = tables.shape[0], case["hq"], case["hk"], case["dim"]
    kc, vc = _sides(s["kv"], case["layout"])
    longest = s["max_len"]
    cols = -(-longest // bs)
    ids = tables[:, :cols].long().clamp(min=0)
    k = (kc[ids].float() * s["k_scale"][ids][:, :, None, :, None]).reshape(reqs, cols * bs, hk, dim)
    k = k[:, :longest].permute(0, 2, 3, 1)  # [reqs, hk, dim, keys]
    q, n = s["q"], s["q"].shape[0]
    r, i = _rows(s["query_start"], n, reqs)
    most = s["max_new"]
    padded = torch.zeros(reqs, most, hq, dim, device=DEV)
    padded[r, i] = q.float()
    rows = padded.view(reqs, most, hk, hq // hk, dim).permute(0, 2, 1, 3, 4).reshape(reqs, hk, -1, dim)
    scores = (rows @ k) / math.sqrt(dim)
    del k
    new = s["query_start"].long().diff()
    at = (s["seq_lens"].long() - new)[:, None] + torch.arange(most, device=DEV)  # [reqs, most]
    key = torch.arange(longest, device=DEV)
    seen = key <= at[..., None]
    if case["window"]:
        seen &= key > at[..., None] - case["window"]
    seen = seen[:, None, :, None, :].expand(-1, -1, -1, hq // hk, -1).reshape(reqs, 1, -1, longest)
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top.isfinite(), top, 0)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = (vc[ids].float() * s["v_scale"][ids][:, :, None, :, None]).reshape(reqs, cols * bs, hk, dim)[:, :longest]
    there = key[None, :] < s["seq_lens"].long()[:, None]
    v = torch.where(there[:, :, None, None], v, 0).permute(0, 2, 1, 3)
    out = (p @ v) / torch.where(total > 0, total, 1)
    lse = top + total.log()
    out = out.view(reqs, hk, most, hq // hk, dim).permute(0, 2, 1, 3, 4).reshape(reqs, most, hq, dim)
    lse = lse.view(reqs, hk, most, hq // hk).permute(0, 2, 1, 3).reshape(reqs, most, hq)
    return [out[r, i].to(q.dtype), lse[r, i].contiguous()]


# --------------------------------------------------------------------- run
def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    return {"maps": _plain_maps, "rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}[op](s)


def _own(s, op):
    if op == "maps":
        from marathon_b200.block_maps import block_maps

        m = block_maps(s["cached"], s["new"], s["tables"], s["free"], s["head"], s["case"]["bs"], s["tokens"])
        return [m.query_start, m.seq_lens, m.slots, m.positions, m.free_head, s["tables"]]
    if op == "rotary":
        from marathon_b200.rotary import rotary_axes

        return list(rotary_axes(s["q"], s["k"], s["positions"], s["inv_freq"], s["axes"],
                                inverse=s["case"]["inverse"]))
    from marathon_b200.block_scaled import append_block_scaled, attend_block_scaled

    case = s["case"]
    if op == "append":
        append_block_scaled(s["k"], s["v"], s["kv"], s["k_scale"], s["v_scale"], s["tables"], s["query_start"],
                            s["seq_lens"], case["bs"], case["layout"])
        return [s["kv"], s["k_scale"], s["v_scale"]]
    return list(attend_block_scaled(s["q"], s["kv"], s["k_scale"], s["v_scale"], s["tables"], s["query_start"],
                                    s["seq_lens"], case["bs"], case["layout"], max_query_len=s["max_new"],
                                    max_seq_len=s["max_len"], window=case["window"], return_lse=True))


# -------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "rotary":
        es = 4 if case["dtype"] == "fp32" else 2
        n, heads = case["tokens"], case["hq"] + case["hk"]
        return {"bytes": 2 * n * heads * case["dim"] * es + 8 * n * case["axes"] + 4 * case["rotary"],
                "flops": 3 * n * heads * case["rotary"]}
    first, new = _lengths(case)
    bs, reqs, n = case["bs"], case["reqs"], sum(new)
    if op == "maps":
        fresh = sum(-(-(c + m) // bs) - -(-c // bs) for c, m in zip(first, new))
        return {"bytes": 8 * reqs + 4 * (2 * reqs + 1) + 16 * (n + case["pad"]) + 8 * fresh + 4 * reqs + 8,
                "flops": 4 * n}
    dim = case["dim"]
    if op == "append":
        es, heads = (4 if case["dtype"] == "fp32" else 2), case["heads"]
        blocks = sum(-(-(c + m) // bs) - c // bs for c, m in zip(first, new) if m)
        return {"bytes": 2 * n * heads * dim * (es + 1) + blocks * (4 + 2 * 2 * 4 * heads),
                "flops": 4 * n * heads * dim}
    keys = pairs = 0
    for length, m in zip(first, new):
        w = case["window"] or length
        low = max(0, length - m - w + 1)
        keys += length - low
        if w >= length:
            pairs += m * length - m * (m - 1) // 2
        else:
            pairs += sum(min(w, length - m + i + 1) for i in range(m))
    return {"bytes": 2 * keys * case["hk"] * dim + (keys // bs + reqs) * (4 + 8 * case["hk"])
            + n * case["hq"] * (4 * dim + 4), "flops": 4 * dim * case["hq"] * pairs}


# ------------------------------------------------------------------- exact
def _e4m3_f64(x):
    """The e4m3 value nearest to x (ties to the even code), in 64 bits."""
    a = x.abs().clamp(max=FMAX)
    e = torch.floor(torch.log2(a.clamp(min=2.0 ** -6))).clamp(min=-6)
    e = torch.where(torch.exp2(e) > a.clamp(min=2.0 ** -6), e - 1, e)
    step = torch.exp2(e - 3)
    return torch.copysign((a / step).round() * step, x)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "maps":
        return None
    if op == "rotary":
        ang = torch.stack([s["positions"][a].double() * f for a, f in zip(_axes(case), s["inv_freq"].double())], 1)
        turn = torch.polar(torch.ones_like(ang), -ang if case["inverse"] else ang)[:, None]
        half = case["rotary"] // 2
        got = []
        for x in (s["q"], s["k"]):
            y = x.double()
            z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
            y[..., :half], y[..., half:2 * half] = z.real, z.imag
            got.append(y)
        return got
    first, new = _lengths(case)
    bs = case["bs"]
    kv = s["kv"].double()
    k, v = _sides(kv, case["layout"])
    starts = _cum(new)
    if op == "append":
        if case["reqs"] > 1 and sum(new) > 40000:
            return None
        ks, vs = s["k_scale"].double(), s["v_scale"].double()
        table = s["tables"].tolist()
        old = [(c, m, c // bs, -(-(c + m) // bs)) for c, m in zip(first, new)]
        for x, cache, scale in ((s["k"].double(), k, ks), (s["v"].double(), v, vs)):
            for i, (c, m, b0, b1) in enumerate(old):
                ids = torch.tensor(table[i][b0:b1], device=DEV)
                # the request's new rows laid out by block, zeros before and behind them
                lay = torch.zeros((b1 - b0) * bs, *x.shape[1:], dtype=torch.float64, device=DEV)
                lay[c - b0 * bs: c - b0 * bs + m] = x[starts[i]: starts[i + 1]]
                lay = lay.view(b1 - b0, bs, *x.shape[1:])
                peak = lay.abs().amax((1, 3))
                want = torch.exp2(torch.ceil(torch.log2((peak / FMAX).clamp(min=FLOOR)))).clamp(min=FLOOR)
                if c % bs:  # the first block holds earlier tokens
                    want[0] = torch.maximum(want[0], scale[ids[0]])
                    kept = cache[ids[0], : c % bs] * (scale[ids[0]] / want[0])[None, :, None]
                    cache[ids[0], : c % bs] = _e4m3_f64(kept)
                codes = _e4m3_f64(lay / want[:, None, :, None])
                flat = torch.arange(c, c + m, device=DEV)
                cache[ids[flat // bs - b0], flat % bs] = codes.view(-1, *x.shape[1:])[c - b0 * bs: c - b0 * bs + m]
                scale[ids] = want
        return [kv, ks, vs]
    hq, hk, dim = case["hq"], case["hk"], case["dim"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for i, (length, m) in enumerate(zip(first, new)):
        ids = s["tables"][i, : -(-length // bs)].long()
        kk = (k[ids] * s["k_scale"][ids].double()[:, None, :, None]).reshape(-1, hk, dim)[:length]
        vv = (v[ids] * s["v_scale"][ids].double()[:, None, :, None]).reshape(-1, hk, dim)[:length]
        at = torch.arange(length - m, length, device=DEV)[:, None]
        key = torch.arange(length, device=DEV)[None]
        hide = key > at
        if case["window"]:
            hide = hide | (key <= at - case["window"])
        for h in range(hq):
            sc = q[starts[i]: starts[i + 1], h] @ kk[:, h // (hq // hk)].T / dim ** 0.5
            sc = sc.masked_fill(hide, -math.inf)
            lse[starts[i]: starts[i + 1], h] = torch.logsumexp(sc, -1)
            out[starts[i]: starts[i + 1], h] = torch.softmax(sc, -1) @ vv[:, h // (hq // hk)]
    return [out, lse]
