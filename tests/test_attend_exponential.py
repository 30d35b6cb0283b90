"""The exponential that a quarter of the attention's scores take on the FMA units, restated on the CPU.

The constants are read from the kernel's source.  A product of two fp32 numbers is exact in 64 bits, and a sum
with a third is rounded once to 64 and once to 32 bits, which the fused operation's single rounding
differs from by less than 2^-52 of the value.

Bounds.  The fit itself is within 7.5e-8.  Rounding its coefficients to fp32 adds at most 2^-24 (the constant,
just above one) + 2^-25 / 2 + 2^-27 / 4 + ... < 7.8e-8, over 2^f >= 0.707: 1.9e-7 in all.  The last fused step
rounds by 2^-24 of a value in [0.707, 1.415], at most 8.5e-8 of it, and the one before by 2^-25 |f| <= 2^-26,
2.2e-8; those before count for under a quarter of that: 3.1e-7.
"""

from __future__ import annotations

import re
from pathlib import Path

import numpy as np

SOURCE = Path(__file__).resolve().parent.parent / "marathon_b200" / "csrc" / "attend_rows.cu"


def _coefficients():
    body = SOURCE.read_text()
    body = body[body.index("exp2_pair(float x0"):]
    body = body[: body.index("\n}")]
    pairs = re.findall(r"pair\((0x1\.[0-9a-f]+p[+-]\d+)f, (0x1\.[0-9a-f]+p[+-]\d+)f\)", body)
    assert len(pairs) == 6 and all(a == b for a, b in pairs)
    return [float.fromhex(a) for a, _ in pairs]


def _fma(a, b, c):
    return (a.astype(np.float64) * b + c).astype(np.float32)


def _exp2(x):
    magic = np.float32(12582912.0)
    x = np.maximum(x, np.float32(-126.0))
    t = x + magic
    f = x + _fma(t, np.float64(-1.0), np.float64(magic))
    c = _coefficients()
    r = _fma(f, c[0], c[1])
    for k in c[2:]:
        r = _fma(r, f.astype(np.float64), k)
    return (r.view(np.uint32) + (t.view(np.uint32) << np.uint32(23))).view(np.float32)


def test_the_polynomial_is_two_to_the_f():
    f = np.linspace(-0.5, 0.5, 400_001)
    assert np.abs(np.polyval(_coefficients(), f) / np.exp2(f) - 1).max() < 1.9e-7


def test_the_exponential_in_fp32():
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.uniform(-126, 8, 1_000_000), np.linspace(-3, 3, 100_001), np.arange(-126, 9) + 0.5,
                        np.arange(-126, 9)]).astype(np.float32)
    assert np.abs(_exp2(x) / np.exp2(x.astype(np.float64)) - 1).max() < 3.1e-7
    # masked scores and what is below fp32's normal range: nothing, once it is f16
    low = _exp2(np.array([-np.inf, -1e30, -127.5, -126.0], np.float32))
    assert (np.abs(low / np.float32(2.0**-126) - 1) < 3.1e-7).all() and (low.astype(np.float16) == 0).all()
