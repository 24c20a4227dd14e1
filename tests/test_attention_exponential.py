"""The polynomial 2^x of csrc/fl_attn.cuh, with its coefficients read from there, step by step in FP32 on the CPU.

Its approximation is off by 1.1e-7 of the value.  The last step rounds a value in [0.70, 1.42] (2^-24 of it at
most), the one before a value in [0.58, 0.83] (2^-25) that |f| <= 1/2 halves, the others less than half of that
again: 1.1e-7 + 2^-24 + 2^-26 + 2^-26 < 2^-22.  The argument's split and the power of two are exact."""
import os
import re

import numpy as np

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spilltune_b200", "csrc",
                      "fl_attn.cuh")


def _coefficients():
    with open(SOURCE) as f:
        body = re.search(r"void ex2_pair\(.*?\n}", f.read(), re.S).group(0)
    return [float(c) for c in re.findall(r"pair\((0\.\d+|1\.0)f, \1f\)", body)]


def _fma(a, b, c):  # the product of two FP32 numbers is exact in FP64
    return (a.astype(np.float64) * b.astype(np.float64) + np.float64(c)).astype(np.float32)


def _exp2(x):
    f32 = np.float32
    x = np.maximum(x, f32(-127))
    i = (x + f32(12582912)) - f32(12582912)
    f = (x - i).astype(f32)
    first, *rest = (f32(c) for c in _coefficients())
    p = _fma(f, np.full_like(f, first), rest[0])
    for c in rest[1:]:
        p = _fma(f, p, c)
    power = (i.astype(np.int32) * (1 << 23) + 0x3F800000).astype(np.int32).view(f32)
    return p * power


def test_polynomial():
    assert len(_coefficients()) == 6 and _coefficients()[-1] == 1.0
    rng = np.random.default_rng(1)
    x = np.concatenate([np.linspace(-1, 1, 400001), rng.uniform(-126, 10, 400000), np.arange(-126, 11) + 0.5,
                        np.arange(-125, 11)]).astype(np.float32)
    got, want = _exp2(x).astype(np.float64), np.exp2(x.astype(np.float64))
    assert np.abs(got / want - 1).max() <= 2.0 ** -22
    assert np.array_equal(_exp2(np.arange(-126, 11, dtype=np.float32)), np.exp2(np.arange(-126, 11)).astype(np.float32))
    assert not _exp2(np.array([-126.75, -127, -1000, -np.inf], np.float32)).any()
