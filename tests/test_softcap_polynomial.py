"""The softcap's polynomial as it stands in the source, against tanh in extended precision, on the CPU."""
import re

import numpy as np
import pytest

from conftest import PKG

mpmath = pytest.importorskip("mpmath")
U = 2.0 ** -24


def coefficients():
    text = (PKG / "csrc" / "logit_rows.cuh").read_text()
    body = re.search(r"tanh_coef\(int i\).*?\{([-0-9.f, e]+)\}", text, re.S).group(1)
    return [np.float32(c.strip().rstrip("f")) for c in body.split(",")]


def test_distance_from_tanh():
    """Of the stored coefficients: 0.93 u on 0 < z <= 1."""
    c = [mpmath.mpf(float(a)) for a in coefficients()]
    assert len(c) == 6
    worst = mpmath.mpf(0)
    with mpmath.workdps(30):
        for i in range(1, 3001):
            w = (1 - mpmath.cos(mpmath.pi * i / 3000)) / 2
            z = mpmath.sqrt(w)
            p = mpmath.mpf(0)
            for a in reversed(c):
                p = p * w + a
            worst = max(worst, abs((1 + w * p) * z / mpmath.tanh(z) - 1))
    assert worst <= 0.93 * U


@pytest.mark.parametrize("cap", [0.7, 5.0, 30.0, 50.0, 2.0e4])
def test_evaluated_in_fp32(cap):
    """x P((x / cap)^2) with every step rounded to fp32 is within 5 u of cap tanh(x / cap).  A fused
    multiply-add is formed in 64 bits here: its product is exact there, its sum is rounded at 2^-53."""
    f = np.float32
    inv = f(1.0 / f(cap))
    x = np.concatenate([np.linspace(1e-4, 1.0, 4001), 10.0 ** np.linspace(-6, 0, 500)]).astype(f) * f(cap)
    x = x[x <= f(cap)]
    z = x * inv
    w = z * z
    c = coefficients()
    p = np.full_like(x, c[5])
    for a in [*c[4::-1], f(1.0)]:
        p = (p.astype(np.float64) * w + np.float64(a)).astype(f)
    got = (x * p).astype(np.float64)
    with mpmath.workdps(30):
        want = [float(mpmath.mpf(float(f(cap))) * mpmath.tanh(mpmath.mpf(float(v)) / mpmath.mpf(float(f(cap))))) for v in x]
    assert np.abs(got / np.array(want) - 1).max() <= 5 * U + 2.0 ** -50
