"""rotary_tables at far positions against angles reduced in 60 digits.

Bound.  Reducing position * f leaves roundings of numbers below one turn only, 2^-50 with those of its cosine and sine.  Every
rotation step behind it (64 at most) adds the errors of the step's cosine and sine (an ulp each, 2^-52 sqrt 2 as a
vector), of its angle (2^-52) and of the four operations (2^-52 sqrt 2): below 2^-50.  The entry is then rounded once to
its type: half a step of it.
"""
import math
from decimal import Decimal, getcontext

import pytest
import torch

pytestmark = pytest.mark.gpu

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def exact_angle(position, f):
    """position * f less whole turns, in [-pi, pi]."""
    getcontext().prec = 60
    a = Decimal(position) * Decimal(f)
    return float(a - (a / (2 * PI)).to_integral_value() * 2 * PI)


@pytest.mark.parametrize("start", [0, 200000, 2**31 - 600])
@pytest.mark.parametrize("freqs,amplitude", [
    ([1.0, 1e6 ** (-2 / 128), 0.31, 1e-7], 1.0), ([12345.678, 1e6, math.pi, 2 * math.pi], 1.25)])
def test_far_positions(ops, freqs, amplitude, start):
    n = 500
    f = torch.tensor(freqs, dtype=torch.float64)
    cos, sin = ops.rotary_tables(f, n, amplitude=amplitude, start=start, dtype=torch.float32)
    want_c, want_s = torch.empty(n, len(freqs), dtype=torch.float64), torch.empty(n, len(freqs), dtype=torch.float64)
    for i in range(n):
        for j, x in enumerate(freqs):
            a = exact_angle(start + i, x)
            want_c[i, j], want_s[i, j] = amplitude * math.cos(a), amplitude * math.sin(a)
    for got, want in ((cos, want_c), (sin, want_s)):
        err = (got.double().cpu() - want).abs()
        tol = 2.0 ** -24 * (1 + 2.0 ** -20) * want.abs() + amplitude * (1 + 64) * 2.0 ** -50
        assert bool((err <= tol).all()), float((err / tol).max())
