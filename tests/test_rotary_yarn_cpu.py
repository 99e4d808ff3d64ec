"""Which end of the spectrum yarn scaling divides: the contract of b200ops_rotary_frequencies, index by index."""
import math

import pytest


@pytest.mark.parametrize("dim,base,original,low,high", [(128, 1e4, 4096, 1.0, 32.0), (64, 5e5, 8192, 1.0, 32.0), (128, 1e6, 32768, 2.0, 20.0)])
def test_yarn_keeps_the_high_frequencies(cabi, dim, base, original, low, high):
    factor = 8.0
    plain, _ = cabi.rotary_frequencies(dim, base=base)
    f, _ = cabi.rotary_frequencies(dim, base=base, scaling=cabi.ROTARY_YARN, factor=factor, original_positions=original,
                                   low=low, high=high)

    def index(turns):
        return dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))

    first, last = math.floor(index(high)), math.ceil(index(low))
    assert 0 < first < last < dim // 2
    for j in range(dim // 2):
        if j <= first:
            assert f[j] == plain[j]
        elif j >= last:
            assert f[j] == pytest.approx(plain[j] / factor, rel=1e-14)
        else:
            keep = 1 - (j - first) / (last - first)
            assert f[j] == pytest.approx(plain[j] * keep + plain[j] / factor * (1 - keep), rel=1e-13)
