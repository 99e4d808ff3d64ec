"""ops.chunked_paged_attention where probabilities are tiny: what many of them add up to, and what a non-finite value of
such a key does; and scores of -inf.

The scores are set through channel 0 alone: q has sqrt(D) there and 0 elsewhere, so a key's score is its value in
channel 0, up to the rounding of sqrt(D) to float16, which the reference applies too.
"""
import math

import pytest
import torch

import decode_workloads as wl

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NHD, NZ = wl.KV_LAYOUT_NHD, wl.KV_LAYOUT_NZ


def state(news, scores, values, hq, hkv, page, layout=NHD):
    """Sequences of `news` new tokens that all see the same context: `scores` [L], `values` [L, hkv, D]."""
    length, _, d = values.shape
    pages = -(-length // page)
    kc = torch.full((pages * page, hkv, d), float("nan"))
    vc = kc.clone()
    kc[:length], vc[:length] = 0, values
    kc[:length, :, 0] = scores[:, None]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(pages))
    place = torch.empty_like(order)
    place[order] = torch.arange(pages)  # page i of the context lies in page place[i] of the cache
    kc, vc = (x.view(pages, page, hkv, d)[order].half() for x in (kc, vc))
    if layout == NZ:
        kc, vc = (x.reshape(pages, page, hkv * d // 16, 16).transpose(1, 2).contiguous() for x in (kc, vc))
    q = torch.zeros(sum(news), hq, d)
    q[..., 0] = math.sqrt(d)
    starts = torch.tensor([0] + list(news), dtype=torch.int32).cumsum(0).int()
    return dict(q=q.half().to(DEV), kc=kc.to(DEV), vc=vc.to(DEV), layout=layout, news=news, scores=scores, values=values,
                table=place.int()[None].repeat(len(news), 1).to(DEV), starts=starts.to(DEV),
                ctx=torch.full((len(news),), length, dtype=torch.int32, device=DEV))


def call(ops, s):
    return ops.chunked_paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["starts"])


@pytest.fixture(autouse=True)
def _no_wait_ran_out(cabi):
    yield
    assert cabi.pipeline_status() == 0


SHAPES = [(28, 4, 128, 128, NHD), (8, 2, 64, 16, NHD), (8, 2, 128, 16, NZ), (4, 2, 32, 3, NHD), (2, 1, 256, 16, NHD)]


@pytest.mark.parametrize("hq,hkv,d,page,layout", SHAPES)
@pytest.mark.parametrize("news", [[1], [1] * 320, [150], [40] * 90])
def test_many_small_probabilities(ops, hq, hkv, d, page, layout, news):
    """One key with the highest score and values 0, the others 18 below it (probability 2^-26 of its) with large values:
    the result is the others' alone.

    Rounding a probability to float16 moves it by 2^-11 of itself, or, where it is subnormal, by 2^-32 of the row's
    largest (the kernels keep the largest at 2^7 or more: 2^-25 / 2^7).  The rest as for any row: the result's rounding,
    scores and exponentials off by (2 * 18 + 4) 2^-22 + (d + 4) 2^-23 * 18, sums by (L / 8 + 64) 2^-23.
    """
    length = 4096
    g = torch.Generator().manual_seed(d)
    scores = torch.full((length,), -18.0)
    scores[0] = 0
    values = (torch.rand(length, hkv, d, generator=g) + 1) * 16384
    values[0] = 0
    s = state(news, scores, values.half().float(), hq, hkv, page, layout)
    out = call(ops, s).double().cpu()
    step = float(s["q"][0, 0, 0]) / math.sqrt(d)
    v = s["values"].double().repeat_interleave(hq // hkv, 1)
    p = torch.exp(s["scores"].double() * step)
    t = 0
    for n in news[:3]:
        for i in sorted({0, n // 2, n - 1}):
            last = length - n + i + 1
            l = p[:last].sum()
            want = torch.einsum("s,shd->hd", p[:last], v[:last]) / l
            e = (2 * 18 + 4) * 2.0 ** -22 + (d + 4) * 2.0 ** -23 * 18
            tol = want * (2 * 2.0 ** -11 + 2 * e + 2 * (length / 8 + 64) * 2.0 ** -23) + 2.0 ** -32 * v[:last].sum(0) / l
            err = (out[t + i] - want).abs()
            assert bool((err <= tol).all()), (n, i, float((err / tol).max()), float(want.mean()))
        t += n


@pytest.mark.parametrize("hq,hkv,d,page,layout", SHAPES)
@pytest.mark.parametrize("length", [300, 9000])  # in one piece, and cut into parts
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_non_finite_values_of_unlikely_keys(ops, hq, hkv, d, page, layout, length, value):
    """A visible key 300 below the highest score, which is the last one: its probability is 0 in fp32, but by the definition
    it is not, so a non-finite value of it makes its channel non-finite; the other channels stay as they were."""
    g = torch.Generator().manual_seed(length)
    scores = torch.randn(length, generator=g) - 300
    scores[-1] = 0
    values = torch.randn(length, hkv, d, generator=g)
    clean = call(ops, state([1, 1], scores, values, hq, hkv, page, layout))
    assert bool(clean.isfinite().all())
    values[17, 0, 5] = value
    got = call(ops, state([1, 1], scores, values, hq, hkv, page, layout))
    hit = torch.zeros(hq, d, dtype=torch.bool, device=DEV)
    hit[:hq // hkv, 5] = True
    assert not bool(got[:, hit].isfinite().any())
    assert torch.equal(got[:, ~hit], clean[:, ~hit])


@pytest.mark.parametrize("hq,hkv,d,page,layout", SHAPES)
@pytest.mark.parametrize("low,length,new", [(6, 12, 12), (300, 300, 40), (200, 300, 150), (300, 700, 700), (9000, 9000, 1),
                                            (8999, 9000, 3), (8900, 9000, 200), (4000, 9000, 1)])
def test_scores_of_minus_infinity(ops, hq, hkv, d, page, layout, low, length, new):
    """The first `low` keys have the score -inf.  A row that sees no other key is NaN (0 / 0); behind the first other key
    those have no weight."""
    g = torch.Generator().manual_seed(low)
    scores = torch.zeros(length)
    scores[:low] = float("-inf")
    values = torch.randn(length, hkv, d, generator=g)
    got = call(ops, state([new, new], scores, values, hq, hkv, page, layout))
    nothing = max(0, low - (length - new))  # rows that see keys of -inf only
    for t in (0, new):
        assert bool(got[t:t + nothing].isnan().all())
        if nothing < new:
            first = max(low, length - new)  # position of the first row that sees another key
            mean = values[low:].half().double().cumsum(0)[first - low:] / torch.arange(first - low + 1, length - low + 1)[:, None, None]
            size = values[low:].half().double().abs().cumsum(0)[first - low:] / torch.arange(first - low + 1, length - low + 1)[:, None, None]
            # equal weights: exact in float16; the sums' and the result's rounding are left
            tol = 2.0 ** -11 * mean.abs() + 2.0 ** -25 + 2 * (length / 8 + 64) * 2.0 ** -23 * size
            want, tol = (x.repeat_interleave(hq // hkv, 1).to(DEV) for x in (mean, tol))
            assert bool(((got[t + nothing:t + new].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("hq,hkv,d,page,layout", SHAPES)
def test_rows_that_see_nothing_beside_scores_of_minus_infinity(ops, hq, hkv, d, page, layout):
    """More new tokens than context: the first rows stand before every key and are zeros, the others see -inf only."""
    s = state([20], torch.full((12,), float("-inf")), torch.randn(12, hkv, d), hq, hkv, page, layout)
    got = call(ops, s)
    assert bool((got[:8] == 0).all()) and bool(got[8:].isnan().all())
    s["table"].fill_(-1)
    assert bool((call(ops, s) == 0).all())
