"""ops.rotary_frequencies / rotary_tables / rotary against the formulas in 64 bits.

Tolerances.  A table entry is computed in double and rounded once: half a step of its type
(eps/2 relative, 2^-25 absolute for float16's subnormals) plus the double angle's error.  That
angle is position * f: three roundings of relative size 2^-53 on each side (f / 2 pi, the product,
the reduction) are at most position * f * 2^-50 together, and 64 rotation steps add 64 * 2^-52.
A rotated value is a c - b s in fp32 (three roundings of at most 2^-24 of the terms) rounded once.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def reference_frequencies(dim, base, scaling, factor, original, low, high):
    out = []
    if scaling == "ntk":
        base = base * factor ** (dim / (dim - 2))
    for j in range(dim // 2):
        f = base ** (-2 * j / dim)
        keep = 1.0
        if scaling == "linear":
            keep = 0.0
        elif scaling == "yarn":
            lo = max(0, math.floor(dim * math.log(original / (high * 2 * math.pi)) / (2 * math.log(base))))
            hi = min(dim - 1, math.ceil(dim * math.log(original / (low * 2 * math.pi)) / (2 * math.log(base))))
            keep = 1 - min(1.0, max(0.0, (j - lo) / max(hi - lo, 1e-3)))
        elif scaling == "bands":
            keep = min(1.0, max(0.0, (original * f / (2 * math.pi) - low) / (high - low)))
        out.append(f * keep + f / factor * (1 - keep))
    return out, (0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0)


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn", "bands"])
@pytest.mark.parametrize("dim,positions,start,dtype", [
    (128, 4097, 0, torch.float16), (128, 1000, 1 << 20, torch.float32), (2, 1, 7, torch.float32),
    (80, 777, 3, torch.float16), (10, 70001, 123456, torch.float32), (512, 65, 2**31 - 100, torch.float32)])
def test_tables(ops, scaling, dim, positions, start, dtype):
    if scaling == "ntk" and dim == 2:
        pytest.skip("refused: ntk needs more than two channels")
    high = 4.0 if scaling == "bands" else 32.0
    freq, amp = ops.rotary_frequencies(dim, base=500000.0, scaling=scaling, factor=8.0, original_positions=8192)
    want, want_amp = reference_frequencies(dim, 500000.0, scaling, 8.0, 8192, 1.0, high)
    assert amp == pytest.approx(want_amp, rel=1e-15)
    torch.testing.assert_close(freq, torch.tensor(want, dtype=torch.float64), rtol=1e-14, atol=0)
    cos, sin = ops.rotary_tables(freq, positions, amplitude=amp, start=start, dtype=dtype)
    assert cos.dtype == dtype and cos.shape == (positions, dim // 2) and cos.device == torch.device(DEV)
    pos = torch.arange(start, start + positions, dtype=torch.float64, device=DEV)
    ang = pos[:, None] * freq.to(DEV)
    slack = amp * (ang * 2.0 ** -50 + 64 * 2.0 ** -52) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    for got, ref in ((cos, ang.cos() * amp), (sin, ang.sin() * amp)):
        err = (got.double() - ref).abs()
        # 1.001: a double on the other side of a rounding border moves the half step by far less
        assert bool((err <= 1.001 * (torch.finfo(dtype).eps / 2) * ref.abs() + slack).all())


def test_tables_of_no_position_and_tables_feed_rope(ops):
    freq, amp = ops.rotary_frequencies(64)
    cos, sin = ops.rotary_tables(freq, 0)
    assert cos.shape == (0, 32)
    cos, sin = ops.rotary_tables(freq, 300)
    q, k = torch.randn(9, 4, 64, device=DEV).half(), torch.randn(9, 2, 64, device=DEV).half()
    pos = torch.randint(0, 300, (9,), device=DEV, dtype=torch.int32)
    for a, b in zip(ops.rope(q, k, pos, cos, sin), ops.rotary(q, k, pos, cos, sin)):
        assert torch.equal(a, b)  # the same arithmetic in the same order


def check_rotary(x, out, pos, cos, sin, interleaved):
    half = cos.shape[1]
    ok = (pos >= 0) & (pos < cos.shape[0])
    idx = pos.clamp(0, cos.shape[0] - 1).long()
    c, s = cos.double()[idx][:, None], sin.double()[idx][:, None]
    j = torch.arange(half, device=x.device)
    d0, d1 = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
    a, b = x.double()[..., d0], x.double()[..., d1]
    want, bound = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    want[..., d0], want[..., d1] = a * c - b * s, b * c + a * s
    bound[..., d0] = (a * c).abs() + (b * s).abs()
    bound[..., d1] = (b * c).abs() + (a * s).abs()
    want[~ok], bound[~ok] = 0, 0
    err = (out.double() - want).abs()
    exact = bound == 0
    assert bool((err[exact] == 0).all())
    assert bool((err <= 2.0 ** -11 * want.abs() * (1 + 2.0 ** -11) + 3 * 2.0 ** -24 * bound + 2.0 ** -25).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rot", [
    (1, 28, 4, 128, 128), (64, 28, 4, 128, 64), (37, 5, 3, 96, 24), (5, 1, 1, 256, 256), (3, 2, 7, 10, 6),
    (130, 32, 8, 128, 128), (7, 3, 1, 64, 2), (33, 9, 2, 80, 48), (4, 40, 10, 64, 32), (2, 1, 1, 16, 16),
    (19, 6, 2, 120, 112)])
def test_rotary(ops, interleaved, dtype, tokens, hq, hkv, dim, rot):
    g = torch.Generator(device=DEV).manual_seed(tokens * 131 + rot)
    q = torch.randn(tokens, hq, dim, generator=g, device=DEV).half()
    k = torch.randn(tokens, hkv, dim, generator=g, device=DEV).half()
    cos = torch.randn(200, rot // 2, generator=g, device=DEV).to(dtype)
    sin = torch.randn(200, rot // 2, generator=g, device=DEV).to(dtype)
    pos = torch.randint(0, 200, (tokens,), generator=g, device=DEV, dtype=torch.int32)
    pos[0] = 199
    if tokens > 2:
        pos[1], pos[2] = -1, 200  # name no row: zeros
    oq, ok = ops.rotary(q, k, pos, cos, sin, interleaved)
    assert oq.shape == q.shape and oq.is_contiguous() and ok.shape == k.shape
    check_rotary(q, oq, pos, cos, sin, interleaved)
    check_rotary(k, ok, pos, cos, sin, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_rotary_of_views(ops, interleaved, pad):
    """q and k as views of a packed projection (token stride = its row), also at odd offsets."""
    tokens, hq, hkv, dim, rot = 21, 6, 2, 64, 32
    buf = torch.randn(tokens, pad + (hq + 2 * hkv) * dim, device=DEV).half()
    q = buf[:, pad:pad + hq * dim].view(tokens, hq, dim)
    k = buf[:, pad + hq * dim:pad + (hq + hkv) * dim].view(tokens, hkv, dim)
    cos, sin = torch.randn(50, rot // 2, device=DEV), torch.randn(50, rot // 2, device=DEV)
    pos = torch.randint(0, 50, (tokens,), device=DEV, dtype=torch.int32)
    oq, ok = ops.rotary(q, k, pos, cos, sin, interleaved)
    check_rotary(q, oq, pos, cos, sin, interleaved)
    check_rotary(k, ok, pos, cos, sin, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,dtype", [
    (701, 28, 5, 128, 128, torch.float16), (5003, 31, 8, 128, 64, torch.float32), (9001, 15, 2, 80, 48, torch.float16),
    (4500, 33, 0, 136, 72, torch.float32)])
def test_rotary_of_many_tokens(ops, interleaved, tokens, hq, hkv, dim, rot, dtype):
    """Several heads per thread, head counts that do not divide by it, packed views, bad positions."""
    buf = torch.randn(tokens, (hq + hkv) * dim + 8, device=DEV).half()
    q = buf[:, :hq * dim].view(tokens, hq, dim)
    k = buf[:, hq * dim:(hq + hkv) * dim].view(tokens, hkv, dim)
    cos, sin = torch.randn(300, rot // 2, device=DEV).to(dtype), torch.randn(300, rot // 2, device=DEV).to(dtype)
    pos = torch.randint(-3, 303, (tokens,), device=DEV, dtype=torch.int32)
    oq, ok = ops.rotary(q, k, pos, cos, sin, interleaved)
    check_rotary(q, oq, pos, cos, sin, interleaved)
    check_rotary(k, ok, pos, cos, sin, interleaved)


def test_rotary_zero_sizes_and_one_row_table(ops):
    cos = torch.ones(1, 8, device=DEV).half()
    for tokens, hq, hkv in ((0, 4, 2), (3, 0, 2), (3, 4, 0)):
        q, k = torch.randn(tokens, hq, 16, device=DEV).half(), torch.randn(tokens, hkv, 16, device=DEV).half()
        pos = torch.zeros(tokens, dtype=torch.int32, device=DEV)
        oq, ok = ops.rotary(q, k, pos, cos, torch.zeros_like(cos))
        assert torch.equal(oq, q) and torch.equal(ok, k)


def test_rotary_on_a_side_stream_and_in_a_graph(ops):
    q, k = torch.randn(40, 8, 128, device=DEV).half(), torch.randn(40, 2, 128, device=DEV).half()
    pos = torch.arange(40, device=DEV, dtype=torch.int32)
    freq, amp = ops.rotary_frequencies(128, scaling="yarn", factor=4.0, original_positions=4096)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cos, sin = ops.rotary_tables(freq, 100, amplitude=amp)
        ops.rotary(q, k, pos, cos, sin)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cos2, sin2 = ops.rotary_tables(freq, 100, amplitude=amp)
        oq, ok = ops.rotary(q, k, pos, cos2, sin2)
    q.copy_(torch.randn_like(q))
    pos.copy_(torch.randperm(100, device=DEV)[:40].int())
    graph.replay()
    assert torch.equal(cos, cos2) and torch.equal(sin, sin2)
    check_rotary(q, oq, pos, cos, sin, False)
    check_rotary(k, ok, pos, cos, sin, False)


def test_tables_rewritten_between_calls(ops, cabi):
    """Tables and inputs rewritten in place between two rotary calls of one stream, launch after launch without a
    pause: every call sees what its predecessor wrote."""
    f = [cabi.rotary_frequencies(128, base=b)[0] for b in (1e4, 3e5)]
    q, k = torch.randn(700, 28, 128, device=DEV).half(), torch.randn(700, 4, 128, device=DEV).half()
    pos = torch.randint(0, 700, (700,), device=DEV, dtype=torch.int32)
    cos, sin = torch.empty(700, 64, device=DEV), torch.empty(700, 64, device=DEV)
    outs = []
    for i in range(12):
        cabi.rotary_tables(f[i % 2], 1.0, 0, cos, sin, 1)
        outs.append(ops.rotary(q, k, pos, cos, sin))
    for i, (oq, ok) in enumerate(outs):
        c, s = ops.rotary_tables(torch.tensor(f[i % 2], dtype=torch.float64), 700, dtype=torch.float32)
        check_rotary(q, oq, pos, c, s, False)
        check_rotary(k, ok, pos, c, s, False)
