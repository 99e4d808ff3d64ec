"""ops.chunked_paged_attention against its definition in 64 bits.

Tolerance.  With A = sum_s p_s |v_s| (p normalised), the kernel's result differs from the exact one by
  - rounding of the result to float16: 2^-11 |out| + 2^-25;
  - rounding of each probability to float16: 2^-11 A, and 2^-25 sum |v_s| / l for subnormal ones,
    l >= 1 the sum relative to the row's maximum;
  - errors of the scores: the dot product adds D products in fp32, (D + 4) 2^-23 sum |q k| / sqrt(D)
    at most; a change e of every score moves the result by at most 2 e A; the exponential's argument and
    value add (|s - m| + 4) 2^-22, at most (2 max |s| + 4) 2^-22;
  - fp32 accumulation over the tokens, in groups of 16 and with one rescaling per tile:
    (tokens / 8 + 64) 2^-23 A for the sums and the same for l.
"""
import ctypes

import pytest
import torch

from conftest import knob

import decode_workloads as wl

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NHD, NZ = wl.KV_LAYOUT_NHD, wl.KV_LAYOUT_NZ


def make(lens, hq, hkv, d, page, layout=NHD, seed=0, extra_pages=3, extra_width=2, tail_rows=0):
    """lens: (new tokens, context) per sequence.  Unused cache slots and spare pages hold NaN, table
    entries past a sequence's pages name no page or a poisoned one."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(ctx, 0) // page) for _, ctx in lens]
    pages = sum(need) + extra_pages
    order = torch.randperm(pages, generator=g)
    width = max(need + [1]) + extra_width
    table = torch.empty(len(lens), width, dtype=torch.int32)
    kc = torch.full((pages, page, hkv, d), float("nan"))
    vc = torch.full((pages, page, hkv, d), float("nan"))
    spare = order[sum(need):]
    o = 0
    for b, (n, ctx) in enumerate(lens):
        mine = order[o:o + need[b]]
        o += need[b]
        table[b] = torch.where(torch.arange(width) % 2 == 0, -1, int(spare[0]))
        table[b, :need[b]] = mine.int()
        for i, p in enumerate(mine.tolist()):
            t = min(page, ctx - i * page)
            kc[p, :t] = torch.randn(t, hkv, d, generator=g)
            vc[p, :t] = torch.randn(t, hkv, d, generator=g)
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1] + tail_rows, hq, d, generator=g)
    kc, vc = kc.half(), vc.half()
    if layout == NZ:
        kc, vc = (x.reshape(pages, page, hkv * d // 16, 16).transpose(1, 2).contiguous() for x in (kc, vc))
    return dict(q=q.half().to(DEV), kc=kc.to(DEV), vc=vc.to(DEV), table=table.to(DEV),
                ctx=torch.tensor([c for _, c in lens], dtype=torch.int32, device=DEV),
                starts=torch.tensor(starts, dtype=torch.int32, device=DEV), hkv=hkv, page=page, layout=layout)


def dense(cache, rows, s, d):
    x = cache[rows]
    if s["layout"] == NZ:
        x = x.transpose(1, 2)
    return x.reshape(-1, s["hkv"], d).double()


def reference(s):
    """(result, tolerance) in 64 bits; rows of no sequence are NaN in the result."""
    q, d, page = s["q"], s["q"].shape[2], s["page"]
    group = q.shape[1] // s["hkv"]
    pages = s["kc"].shape[0]
    cap = s["table"].shape[1] * page
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    starts, ctxs = s["starts"].tolist(), s["ctx"].tolist()
    for b in range(len(ctxs)):
        n, L = starts[b + 1] - starts[b], min(max(ctxs[b], 0), cap)
        if n == 0:
            continue
        rows = slice(starts[b], starts[b] + n)
        out[rows] = 0
        if L == 0:
            continue
        ids = s["table"][b, :-(-L // page)].long()
        ok = ((ids >= 0) & (ids < pages)).repeat_interleave(page)[:L]
        k = dense(s["kc"], ids.clamp(0, pages - 1), s, d)[:L]
        v = dense(s["vc"], ids.clamp(0, pages - 1), s, d)[:L]
        k[~ok], v[~ok] = 0, 0
        pos = torch.arange(L - n, L, device=DEV)
        see = (torch.arange(L, device=DEV)[None] <= pos[:, None]) & ok[None]
        any_seen = see.any(1)
        for h in range(q.shape[1]):
            kk, vv, qq = k[:, h // group], v[:, h // group], q[rows, h].double()
            score = (qq @ kk.T) * d ** -0.5
            size = ((qq.abs() @ kk.abs().T) * d ** -0.5).masked_fill(~see, 0).amax(1, keepdim=True)
            top = score.masked_fill(~see, float("-inf")).amax(1, keepdim=True)
            p = torch.where(see, torch.exp(score - top), 0.0)
            l = p.sum(1, keepdim=True)
            p = torch.where(any_seen[:, None], p / l, 0.0)
            r = p @ vv
            big = p @ vv.abs()
            e = (d + 4) * 2.0 ** -23 * size + (2 * size + 4) * 2.0 ** -22
            t = (2.0 ** -11 * r.abs() + 2.0 ** -25 + big * (2.0 ** -11 + 2 * e + 2 * (L / 8 + 64) * 2.0 ** -23)
                 + 2.0 ** -25 * (see.double() @ vv.abs()) / l)
            out[rows, h] = torch.where(any_seen[:, None], r, 0.0)
            tol[rows, h] = torch.where(any_seen[:, None], t, 0.0)
    return out, tol


def call(ops, s):
    return ops.chunked_paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["starts"])


@pytest.fixture(autouse=True)
def _no_wait_ran_out(cabi):
    yield
    assert cabi.pipeline_status() == 0


def check(got, s):
    want, tol = reference(s)
    owned = ~want.isnan()
    err = (got.double() - want).abs()
    bad = owned & ~(err <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(err[owned].max()), bad.nonzero()[:4].tolist())


LENS = [
    [(1, 1)],
    [(1, 700), (1, 1), (1, 129), (1, 64)],
    [(5, 5), (1, 300), (0, 10), (17, 40), (128, 128)],
    [(33, 290), (200, 200), (64, 1000), (1, 5)],
    [(3, 2), (1, 0), (20, 7), (2, 2)],  # more new tokens than context: the first ones see nothing
    [(300, 700)],
]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("hq,hkv,d,page,layout", [
    (28, 4, 128, 128, NHD), (8, 8, 128, 16, NHD), (8, 1, 64, 64, NHD), (12, 4, 64, 16, NHD), (3, 1, 32, 8, NHD),
    (2, 2, 256, 32, NHD), (28, 4, 128, 128, NZ), (8, 2, 64, 16, NZ), (5, 1, 128, 7, NHD), (6, 2, 128, 1, NHD),
    (4, 2, 32, 24, NZ), (64, 2, 128, 64, NHD), (20, 2, 128, 40, NHD), (160, 2, 64, 16, NHD), (4, 4, 128, 48, NZ)])
def test_shapes(ops, lens, hq, hkv, d, page, layout):
    s = make(lens, hq, hkv, d, page, layout, seed=len(lens) * 7 + hq)
    check(call(ops, s), s)


@pytest.mark.parametrize("hq,hkv,d,page", [(28, 4, 128, 128), (8, 2, 64, 16), (4, 1, 128, 5), (16, 1, 128, 32)])
@pytest.mark.parametrize("lens", [
    [(1, 9000)],                              # one token, one long context: split and merged
    [(7, 5000), (1, 3), (40, 6000)],
    [(1, c) for c in range(1, 130, 7)],
    [(130, 2100), (513, 513), (1, 4000), (1, 4096), (1, 4097)]])
def test_long_contexts(ops, lens, hq, hkv, d, page):
    s = make(lens, hq, hkv, d, page, seed=hq + page)
    check(call(ops, s), s)


def test_single_tokens_agree_with_decode_attention(ops):
    s = make([(1, c) for c in (1, 17, 700, 128, 2049, 4000)], 28, 4, 128, 128, seed=4)
    a = call(ops, s)
    b = ops.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["ctx"])
    _, tol = reference(s)
    assert bool(((a.double() - b.double()).abs() <= 2 * tol).all())


@pytest.mark.parametrize("hq,hkv,d,page,layout", [(28, 4, 128, 64, NHD), (8, 2, 64, 16, NHD), (8, 2, 128, 16, NZ), (4, 2, 32, 3, NHD)])
def test_pages_that_name_nothing(ops, hq, hkv, d, page, layout):
    """Entries outside the cache inside a context: their tokens are left out, also when that leaves a row nothing."""
    s = make([(70, 300), (1, 200), (5, 5), (3, 130)], hq, hkv, d, page, layout, seed=9)
    s["table"][0, 1] = -1
    s["table"][0, 2] = s["kc"].shape[0]
    s["table"][1, 0] = -7
    s["table"][2, :] = 2**31 - 1
    s["table"][3, :] = -(2**31)
    check(call(ops, s), s)


@pytest.mark.parametrize("hq,hkv,d,page,layout", [(28, 4, 128, 64, NHD), (8, 2, 64, 16, NHD), (8, 2, 128, 16, NZ), (4, 2, 32, 3, NHD), (2, 1, 256, 16, NHD)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_values_behind_a_row_do_not_reach_it(ops, hq, hkv, d, page, layout, value):
    """Non-finite keys and values of the chunk's later tokens: earlier rows keep their results, bit for bit."""
    s = make([(150, 400), (20, 20)], hq, hkv, d, page, layout, seed=5)
    clean = call(ops, s)
    hit = 340  # position inside the first sequence's chunk: rows 90.. see it
    pg, off = int(s["table"][0, hit // page]), hit % page
    at = (pg, off, 0, 3) if layout == NHD else (pg, 0, off, 3)
    s["vc"][at] = value
    got = call(ops, s)
    first = hit - 250
    assert torch.equal(got[:first], clean[:first]) and torch.equal(got[150:], clean[150:])
    group = hq // hkv
    assert torch.equal(got[first:150, group:], clean[first:150, group:])
    col = got[first:150, :group, 3].double()
    assert bool(col.isnan().all()) if value != value else bool((col == value).all())
    others = [i for i in range(d) if i != 3]
    assert torch.equal(got[first:150, :group][..., others], clean[first:150, :group][..., others])
    s["vc"][at] = 1.0
    s["kc"][at] = value
    got = call(ops, s)
    assert torch.equal(got[:first], clean[:first]) and torch.equal(got[150:], clean[150:])


def test_rows_of_no_sequence_are_left_alone(cabi):
    s = make([(4, 90), (9, 9)], 28, 4, 128, 128, seed=2, tail_rows=6)
    out = torch.full_like(s["q"], 7.25)
    ws = torch.full((cabi.chunked_paged_attention_workspace_size(19, 2, 28, 4, 128, 128, s["table"].shape[1]),), 0xA5,
                    dtype=torch.uint8, device=DEV)
    cabi.chunked_paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["starts"], out, 4, 128, NHD, ws)
    torch.cuda.synchronize()
    assert bool((out[13:] == 7.25).all())
    check(out[:13], {**s, "q": s["q"][:13]})


def test_context_above_the_tables_capacity_and_odd_starts(ops):
    s = make([(3, 256), (2, 100)], 8, 2, 128, 64, seed=8, extra_width=0)
    want = call(ops, s)
    s["ctx"][0] = 2**31 - 1
    assert torch.equal(call(ops, s), want)
    s["starts"][2] = 1 << 30  # past the rows there are
    assert torch.equal(call(ops, s), want)
    s["ctx"][1] = -5
    assert bool((call(ops, s)[3:] == 0).all())


def test_empty_calls(ops):
    s = make([(2, 5)], 4, 2, 64, 16)
    assert ops.chunked_paged_attention(s["q"][:0], s["kc"], s["vc"], s["table"], s["ctx"], s["starts"]).shape == (0, 4, 64)
    none = ops.chunked_paged_attention(s["q"], s["kc"], s["vc"], s["table"][:0], s["ctx"][:0], s["starts"][:1])
    assert none.shape == s["q"].shape


def test_large_scores_and_one_dominant_key(ops):
    """Scores of several hundred, with the maximum found early, late and growing tile by tile."""
    s = make([(40, 1500)], 4, 2, 128, 64, seed=6)
    flat = s["kc"][s["table"][0, :24].long()].reshape(-1, 2, 128)
    ramp = torch.linspace(0.02, 1.0, 1500, device=DEV)
    flat[:1500] = (s["q"][20:21, ::2] * 4 * ramp[:, None, None]).half()
    s["kc"][s["table"][0, :24].long()] = flat.reshape(24, 64, 2, 128)
    check(call(ops, s), s)
    s["kc"][s["table"][0, :24].long()] = torch.cat((flat[:1500].flip(0), flat[1500:])).reshape(24, 64, 2, 128)
    check(call(ops, s), s)


def test_repeatable_on_streams_and_from_graphs(ops):
    """Bitwise the same eagerly, on another stream, and from graphs replayed with other lengths; two
    graphs share one memory pool, so also their workspaces' memory."""
    s = make([(60, 500), (1, 3000), (1, 60), (90, 90)], 28, 4, 128, 128, seed=12)
    want = call(ops, s)
    for _ in range(5):
        assert torch.equal(call(ops, s), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(ops, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = call(ops, s)
    with torch.cuda.graph(g2, pool=g1.pool()):
        o2 = call(ops, s)
    for _ in range(2):
        g1.replay()  # in the order of capture, as a shared pool asks: g2's tensors may lie where g1 had scratch
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(o1, want) and torch.equal(o2, want)
    s["starts"].copy_(torch.tensor([0, 1, 61, 62, 152], dtype=torch.int32))
    s["ctx"].copy_(torch.tensor([450, 2000, 33, 90], dtype=torch.int32))
    g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(o2, call(ops, s))
    check(o2, s)


def test_guards_around_output_and_workspace(cabi):
    s = make([(60, 500), (1, 3000), (2, 60)], 28, 4, 128, 128, seed=13)
    n = s["q"].numel()
    raw = torch.full((n + 8192,), 0x7B3C, dtype=torch.int16, device=DEV)
    out = raw[4096:4096 + n].view(torch.float16).view(s["q"].shape)
    need = cabi.chunked_paged_attention_workspace_size(63, 3, 28, 4, 128, 128, s["table"].shape[1])
    ws = torch.full((need + 8192,), 0x5C, dtype=torch.uint8, device=DEV)
    cabi.chunked_paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["starts"], out, 4, 128, NHD,
                                 ws[4096:4096 + need])
    torch.cuda.synchronize()
    assert bool((raw[:4096] == 0x7B3C).all()) and bool((raw[4096 + n:] == 0x7B3C).all())
    assert bool((ws[:4096] == 0x5C).all()) and bool((ws[4096 + need:] == 0x5C).all())
    check(out, s)


@pytest.mark.parametrize("hq,hkv,d,page", [(28, 4, 128, 128), (8, 2, 64, 8), (128, 1, 128, 32)])
def test_general_kernel_on_the_same_shapes(ops, monkeypatch, hq, hkv, d, page):
    s = make([(33, 290), (1, 2000), (70, 70), (2, 1)], hq, hkv, d, page, seed=21)
    fast = call(ops, s)
    knob(monkeypatch, "B200OPS_PA_MODE", 2)
    general = call(ops, s)
    check(fast, s)
    check(general, s)


def test_many_sequences(ops):
    g = torch.Generator().manual_seed(3)
    lens = [(int(n), int(n + c)) for n, c in torch.randint(0, 12, (1500, 2), generator=g)]
    s = make(lens, 4, 2, 64, 16, seed=3)
    check(call(ops, s), s)


def test_offsets_past_32_bits(ops):
    """A cache of more than 2^31 elements, its last pages in use."""
    pages, page, hkv, d = 132000, 128, 1, 128
    kc = torch.empty(pages, page, hkv, d, dtype=torch.float16, device=DEV)
    vc = torch.empty_like(kc)
    ids = torch.tensor([pages - 1, 3, pages - 2], device=DEV)
    kc[ids], vc[ids] = torch.randn(3, page, hkv, d, device=DEV).half(), torch.randn(3, page, hkv, d, device=DEV).half()
    s = dict(q=torch.randn(37, 4, d, device=DEV).half(), kc=kc, vc=vc, table=ids.int()[None].contiguous(),
             ctx=torch.tensor([370], dtype=torch.int32, device=DEV),
             starts=torch.tensor([0, 37], dtype=torch.int32, device=DEV), hkv=hkv, page=page, layout=NHD)
    check(call(ops, s), s)


@pytest.mark.parametrize("hq,hkv,d,page", [
    (28, 4, 128, 8), (8, 2, 128, 64), (6, 2, 64, 8), (16, 1, 64, 128), (12, 4, 128, 32), (14, 2, 128, 56), (3, 3, 64, 40)])
@pytest.mark.parametrize("lens", [
    [(5, 5), (1, 300), (0, 10), (17, 40), (128, 128)], [(3, 2), (1, 0), (20, 7), (2, 2)], [(300, 1700), (1, 2500)]])
def test_caches_in_rows_of_16_channels(ops, lens, hq, hkv, d, page):
    s = make(lens, hq, hkv, d, page, NZ, seed=hq + page)
    check(call(ops, s), s)


@pytest.mark.parametrize("layout", [NHD, NZ])
@pytest.mark.parametrize("hq,hkv,d,page,lens", [
    (14, 2, 128, 32, [(1, 700)] * 200),
    (14, 2, 128, 128, [(400, 400)] * 6),
    (8, 2, 64, 16, [(1, 300), (100, 260), (1, 900), (73, 800)] * 20),
    (28, 4, 128, 128, [(1, 5), (0, 40), (36, 36), (1, 1), (19, 500), (2, 1), (18, 4000), (1, 66)] * 8)])
def test_many_pieces_of_work_in_a_row(ops, layout, hq, hkv, d, page, lens):
    """Every CTA goes through several items of both kinds; the same bits each time, also back to back."""
    s = make(lens, hq, hkv, d, page, layout, seed=len(lens))
    outs = [call(ops, s) for _ in range(4)]
    check(outs[0], s)
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


@pytest.mark.parametrize("hq,hkv,d,lens", [
    (7, 1, 128, [(1, 30000)]), (2, 2, 128, [(1, 1024), (1, 1100), (1, 1600), (1, 2100)]), (4, 1, 64, [(1, 12000), (3, 9000)]),
    (4, 1, 128, [(200, 9000)]), (128, 1, 128, [(2, 6000)])])
def test_contexts_cut_into_many_parts(ops, hq, hkv, d, lens):
    s = make(lens, hq, hkv, d, 64, seed=hq)
    check(call(ops, s), s)


def test_non_finite_query_rows_stay_by_themselves(ops):
    """A NaN and an infinite query: their rows are NaN, all others keep their bits."""
    s = make([(50, 900), (1, 700)], 28, 4, 128, 128, seed=30)
    clean = call(ops, s)
    s["q"][7, 3, 5] = float("nan")
    s["q"][20, 27] = float("inf")
    got = call(ops, s)
    assert bool(got[7, 3].isnan().all()) and bool(got[20, 27].isnan().all())
    hit = torch.zeros(51, 28, dtype=torch.bool, device=DEV)
    hit[7, 3] = hit[20, 27] = True
    assert torch.equal(got[~hit], clean[~hit])


def test_output_aligned_to_16_bytes_only(cabi):
    s = make([(60, 500), (1, 3000), (2, 60)], 28, 4, 128, 128, seed=14)
    raw = torch.zeros(s["q"].numel() + 16, dtype=torch.float16, device=DEV)
    shift = 8 if raw.data_ptr() % 32 == 0 else 0
    out = raw[shift:shift + s["q"].numel()].view(s["q"].shape)
    assert out.data_ptr() % 32 == 16
    ws = torch.empty(cabi.chunked_paged_attention_workspace_size(63, 3, 28, 4, 128, 128, s["table"].shape[1]),
                     dtype=torch.uint8, device=DEV)
    cabi.chunked_paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["starts"], out, 4, 128, NHD, ws)
    check(out, s)


def test_two_calls_at_once(ops):
    """Two streams, each with calls of its own, at the same time on the device."""
    a, b = make([(60, 2500), (1, 3000)], 28, 4, 128, 128, seed=15), make([(300, 300), (1, 900)], 8, 2, 64, 16, seed=16)
    want_a, want_b = call(ops, a), call(ops, b)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(8):
        with torch.cuda.stream(sa):
            outs.append((call(ops, a), want_a))
        with torch.cuda.stream(sb):
            outs.append((call(ops, b), want_b))
    torch.cuda.synchronize()
    for got, want in outs:
        assert torch.equal(got, want)


def test_workspace_aligned_to_16_bytes_only(cabi):
    for seed, (hq, hkv, d, page) in enumerate([(28, 4, 128, 128), (4, 2, 32, 16)]):
        s = make([(60, 5000), (1, 3000), (2, 60)], hq, hkv, d, page, seed=seed)
        need = cabi.chunked_paged_attention_workspace_size(63, 3, hq, hkv, d, page, s["table"].shape[1])
        raw = torch.full((need + 512,), 0x5C, dtype=torch.uint8, device=DEV)
        assert raw.data_ptr() % 256 == 0
        for at in (16, 240):
            out = torch.empty_like(s["q"])
            cabi.chunked_paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["starts"], out, hkv, page, NHD,
                                         raw[at:at + need])
            check(out, s)
            assert bool((raw[:at] == 0x5C).all()) and bool((raw[at + need:] == 0x5C).all())
            raw.fill_(0x5C)


@pytest.mark.parametrize("hq,hkv,d,page,layout", [
    (28, 4, 128, 64, NHD), (8, 2, 64, 16, NHD), (8, 2, 128, 16, NZ), (3, 3, 64, 8, NZ), (4, 2, 32, 3, NHD)])
def test_many_non_finite_values(ops, hq, hkv, d, page, layout):
    """Infinities and NaN in a tenth of a percent to a half of the values of the chunk and in a few before it: a row is
    what those at its positions make it, channel by channel, and keeps its bits where there are none."""
    n, L = 150, 410
    s = make([(n, L), (20, 20)], hq, hkv, d, page, layout, seed=40)
    clean = call(ops, s)
    g = torch.Generator().manual_seed(41)
    density = torch.zeros(L, 1, 1)
    density[L - n:L - n + 40] = 0.001
    density[L - n + 60:L - n + 70] = 0.02
    density[L - 40:] = 0.5
    density[5] = 0.01
    put = torch.rand(L, hkv, d, generator=g) < density
    bad = torch.tensor([float("inf"), float("-inf"), float("nan")])[torch.randint(0, 3, (L, hkv, d), generator=g)]
    vc = s["vc"].cpu() if layout == NHD else s["vc"].cpu().transpose(1, 2).reshape(-1, page, hkv, d)
    for p in range(L):
        at = (int(s["table"][0, p // page]), p % page)
        vc[at] = torch.where(put[p], bad[p].half(), vc[at])
    s["vc"] = (vc if layout == NHD else vc.reshape(-1, page, hkv * d // 16, 16).transpose(1, 2)).contiguous().to(DEV)
    got = call(ops, s).cpu()
    assert torch.equal(got[n:], clean[n:].cpu())
    seen = torch.where(put, bad, torch.zeros(())).double().cumsum(0)[L - n:]  # inf - inf and NaN: NaN
    seen = seen.repeat_interleave(hq // hkv, 1)
    hit = put.cumsum(0)[L - n:].repeat_interleave(hq // hkv, 1) > 0
    assert torch.equal(got[:n][~hit], clean[:n].cpu()[~hit])
    assert torch.equal(got[:n][hit].double().nan_to_num(nan=1.0), seen[hit].nan_to_num(nan=1.0))
