"""ops.copy_pages and ops.compact_pages: bit-exact against a loop over the definition."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def caches(shape, tensors, dtype=torch.float16, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    for _ in range(tensors):
        raw = torch.randint(0, 256, (*shape, torch.empty(0, dtype=dtype).element_size()), generator=g, device=DEV,
                            dtype=torch.uint8)
        out.append(raw.view(dtype).squeeze(-1))
    return out


def same_bytes(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def loop_copy(cs, src, dst):
    cs = [c.clone() for c in cs]
    pages = cs[0].shape[0]
    for s, d in zip(src, dst):
        if 0 <= s < pages and 0 <= d < pages:
            for c in cs:
                c[d] = c[s].clone()
    return cs


SHAPES = [(40, 16, 2, 64), (40, 8, 16, 16), (40, 3, 5, 7), (40, 1, 1, 1), (40, 5, 2, 2)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.uint8, torch.float32])
@pytest.mark.parametrize("tensors", [1, 3])
@pytest.mark.parametrize("src,dst", [
    ([3], [5]), ([0, 39], [39, 1]), ([3, 3, 3], [5, 6, 7]),
    ([1, 2, 3], [7, 7, 7]),          # the last pair stays
    ([1, 2], [2, 1]),                # not a swap: the second pair copies page 1 back
    ([1, 2, 3, 4], [2, 3, 4, 5]),    # a chain carries page 1 all the way
    ([4, 3, 2, 1], [5, 4, 3, 2]),    # a shift by one
    ([6, -1, 40, 2, 2**31 - 1], [6, 3, 3, -5, 4]),  # nothing to do
    ([1, 9], [40, 3])])
def test_copy_pages(ops, shape, dtype, tensors, src, dst):
    cs = caches(shape, tensors, dtype)
    want = loop_copy(cs, src, dst)
    ops.copy_pages(cs, torch.tensor(src, dtype=torch.int32, device=DEV), torch.tensor(dst, dtype=torch.int32, device=DEV))
    for a, b in zip(cs, want):
        assert same_bytes(a, b)


@pytest.mark.parametrize("pages,pairs,conflicts", [(9000, 4096, False), (9000, 4400, False), (300, 5000, True),
                                                   (64, 30, False), (2000, 999, True)])
def test_copy_many_pages(ops, pages, pairs, conflicts):
    g = torch.Generator().manual_seed(pairs)
    order = torch.randperm(pages, generator=g)
    if conflicts:
        src, dst = torch.randint(-2, pages + 2, (2, pairs), generator=g)
    else:
        dst, rest = order[:pairs], order[pairs:]
        src = rest[torch.randint(0, len(rest), (pairs,), generator=g)]
    cs = caches((pages, 4, 1, 16), 2, seed=1)
    # the loop on one number per page first: which original page each page ends up holding
    origin = list(range(pages))
    for s, d in zip(src.tolist(), dst.tolist()):
        if 0 <= s < pages and 0 <= d < pages:
            origin[d] = origin[s]
    want = [c[torch.tensor(origin, device=DEV)].clone() for c in cs]
    ops.copy_pages(cs, src.int().to(DEV), dst.int().to(DEV))
    for a, b in zip(cs, want):
        assert same_bytes(a, b)


def test_copy_pages_of_many_tensors_and_unaligned_memory(ops):
    cs = caches((12, 2, 1, 8), 300, seed=2)
    want = loop_copy(cs, [0, 5], [11, 3])
    ops.copy_pages(cs, torch.tensor([0, 5], dtype=torch.int32, device=DEV), torch.tensor([11, 3], dtype=torch.int32, device=DEV))
    assert all(same_bytes(a, b) for a, b in zip(cs, want))
    raw = torch.randn(1 + 12 * 16, device=DEV).half()
    odd = [raw[1:].view(12, 16)]  # two bytes off any vector's alignment
    want = loop_copy(odd, [0, 5], [11, 3])
    first = raw[0].item()
    ops.copy_pages(odd, torch.tensor([0, 5], dtype=torch.int32, device=DEV), torch.tensor([11, 3], dtype=torch.int32, device=DEV))
    assert same_bytes(odd[0], want[0]) and raw[0].item() == first


def loop_compact(cs, table, counts):
    cs = [c.clone() for c in cs]
    pages = cs[0].shape[0]
    live = sorted({p for row, n in zip(table, counts) for p in row[:max(n, 0)] if 0 <= p < pages})
    m = len(live)
    to = {p: p for p in live}
    for p, h in zip([p for p in live if p >= m], [h for h in range(m) if h not in to]):
        to[p] = h
        for c in cs:
            c[h] = c[p].clone()
    new = [[to.get(p, p) if i < n else p for i, p in enumerate(row)] for row, n in zip(table, counts)]
    return cs, new, [to.get(p, -1) for p in range(pages)], m


@pytest.mark.parametrize("pages,seqs,width,fill,shape", [
    (40, 5, 8, 0.6, (16, 2, 64)), (33, 1, 40, 1.0, (4, 1, 16)), (64, 7, 3, 0.9, (3, 5, 7)), (1, 2, 2, 1.0, (2, 2, 8)),
    (1025, 60, 20, 0.5, (8, 1, 16)), (40000, 64, 300, 0.8, (1, 1, 8)), (31, 4, 5, 0.0, (4, 1, 16)),
    (524288, 16, 1000, 0.7, (1, 1, 1))])
def test_compact_pages(ops, pages, seqs, width, fill, shape):
    g = torch.Generator().manual_seed(pages + seqs)
    table = torch.randint(-1, pages + 1, (seqs, width), generator=g)  # shared pages, and entries that name none
    counts = (torch.rand(seqs, generator=g) * (width + 1) * fill).int()
    if seqs > 2 and fill > 0:
        counts[0], counts[1] = -3, width + 5
    cs = caches((pages, *shape), 2, seed=3)
    want, new, page_map, m = loop_compact(cs, table.tolist(), counts.tolist()) if pages < 500 else (None,) * 4
    if want is None:  # the same in bulk
        used = torch.arange(width)[None] < counts[:, None]
        ok = used & (table >= 0) & (table < pages)
        live = torch.zeros(pages, dtype=torch.bool)
        live[table[ok]] = True
        m = int(live.sum())
        idx = torch.arange(pages)
        src, dst = idx[live & (idx >= m)], idx[~live & (idx < m)]
        page_map = torch.where(live, idx, -1)
        page_map[src] = dst
        new = torch.where(ok, page_map[table.clamp(0, pages - 1)], table).tolist()
        page_map = page_map.tolist()
        want = [c.clone() for c in cs]
        for c in want:
            c[dst.to(DEV)] = c[src.to(DEV)]
    tab = table.int().to(DEV)
    got, got_map, live_n = ops.compact_pages(cs, tab, counts.to(DEV))
    assert live_n.tolist() == [m]
    assert got.tolist() == new and got_map.tolist() == page_map
    assert torch.equal(tab.cpu(), table.int())  # the old tables are left alone
    for a, b in zip(cs, want):
        assert same_bytes(a, b)


def test_compact_pages_without_sequences_or_entries(ops):
    cs = caches((10, 4, 1, 16), 1)
    before = cs[0].clone()
    for shape in ((0, 5), (3, 0), (0, 0)):
        tab = torch.zeros(shape, dtype=torch.int32, device=DEV)
        new, page_map, m = ops.compact_pages(cs, tab, torch.ones(shape[0], dtype=torch.int32, device=DEV))
        assert new.shape == shape and page_map.tolist() == [-1] * 10 and m.item() == 0
    assert same_bytes(cs[0], before)


def test_pages_in_a_graph_and_on_a_side_stream(ops):
    """Replays with other pairs and tables; two graphs captured from one pool of memory."""
    cs = caches((64, 16, 2, 64), 2, seed=5)
    src = torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV)
    dst = torch.tensor([4, 5, 6], dtype=torch.int32, device=DEV)
    tab = torch.tensor([[9, 63, 20], [30, 9, 2]], dtype=torch.int32, device=DEV)
    cnt = torch.tensor([3, 2], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.compact_pages([c.clone() for c in cs], tab, cnt)
        ops.copy_pages([c.clone() for c in cs], src, dst)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        ops.copy_pages(cs, src, dst)
    with torch.cuda.graph(g2, pool=g1.pool()):
        new, page_map, m = ops.compact_pages(cs, tab, cnt)
    for k in range(3):
        src.copy_(torch.tensor([7 + k, 8, 9], dtype=torch.int32))
        dst.copy_(torch.tensor([8, 40 + k, 7], dtype=torch.int32))  # a chain
        want = loop_copy(cs, src.tolist(), dst.tolist())
        want, want_tab, want_map, want_m = loop_compact(want, tab.tolist(), cnt.tolist())
        g1.replay()
        g2.replay()
        assert new.tolist() == want_tab and page_map.tolist() == want_map and m.item() == want_m
        assert all(same_bytes(a, b) for a, b in zip(cs, want))
