"""The operators of long-context serving together, as a server uses them: tables for a stretched
context, rotary embedding of views of a packed projection, the scatter into the paged cache,
attention of the chunks, a fork of a sequence by copying its last page, and compaction."""
import pytest
import torch

import decode_workloads as wl
from test_chunk_attention_gpu import check
from test_rotary_gpu import check_rotary

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NHD, NZ = wl.KV_LAYOUT_NHD, wl.KV_LAYOUT_NZ


class Server:
    def __init__(self, ops, layout, hq=28, hkv=4, d=128, page=32, pages=90, rows=3, width=24, interleaved=False):
        self.ops, self.layout, self.hq, self.hkv, self.d, self.page = ops, layout, hq, hkv, d, page
        self.interleaved = interleaved
        freq, amp = ops.rotary_frequencies(d, scaling="yarn", factor=4.0, original_positions=256)
        self.cos, self.sin = ops.rotary_tables(freq, 1024, amplitude=amp, dtype=torch.float32)
        shape = (pages, page, hkv, d) if layout == NHD else (pages, hkv * d // 16, page, 16)
        self.kc = torch.full(shape, float("nan"), device=DEV, dtype=torch.float16)
        self.vc = self.kc.clone()
        self.table = torch.full((rows, width), -1, dtype=torch.int32)
        self.len = [0] * rows
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()

    def pages_of(self, b):
        return -(-self.len[b] // self.page)

    def step(self, new):
        """new[b] more tokens for each sequence; the attention's output, checked."""
        slots, pos = [], []
        for b, n in enumerate(new):
            for p in range(self.len[b], self.len[b] + n):
                if p % self.page == 0:
                    self.table[b, p // self.page] = self.free.pop()
                slots.append(int(self.table[b, p // self.page]) * self.page + p % self.page)
                pos.append(p)
            self.len[b] += n
        total, hq, hkv, d = sum(new), self.hq, self.hkv, self.d
        packed = torch.randn(total, (hq + 2 * hkv) * d, device=DEV).half()
        q = packed[:, :hq * d].view(total, hq, d)
        k = packed[:, hq * d:(hq + hkv) * d].view(total, hkv, d)
        v = packed[:, (hq + hkv) * d:].reshape(total, hkv, d).contiguous()
        pos = torch.tensor(pos, dtype=torch.int32, device=DEV)
        rq, rk = self.ops.rotary(q, k, pos, self.cos, self.sin, self.interleaved)
        check_rotary(q, rq, pos, self.cos, self.sin, self.interleaved)
        check_rotary(k, rk, pos, self.cos, self.sin, self.interleaved)
        self.ops.reshape_and_cache(rk, v, self.kc, self.vc, torch.tensor(slots, dtype=torch.int32, device=DEV))
        starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).int().to(DEV)
        s = dict(q=rq, kc=self.kc, vc=self.vc, table=self.table.to(DEV), starts=starts, hkv=hkv, page=self.page,
                 ctx=torch.tensor(self.len, dtype=torch.int32, device=DEV), layout=self.layout)
        out = self.attend(s)
        check(out, s)
        return s, out

    def attend(self, s):
        return self.ops.chunked_paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["starts"])

    def fork(self, src, dst):
        """Sequence dst continues src: full pages are shared, the begun one is copied."""
        n = self.pages_of(src)
        self.table[dst] = self.table[src]
        self.len[dst] = self.len[src]
        if self.len[src] % self.page:
            self.table[dst, n - 1] = self.free.pop()
            pair = [torch.tensor([int(self.table[x, n - 1])], dtype=torch.int32, device=DEV) for x in (src, dst)]
            self.ops.copy_pages([self.kc, self.vc], *pair)


@pytest.mark.parametrize("layout,page,d,interleaved", [(NHD, 32, 128, False), (NZ, 16, 128, True), (NHD, 24, 64, True), (NZ, 32, 64, False)])
def test_prefill_decode_fork_and_compact(ops, cabi, layout, page, d, interleaved):
    sv = Server(ops, layout, page=page, d=d, interleaved=interleaved)
    sv.step([150, 3, 0])           # the first chunk of a prompt beside a short one
    sv.step([101, 1, 0])           # its second chunk, another sequence decodes
    sv.fork(0, 2)
    before = sv.kc.clone()
    s, out = sv.step([1, 1, 1])    # both branches decode
    shared = sv.table[0, :sv.len[0] // page - 1].long().to(DEV)
    assert torch.equal(sv.kc[shared], before[shared])  # the branches wrote into pages of their own
    counts = torch.tensor([sv.pages_of(b) for b in range(3)], dtype=torch.int32, device=DEV)
    table, page_map, live = ops.compact_pages([sv.kc, sv.vc], s["table"], counts)
    used = {int(p) for b in range(3) for p in sv.table[b, :sv.pages_of(b)]}
    assert int(live) == len(used) and int(table.max()) == len(used) - 1
    sv.kc[len(used):], sv.vc[len(used):] = float("nan"), float("nan")  # what compaction freed may be overwritten
    assert torch.equal(sv.attend({**s, "table": table}), out)
    sv.table, sv.free = table.cpu(), list(range(len(used), sv.kc.shape[0]))
    sv.step([2, 40, 1])            # and the server goes on with the new numbers
    assert cabi.pipeline_status() == 0


def test_the_whole_step_in_a_graph(ops):
    """Rotary, scatter and attention captured once and replayed with other inputs, lengths and pages."""
    hq, hkv, d, page, bs = 14, 2, 128, 64, 5
    g = torch.Generator(device=DEV).manual_seed(3)
    freq, amp = ops.rotary_frequencies(d, scaling="bands", factor=8.0, original_positions=512)
    cos, sin = ops.rotary_tables(freq, 2048, amplitude=amp)
    kc = torch.randn(64, page, hkv, d, generator=g, device=DEV).half()
    vc = torch.randn(64, page, hkv, d, generator=g, device=DEV).half()
    x = dict(q=torch.empty(bs, hq, d, device=DEV).half(), k=torch.empty(bs, hkv, d, device=DEV).half(),
             v=torch.empty(bs, hkv, d, device=DEV).half(), pos=torch.empty(bs, dtype=torch.int32, device=DEV),
             slots=torch.empty(bs, dtype=torch.int32, device=DEV), table=torch.empty(bs, 12, dtype=torch.int32, device=DEV),
             starts=torch.arange(bs + 1, dtype=torch.int32, device=DEV))

    def fill(seed):
        h = torch.Generator(device=DEV).manual_seed(seed)
        for n in "qkv":
            x[n].copy_(torch.randn(x[n].shape, generator=h, device=DEV))
        x["table"].copy_(torch.randperm(64, generator=h, device=DEV)[:60].view(bs, 12).int())
        x["pos"].copy_(torch.randint(0, 700, (bs,), generator=h, device=DEV).int())
        at = x["pos"].long()
        x["slots"].copy_((x["table"].gather(1, (at // page)[:, None])[:, 0] * page + at % page).int())

    def step():
        rq, rk = ops.rotary(x["q"], x["k"], x["pos"], cos, sin)
        ops.reshape_and_cache(rk, x["v"], kc, vc, x["slots"])
        return rq, ops.chunked_paged_attention(rq, kc, vc, x["table"], x["pos"] + 1, x["starts"])

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rq, out = step()
    for seed in (1, 2, 3):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        check(out, dict(q=rq, kc=kc, vc=vc, table=x["table"], ctx=x["pos"] + 1, starts=x["starts"], hkv=hkv, page=page, layout=NHD))
        got = out.clone()
        assert torch.equal(step()[1], got)
