"""Measured cases of the long-context serving operators: rotary tables and rotary embedding,
attention of chunks of new tokens over the paged KV cache, and copying / compacting the cache's pages.

Each case is a dict of plain values.  `prepare` makes its inputs on the GPU, `run` makes one pass:
in the plain form (elementary torch operations in 32 bits, 64 for angles) or, with `own` set,
through the package's operators.  `exact` restates the definition in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # Attention of new tokens over the cache.  The smallest call: four sequences in single-token
        # decode with contexts of a few hundred tokens, where latency counts.
        dict(name="attn_one_token", op="attn", heads=28, kv_heads=4, dim=128, page=128, layout="NHD",
             seqs=4, mix="decode", chunk=1, min_ctx=300, max_ctx=1500, lens_seed=11),
        # One step of a server that mixes prefill chunks with decoding: the 64-sequence decode batch
        # (contexts 512 to 8192), four of whose sequences are prompts being read 512 tokens at a time.
        dict(name="attn_mixed_batch", op="attn", heads=28, kv_heads=4, dim=128, page=128, layout="NHD",
             seqs=64, mix="mixed", chunk=512, min_ctx=512, max_ctx=8192, lens_seed=3),
        # A long prompt read in chunks of 4096 tokens: its last chunk, 16384 tokens deep.
        dict(name="attn_long_chunk", op="attn", heads=28, kv_heads=4, dim=128, page=128, layout="NHD",
             seqs=1, mix="chunk", chunk=4096, min_ctx=16384, max_ctx=16384, lens_seed=5),
        # Ragged prompts of odd lengths with heads of 64 channels over pages of 16 tokens.
        dict(name="attn_ragged_d64", op="attn", heads=32, kv_heads=8, dim=64, page=16, layout="NHD",
             seqs=24, mix="ragged", chunk=700, min_ctx=1, max_ctx=3700, lens_seed=7),
        # Rotary embedding of one decode step of 64 sequences (the whole head, half-split, fp16 tables).
        dict(name="rotary_decode", op="rotary", tokens=64, heads=28, kv_heads=4, dim=128, rotary_dim=128,
             interleaved=False, f32_tables=False, max_pos=16385),
        # Rotary embedding of a long prefill: half of each head, interleaved pairs, fp32 tables.
        dict(name="rotary_prefill", op="rotary", tokens=16384, heads=32, kv_heads=8, dim=128, rotary_dim=64,
             interleaved=True, f32_tables=True, max_pos=131072),
        # Tables of a short window, unscaled (what a model is loaded with).
        dict(name="tables_window", op="tables", positions=4097, rotary_dim=128, scaling="none", factor=1.0,
             original=4096, f32=False),
        # Tables of a context stretched eightfold to 262144 positions.
        dict(name="tables_long", op="tables", positions=262144, rotary_dim=128, scaling="yarn", factor=8.0,
             original=32768, f32=True),
        # A few sequences of one layer get their own copy of a shared last page (copy on write).
        dict(name="copy_few", op="copy", tensors=2, pages=1024, page=128, kv_heads=4, dim=128, pairs=8),
        # A beam step or a prefix duplication over four layers at once.
        dict(name="copy_many", op="copy", tensors=8, pages=2048, page=64, kv_heads=8, dim=128, pairs=600),
        # Closing the holes of a small one-layer cache after a few sequences ended.
        dict(name="compact_small", op="compact", tensors=2, pages=250, page=16, kv_heads=4, dim=128, seqs=30,
             live=0.55, shared=0.1),
        # Defragmenting four layers of a large cache before its upper part is given back.
        dict(name="compact_large", op="compact", tensors=8, pages=4096, page=64, kv_heads=4, dim=128, seqs=96,
             live=0.6, shared=0.1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _pair_cost(case):
    """Score entries (query token, key token) of an attention case."""
    return sum(n * (ctx - n) + n * (n + 1) // 2 for n, ctx in _lengths(case))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "rotary", "tables", "copy", "compact"])
    if op == "attn":
        mix = rng.choice(["decode", "mixed", "chunk", "ragged"])
        group, kv = rng.choice([(1, 8), (2, 4), (3, 4), (4, 8), (5, 2), (7, 4), (8, 4), (8, 1), (16, 2)])
        case = dict(op=op, heads=group * kv, kv_heads=kv, dim=rng.choice([64, 128, 128]),
                    page=rng.choice([16, 32, 64, 128]), layout=rng.choice(["NHD", "NHD", "NHD", "NZ"]), mix=mix,
                    seqs=_log_int(rng, 1, 4 if mix == "chunk" else 96),
                    chunk=1 if mix == "decode" else _log_int(rng, 2, 4096),
                    min_ctx=1, max_ctx=_log_int(rng, 64, 16384), lens_seed=rng.randrange(1 << 30))
        # no dearer than the dearest listed case, and at most 2 GB of cache
        limit = 28 * 128 * (4096 * (16384 - 4096) + 4096 * 4097 // 2)
        while (_pair_cost(case) * case["heads"] * case["dim"] > limit or
               sum(c for _, c in _lengths(case)) * kv * case["dim"] * 4 > 2 << 30):
            case["seqs"] = max(1, case["seqs"] // 2)
            case["chunk"] = max(1, case["chunk"] // 2)
            case["max_ctx"] = max(64, case["max_ctx"] * 3 // 4)
        return case
    if op == "rotary":
        dim = rng.choice([64, 96, 128, 256])
        heads, kv = rng.choice([(28, 4), (32, 8), (8, 1), (5, 5), (40, 10)])
        return dict(op=op, tokens=_log_int(rng, 1, 8192), heads=heads, kv_heads=kv, dim=dim,
                    rotary_dim=rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                    f32_tables=rng.random() < 0.5, max_pos=_log_int(rng, 1024, 131072))
    if op == "tables":
        return dict(op=op, positions=_log_int(rng, 500, 262144), rotary_dim=rng.choice([32, 64, 80, 128]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]),
                    factor=rng.choice([2.0, 4.0, 8.0, 32.0]), original=rng.choice([4096, 8192, 32768]),
                    f32=rng.random() < 0.5)
    if op == "copy":
        pages = _log_int(rng, 64, 2048)
        return dict(op=op, tensors=rng.choice([1, 2, 4, 8]), pages=pages, page=rng.choice([16, 32, 64]),
                    kv_heads=rng.choice([1, 4, 8]), dim=rng.choice([64, 128]),
                    pairs=_log_int(rng, 1, max(2, pages // 4)))
    return dict(op=op, tensors=rng.choice([1, 2, 4, 8]), pages=_log_int(rng, 64, 4096),
                page=rng.choice([16, 32, 64]), kv_heads=rng.choice([1, 2, 4]), dim=rng.choice([64, 128]),
                seqs=_log_int(rng, 1, 96), live=round(rng.uniform(0.1, 0.95), 3),
                shared=round(rng.uniform(0.0, 0.3), 3))


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).half()


def _lengths(case):
    """(new tokens, context with them) of every sequence; they belong to the case, not the seed."""
    rng = random.Random(case["lens_seed"])
    out = []
    for i in range(case["seqs"]):
        mix = case["mix"]
        if mix == "decode" or (mix == "mixed" and i % 16 != 5):
            n = 1
        elif mix == "ragged":
            n = rng.randint(1, case["chunk"])
        else:
            n = case["chunk"]
        ctx = rng.randint(case["min_ctx"], case["max_ctx"])
        out.append((n, max(n, ctx)))
    rng.shuffle(out)
    return out


def _attn_prepare(case, seed):
    gen = _gen(seed)
    lens = _lengths(case)
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    need = [-(-ctx // page) for _, ctx in lens]
    pages = sum(need) + 1 + sum(need) // 8
    shape = (pages, page, kv, dim) if case["layout"] == "NHD" else (pages, kv * dim // 16, page, 16)
    ids = torch.randperm(pages, generator=gen, device=DEV)[:sum(need)].int().cpu()
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    o = 0
    for b, k in enumerate(need):
        table[b, :k] = ids[o:o + k]
        o += k
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    return dict(case=case, lens=lens, q=_randn(gen, starts[-1], case["heads"], dim),
                key_cache=_randn(gen, *shape), value_cache=_randn(gen, *shape), block_tables=table.to(DEV),
                context_lens=torch.tensor([c for _, c in lens], dtype=torch.int32, device=DEV),
                query_starts=torch.tensor(starts, dtype=torch.int32, device=DEV))


def _rotary_prepare(case, seed):
    gen = _gen(seed)
    half = case["rotary_dim"] // 2
    inv = 1e6 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    ang = torch.arange(case["max_pos"], device=DEV, dtype=torch.float64)[:, None] * inv
    dt = torch.float32 if case["f32_tables"] else torch.float16
    pos = torch.randint(0, case["max_pos"], (case["tokens"],), generator=gen, device=DEV, dtype=torch.int32)
    return dict(case=case, q=_randn(gen, case["tokens"], case["heads"], case["dim"]),
                k=_randn(gen, case["tokens"], case["kv_heads"], case["dim"]), position_ids=pos,
                cos=ang.cos().to(dt), sin=ang.sin().to(dt))


def _tables_prepare(case, seed):
    rng = random.Random(seed)
    return dict(case=case, base=math.exp(rng.uniform(math.log(1e4), math.log(5e6))),
                start=rng.randrange(0, 1 << 20))


def _caches(case, gen):
    shape = (case["pages"], case["page"], case["kv_heads"], case["dim"])
    return [_randn(gen, *shape) for _ in range(case["tensors"])]


def _copy_prepare(case, seed):
    gen = _gen(seed)
    order = torch.randperm(case["pages"], generator=gen, device=DEV).int()
    pairs = case["pairs"]
    pick = torch.randint(0, case["pages"] - pairs, (pairs,), generator=gen, device=DEV)
    # a source may be copied several times; destinations are fresh pages
    return dict(case=case, caches=_caches(case, gen), src=order[pairs:][pick].contiguous(),
                dst=order[:pairs].contiguous())


def _compact_prepare(case, seed):
    gen = _gen(seed)
    pages, seqs = case["pages"], case["seqs"]
    rng = random.Random(pages * 1000 + seqs)  # row lengths belong to the case, page numbers to the seed
    live = max(1, int(pages * case["live"]))
    order = torch.randperm(pages, generator=gen, device=DEV)[:live].int().tolist()
    cuts = sorted(rng.randint(0, live) for _ in range(seqs - 1))
    rows = [order[a:b] for a, b in zip([0] + cuts, cuts + [live])]
    for i in range(1, seqs):  # some sequences share the front pages of the one before them (a common prefix)
        if rng.random() < case["shared"]:
            rows[i] = rows[i - 1][:max(1, len(rows[i - 1]) // 2)] + rows[i]
    width = max(len(r) for r in rows) + 3
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
    return dict(case=case, caches=_caches(case, gen), block_tables=table.to(DEV),
                page_counts=torch.tensor([len(r) for r in rows], dtype=torch.int32, device=DEV))


def prepare(case, seed):
    return globals()[f"_{case['op']}_prepare"](case, seed)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _dense(cache, rows, layout, kv, dim):
    """The listed pages of a cache as [kv heads, tokens, channels] in 32 bits."""
    x = cache[rows].float()
    if layout == "NZ":
        x = x.permute(0, 2, 1, 3)
    return x.reshape(-1, kv, dim).permute(1, 0, 2)


def _attn_plain(s):
    case = s["case"]
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // kv
    out = torch.empty_like(s["q"])
    t0 = 0
    for b, (n, ctx) in enumerate(s["lens"]):
        rows = s["block_tables"][b, :-(-ctx // page)].long()
        k = _dense(s["key_cache"], rows, case["layout"], kv, dim)[:, :ctx]
        v = _dense(s["value_cache"], rows, case["layout"], kv, dim)[:, :ctx]
        step = max(1, (1 << 27) // (ctx * group))  # bounds the score matrix
        for a in range(0, n, step):
            e = min(n, a + step)
            q = s["q"][t0 + a:t0 + e].float().reshape(e - a, kv, group, dim).permute(1, 2, 0, 3)
            pos = torch.arange(ctx - n + a, ctx - n + e, device=q.device)
            hide = torch.arange(ctx, device=q.device)[None, :] > pos[:, None]
            for h in range(kv):
                score = (q[h].reshape(-1, dim) @ k[h].t()) * dim ** -0.5
                score = score.reshape(group, e - a, ctx).masked_fill(hide, float("-inf"))
                p = torch.exp(score - score.amax(-1, keepdim=True))
                o = (p.reshape(-1, ctx) @ v[h]).reshape(group, e - a, dim) / p.sum(-1, keepdim=True)
                out[t0 + a:t0 + e, h * group:(h + 1) * group] = o.permute(1, 0, 2).half()
        t0 += n
    return out


def _rotate_plain(x, cos, sin, interleaved):
    half = cos.shape[-1]
    r = x[..., :2 * half].float()
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        rot = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :half], r[..., half:]
        rot = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((rot.half(), x[..., 2 * half:]), -1)


def _rotary_plain(s):
    cos, sin = s["cos"][s["position_ids"].long()].float(), s["sin"][s["position_ids"].long()].float()
    flag = s["case"]["interleaved"]
    return _rotate_plain(s["q"], cos, sin, flag), _rotate_plain(s["k"], cos, sin, flag)


def _tables_plain(s):
    case = s["case"]
    dim, base, factor, original = case["rotary_dim"], s["base"], case["factor"], case["original"]
    j = torch.arange(dim // 2, device=DEV, dtype=torch.float64)
    amplitude = 1.0
    if case["scaling"] == "ntk":
        base = base * factor ** (dim / (dim - 2))
    inv = base ** (-2 * j / dim)
    if case["scaling"] == "linear":
        inv = inv / factor
    elif case["scaling"] == "yarn":
        lo, hi = (dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), dim - 1)
        ramp = ((j - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
        amplitude = 0.1 * math.log(factor) + 1.0
    elif case["scaling"] == "bands":
        low, high = 1.0, 4.0
        keep = ((original * inv / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        inv = inv * keep + inv / factor * (1 - keep)
    pos = torch.arange(s["start"], s["start"] + case["positions"], device=DEV, dtype=torch.float64)
    ang = pos[:, None] * inv
    dt = torch.float32 if case["f32"] else torch.float16
    return (ang.cos() * amplitude).to(dt), (ang.sin() * amplitude).to(dt)


def _copy_plain(s):
    src, dst = s["src"].long(), s["dst"].long()
    for c in s["caches"]:
        c[dst] = c[src]
    return s["caches"]


def _compact_plain(s):
    pages = s["case"]["pages"]
    table, counts = s["block_tables"], s["page_counts"]
    used = torch.arange(table.shape[1], device=DEV)[None] < counts[:, None]
    used &= (table >= 0) & (table < pages)
    live = torch.zeros(pages, dtype=torch.bool, device=DEV)
    live[table[used].long()] = True
    total = live.sum()
    idx = torch.arange(pages, device=DEV)
    src = torch.nonzero(live & (idx >= total)).flatten()
    dst = torch.nonzero(~live & (idx < total)).flatten()
    page_map = torch.where(live, idx, -1)
    page_map[src] = dst
    for c in s["caches"]:
        c[dst] = c[src]
    new = torch.where(used, page_map[table.clamp(0, pages - 1).long()], table).int()
    return s["caches"], new, page_map.int(), total.int().reshape(1)


def _attn_own(s, ops):
    return ops.chunked_paged_attention(s["q"], s["key_cache"], s["value_cache"], s["block_tables"],
                                       s["context_lens"], s["query_starts"])


def _rotary_own(s, ops):
    return ops.rotary(s["q"], s["k"], s["position_ids"], s["cos"], s["sin"], interleaved=s["case"]["interleaved"])


def _tables_own(s, ops):
    case = s["case"]
    freq, amplitude = ops.rotary_frequencies(case["rotary_dim"], base=s["base"], scaling=case["scaling"],
                                             factor=case["factor"], original_positions=case["original"])
    return ops.rotary_tables(freq, case["positions"], amplitude=amplitude, start=s["start"],
                             dtype=torch.float32 if case["f32"] else torch.float16)


def _copy_own(s, ops):
    ops.copy_pages(s["caches"], s["src"], s["dst"])
    return s["caches"]


def _compact_own(s, ops):
    return (s["caches"], *ops.compact_pages(s["caches"], s["block_tables"], s["page_counts"]))


def run(state):
    op = state["case"]["op"]
    if not own:
        return globals()[f"_{op}_plain"](state)
    import sys
    if "ascend-ops_b200" not in sys.path:
        sys.path.insert(0, "ascend-ops_b200")
    import ascend910a_extras.ops as ops
    return globals()[f"_{op}_own"](state, ops)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "attn":
        lens = _lengths(case)
        rows = sum(n for n, _ in lens) * case["heads"] * case["dim"] * 2
        kv = sum(ctx for _, ctx in lens) * case["kv_heads"] * case["dim"] * 2 * 2
        table = 4 * sum(-(-ctx // case["page"]) for _, ctx in lens) + 8 * len(lens)
        return {"bytes": 2 * rows + kv + table, "flops": 4 * case["heads"] * case["dim"] * _pair_cost(case)}
    if case["op"] == "rotary":
        elems = case["tokens"] * (case["heads"] + case["kv_heads"])
        row = case["rotary_dim"] * (4 if case["f32_tables"] else 2)  # one row of cos and of sin
        return {"bytes": elems * case["dim"] * 4 + min(case["tokens"], case["max_pos"]) * row + 4 * case["tokens"],
                "flops": 3 * elems * case["rotary_dim"]}
    if case["op"] == "tables":
        elems = case["positions"] * case["rotary_dim"]
        return {"bytes": elems * (4 if case["f32"] else 2), "flops": 20 * elems}
    one = case["page"] * case["kv_heads"] * case["dim"] * 2 * case["tensors"]
    if case["op"] == "copy":
        # a source copied several times needs one read: the distinct ones expected of `pairs` picks
        pool = case["pages"] - case["pairs"]
        distinct = pool * (1 - (1 - 1 / pool) ** case["pairs"])
        return {"bytes": int(one * (case["pairs"] + distinct)) + 8 * case["pairs"], "flops": 0}
    # live pages above the new end, at random places
    moved = int(case["pages"] * case["live"] * (1 - case["live"]))
    return {"bytes": 2 * one * moved + 4 * case["pages"] + 8 * int(case["pages"] * case["live"]), "flops": 0}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _attn_exact(case, seed):
    s = _attn_prepare(case, seed)
    dim, page, kv = case["dim"], case["page"], case["kv_heads"]
    table, lens = s["block_tables"].cpu().numpy(), s["context_lens"].tolist()
    starts = s["query_starts"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, ctx in enumerate(lens):
        tok = np.arange(ctx)
        where = torch.from_numpy(table[b, tok // page].astype(np.int64) * page + tok % page).to(DEV)
        keys = []
        for cache in (s["key_cache"], s["value_cache"]):
            flat = cache if case["layout"] == "NHD" else cache.transpose(1, 2)
            keys.append(flat.reshape(-1, kv, dim)[where].double())
        new = starts[b + 1] - starts[b]
        for head in range(case["heads"]):
            k, v = (x[:, head * kv // case["heads"]] for x in keys)
            step = max(1, (1 << 26) // ctx)
            for lo in range(0, new, step):
                hi = min(new, lo + step)
                sc = s["q"][starts[b] + lo:starts[b] + hi, head].double() @ k.T / math.sqrt(dim)
                seen = torch.ones(hi - lo, ctx, dtype=torch.bool, device=DEV).tril(ctx - new + lo)
                out[starts[b] + lo:starts[b] + hi, head] = torch.softmax(sc.where(seen, -math.inf), 1) @ v
    return out


def _rotary_exact(case, seed):
    s = _rotary_prepare(case, seed)
    half, dim = case["rotary_dim"] // 2, case["dim"]
    j = torch.arange(half, device=DEV)
    first, second = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + half)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["position_ids"].long()].unsqueeze(1)
    res = []
    for x in (s["q"], s["k"]):
        y = x.double()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        res.append(y)
    return tuple(res)


def _tables_exact(case, seed):
    s = _tables_prepare(case, seed)
    dim, fac, orig = case["rotary_dim"], case["factor"], case["original"]
    base, kind, gain = s["base"], case["scaling"], 1.0
    freqs = []
    for i in range(dim // 2):
        f = base ** (-2.0 * i / dim)
        if kind == "linear":
            f /= fac
        elif kind == "ntk":
            f = (base * fac ** (dim / (dim - 2.0))) ** (-2.0 * i / dim)
        elif kind == "yarn":
            edge = [dim * math.log(orig / (2 * math.pi * t)) / (2 * math.log(base)) for t in (32, 1)]
            a, e = max(0, math.floor(edge[0])), min(dim - 1, math.ceil(edge[1]))
            r = min(1.0, max(0.0, (i - a) / max(e - a, 0.001)))
            f, gain = f * (1 - r) + f / fac * r, 1 + 0.1 * math.log(fac)
        elif kind == "bands":
            turns = orig * f / (2 * math.pi)
            if turns < 1.0:
                f /= fac
            elif turns <= 4.0:
                r = (turns - 1.0) / 3.0
                f = f * r + f / fac * (1 - r)
        freqs.append(f)
    pos = s["start"] + np.arange(case["positions"], dtype=np.float64)
    ang = torch.from_numpy(pos).to(DEV).outer(torch.tensor(freqs, dtype=torch.float64, device=DEV))
    return gain * torch.cos(ang), gain * torch.sin(ang)


def _copy_exact(case, seed):
    s = _copy_prepare(case, seed)
    pairs = list(zip(s["src"].tolist(), s["dst"].tolist()))
    for c in s["caches"]:
        for a, b in pairs:
            c[b].copy_(c[a])
    return s["caches"]


def _compact_exact(case, seed):
    s = _compact_prepare(case, seed)
    pages = case["pages"]
    table, counts = s["block_tables"].tolist(), s["page_counts"].tolist()
    live = sorted({p for row, n in zip(table, counts) for p in row[:n] if 0 <= p < pages})
    taken = set(live)
    holes = [p for p in range(len(live)) if p not in taken]
    where = {p: p for p in live}
    for p, h in zip([p for p in live if p >= len(live)], holes):
        where[p] = h
        for c in s["caches"]:
            c[h].copy_(c[p])
    new = [[where.get(p, p) if i < n else p for i, p in enumerate(row)] for row, n in zip(table, counts)]
    ints = dict(dtype=torch.int32, device=DEV)
    return (s["caches"], torch.tensor(new, **ints), torch.tensor([where.get(p, -1) for p in range(pages)], **ints),
            torch.tensor([len(live)], **ints))


def exact(case, seed):
    return globals()[f"_{case['op']}_exact"](case, seed)
