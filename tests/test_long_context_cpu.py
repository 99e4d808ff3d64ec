"""Refusals of the long-context operators, and the host arithmetic of the rotary frequencies: all
before any CUDA call."""
import ctypes
import math

import pytest
import torch

ONE = ctypes.c_void_p(256)  # never dereferenced
NULL = ctypes.c_void_p(None)


def test_rotary_frequencies_host(cabi):
    f, a = cabi.rotary_frequencies(8)
    assert f == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14) and a == 1.0
    f, a = cabi.rotary_frequencies(8, scaling=cabi.ROTARY_LINEAR, factor=4.0)
    assert f == pytest.approx([0.25, 0.025, 0.0025, 0.00025], rel=1e-14)
    f, _ = cabi.rotary_frequencies(8, scaling=cabi.ROTARY_NTK, factor=4.0)
    assert f[0] == 1.0 and f[-1] == pytest.approx(0.001 / 4.0, rel=1e-13)
    f, a = cabi.rotary_frequencies(128, scaling=cabi.ROTARY_YARN, factor=8.0, original_positions=4096)
    plain, _ = cabi.rotary_frequencies(128)
    assert f[0] == plain[0] and f[-1] == pytest.approx(plain[-1] / 8, rel=1e-14)
    assert a == pytest.approx(0.1 * math.log(8) + 1, rel=1e-15)
    assert all(x > y for x, y in zip(f, f[1:]))
    f, a = cabi.rotary_frequencies(128, scaling=cabi.ROTARY_BANDS, factor=8.0, original_positions=8192, high=4.0)
    for x, p in zip(f, plain):
        turns = 8192 * p / (2 * math.pi)
        if turns >= 4:
            assert x == p
        elif turns <= 1:
            assert x == pytest.approx(p / 8, rel=1e-14)
        else:
            assert p / 8 < x < p
    assert a == 1.0


@pytest.mark.parametrize("kw,text", [
    (dict(rotary_dim=7), "even"), (dict(rotary_dim=0), "even"), (dict(rotary_dim=514), "even"),
    (dict(rotary_dim=8, base=1.0), "base"), (dict(rotary_dim=8, base=float("nan")), "base"),
    (dict(rotary_dim=8, base=float("inf")), "base"),
    (dict(rotary_dim=8, scaling=5), "unknown scaling"), (dict(rotary_dim=8, scaling=-1), "unknown scaling"),
    (dict(rotary_dim=8, scaling=1, factor=0.5), "factor"), (dict(rotary_dim=8, scaling=1, factor=float("nan")), "factor"),
    (dict(rotary_dim=2, scaling=2, factor=2.0), "ntk"), (dict(rotary_dim=8, scaling=3, factor=2.0), "original_positions"),
    (dict(rotary_dim=8, scaling=4, factor=2.0, original_positions=64, low=4.0, high=4.0), "low"),
])
def test_rotary_frequencies_refusals(cabi, kw, text):
    with pytest.raises(cabi.B200OpsError, match=text) as e:
        cabi.rotary_frequencies(**kw)
    assert e.value.code == cabi.EINVAL


def test_rotary_refusals(cabi):
    lib = cabi.load()
    f = (ctypes.c_double * 4)(1.0, 0.1, 0.01, float("nan"))
    t = lib.b200ops_rotary_tables
    assert t(f, 4, 1.0, 0, 10, ONE, ONE, 0, NULL) == cabi.EINVAL and "frequency 3" in cabi.last_error()
    assert t(f, 3, float("inf"), 0, 10, ONE, ONE, 0, NULL) == cabi.EINVAL
    assert t(f, 3, 1.0, -1, 10, ONE, ONE, 0, NULL) == cabi.EINVAL
    assert t(f, 3, 1.0, 0, 10, ONE, ONE, 2, NULL) == cabi.EINVAL
    assert t(f, 257, 1.0, 0, 10, ONE, ONE, 0, NULL) == cabi.EINVAL
    assert t(f, 3, 1.0, 0, 10, ONE, NULL, 0, NULL) == cabi.EINVAL
    assert t(f, 3, 1.0, 0, 0, NULL, NULL, 0, NULL) == cabi.OK
    def rot(tokens=2, hq=4, hkv=2, d=64, r=64, qs=256, ks=128, maxpos=16, typ=0, q=ONE):
        return lib.b200ops_rotary(q, ONE, ONE, ONE, ONE, typ, ONE, ONE, tokens, hq, hkv, d, r, qs, ks, maxpos, 0, NULL)
    assert rot(r=63) == cabi.EINVAL and rot(r=66) == cabi.EINVAL and rot(r=0) == cabi.EINVAL
    assert rot(qs=255) == cabi.EINVAL and "strides" in cabi.last_error()
    assert rot(typ=3) == cabi.EINVAL and rot(maxpos=2**31) == cabi.EINVAL and rot(q=NULL) == cabi.EINVAL
    assert rot(tokens=-1) == cabi.EINVAL and rot(tokens=0) == cabi.OK


def test_page_refusals(cabi):
    lib = cabi.load()
    def copy(ptrs=(4096,), pages=4, size=64, pairs=1, src=ONE):
        table = (ctypes.c_void_p * max(len(ptrs), 1))(*ptrs)
        return lib.b200ops_copy_pages(table, len(ptrs), pages, size, src, ONE, pairs, NULL)
    assert copy(ptrs=()) == cabi.EINVAL and copy(ptrs=(0,)) == cabi.EINVAL and copy(pages=0) == cabi.EINVAL
    assert copy(size=0) == cabi.EINVAL and copy(pairs=-1) == cabi.EINVAL and copy(src=NULL) == cabi.EINVAL
    assert copy(ptrs=(4096, 4096)) == cabi.EINVAL and "overlap" in cabi.last_error()
    assert copy(ptrs=(8192, 4096, 8192 + 255)) == cabi.EINVAL
    assert copy(ptrs=tuple(4096 * i for i in range(1, 1026))) == cabi.EINVAL
    assert copy(ptrs=(8192, 4096, 8192 + 256), pairs=0) == cabi.OK
    assert lib.b200ops_compact_pages_workspace_size(0) == 0
    need = lib.b200ops_compact_pages_workspace_size(1000)
    assert need >= 8000
    def compact(pages=1000, seqs=2, width=3, new=8192, ws=ONE, size=need, live=ONE):
        table = (ctypes.c_void_p * 1)(1 << 20)
        return lib.b200ops_compact_pages(table, 1, pages, 64, ONE, ONE, seqs, width, ctypes.c_void_p(new), ONE, live,
                                         ws, size, NULL)
    assert compact(ws=NULL) == cabi.EWORKSPACE and compact(size=need - 1) == cabi.EWORKSPACE
    assert compact(new=256) == cabi.EINVAL and "memory of their own" in cabi.last_error()
    assert compact(live=NULL) == cabi.EINVAL and compact(seqs=-1) == cabi.EINVAL and compact(seqs=1 << 20, width=1 << 20) == cabi.EINVAL
    assert compact(pages=524289) == cabi.EUNSUPPORTED


def test_chunked_attention_refusals(cabi):
    lib = cabi.load()
    size = lib.b200ops_chunked_paged_attention_workspace_size
    need = size(64, 2, 8, 2, 128, 16, 64)
    assert need > 0 and size(0, 2, 8, 2, 128, 16, 64) == 0 and size(64, 2, 8, 3, 128, 16, 64) == 0
    def att(tokens=64, bs=2, hq=8, hkv=2, d=128, pages=100, page=16, width=64, layout=1, ws=ONE, n=need, q=ONE):
        return lib.b200ops_chunked_paged_attention(q, ONE, ONE, ONE, ONE, ONE, ONE, tokens, bs, hq, hkv, d, pages, page,
                                                   width, layout, ws, n, NULL)
    assert att(hkv=3) == cabi.EINVAL and "multiple of num_kv_heads" in cabi.last_error()
    assert att(d=96) == cabi.EINVAL and "head_dim" in cabi.last_error()
    assert att(layout=2) == cabi.EINVAL and att(pages=0) == cabi.EINVAL and att(page=0) == cabi.EINVAL
    assert att(tokens=-1) == cabi.EINVAL and att(bs=70000) == cabi.EINVAL and att(tokens=1 << 25) == cabi.EINVAL
    assert att(q=NULL) == cabi.EINVAL and att(q=ctypes.c_void_p(264)) == cabi.EINVAL
    assert att(ws=NULL) == cabi.EWORKSPACE and att(n=need - 1) == cabi.EWORKSPACE
    assert att(tokens=0) == cabi.OK and att(bs=0) == cabi.OK


def test_python_layer_refusals(ops):
    q, pos = torch.zeros(2, 4, 64).half(), torch.zeros(2, dtype=torch.int32)
    tab = torch.zeros(8, 32).half()
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rotary(q, q, pos, tab, tab)
    with pytest.raises(RuntimeError, match="3D"):
        ops.rotary(q[0], q, pos, tab, tab)
    with pytest.raises(RuntimeError, match="agree"):
        ops.rotary(q, q, pos[:1], tab, tab)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.copy_pages([q], pos, pos)
    with pytest.raises(RuntimeError, match="at least one"):
        ops.copy_pages([], pos, pos)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.compact_pages([q], pos[None], pos[:1])
    with pytest.raises(RuntimeError, match="scaling must be one of"):
        ops.rotary_frequencies(64, scaling="other")
    with pytest.raises(RuntimeError, match="factor"):
        ops.rotary_frequencies(64, scaling="linear", factor=0.0)
    c = torch.zeros(4, 16, 2, 64).half()
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.chunked_paged_attention(q, c, c, pos[None], pos[:1], pos)
    with pytest.raises(RuntimeError, match="4D"):
        ops.chunked_paged_attention(q, c[0], c, pos[None], pos[:1], pos)
    f, a = ops.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,) and a == 1.0
    with pytest.raises(RuntimeError, match="CUDA device"):
        ops.rotary_tables(f, 4, device="cpu")
    with pytest.raises(RuntimeError, match="float64 CPU"):
        ops.rotary_tables(f.float(), 4, device="cuda:0")


def test_workspaces_off_their_alignment_are_refused(cabi):
    lib = cabi.load()
    table = (ctypes.c_void_p * 1)(1 << 20)
    need = lib.b200ops_compact_pages_workspace_size(10)
    assert lib.b200ops_compact_pages(table, 1, 10, 64, ONE, ONE, 2, 3, ctypes.c_void_p(8192), ONE, ONE,
                                     ctypes.c_void_p(4096 + 2), need, NULL) == cabi.EINVAL
    assert "aligned" in cabi.last_error()
    need = lib.b200ops_chunked_paged_attention_workspace_size(64, 2, 8, 2, 128, 16, 64)
    assert lib.b200ops_chunked_paged_attention(ONE, ONE, ONE, ONE, ONE, ONE, ONE, 64, 2, 8, 2, 128, 100, 16, 64, 1,
                                               ctypes.c_void_p(4096 + 8), need, NULL) == cabi.EINVAL
