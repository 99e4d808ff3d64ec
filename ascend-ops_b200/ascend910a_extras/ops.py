"""Operator API, identical in names, argument order, defaults and return types to the
reference's ascend910a_extras/ops.py:7-59.  Every function forwards to the torch extension,
which validates, allocates outputs and launches the sm_100a kernel on the current CUDA
stream without synchronising.  `matmul` is the dense NT product of the reference's earlier
single-call interface (_csrc/ffi.cpp:408-442), served by the same GEMM kernels.
"""
import torch

import ascend910a_extras.ascend910a_extras_C as _C


def rope(
    q: torch.Tensor,
    k: torch.Tensor,
    position_ids: torch.Tensor,
    cos_cache: torch.Tensor,
    sin_cache: torch.Tensor,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Half-split rotary embedding of q [B,Hq,D] and k [B,Hkv,D]; returns (out_q, out_k)."""
    out = _C.ops.rope(q, k, position_ids, cos_cache, sin_cache)
    return out[0], out[1]


def swiglu(x: torch.Tensor) -> torch.Tensor:
    """silu(x[:, :d]) * x[:, d:] for x [T, 2d] float16."""
    return _C.ops.swiglu(x)


def grouped_matmul(
    x: torch.Tensor, w: torch.Tensor, group_list: torch.Tensor
) -> torch.Tensor:
    """y[gl[e-1]:gl[e]] = x[gl[e-1]:gl[e]] @ w[e]; w is [E, K, N] with K contiguous."""
    return _C.ops.grouped_matmul(x, w, group_list)


def matmul(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """y = x @ w.T for x [m, k] and w [n, k], both contiguous float16 (_csrc/ffi.cpp:408-442).
    Any m, n, k: with k and n multiples of 64 the product runs on the tensor-core GEMM kernels
    (one group), other shapes on a plain tiled kernel."""
    return _C.ops.matmul(x, w)


def add_rms_norm(
    x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, epsilon: float = 1e-5
) -> tuple[torch.Tensor, torch.Tensor]:
    """Returns (rmsnorm(x + residual) * weight, x + residual)."""
    return _C.ops.add_rms_norm(x, residual, weight, epsilon)


def reshape_and_cache(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_indices: torch.Tensor,
) -> None:
    """Scatter key/value rows into the paged caches in place; value/value_cache may be None."""
    if value is None:
        value = torch.empty(0, device=key.device, dtype=key.dtype)
    if value_cache is None:
        value_cache = torch.empty(0, device=key_cache.device, dtype=key_cache.dtype)
    return _C.ops.reshape_and_cache(key, value, key_cache, value_cache, slot_indices)


def print_info():
    """Print the current device's SM count, memory sizes and nominal bandwidth."""
    device_id = torch.cuda.current_device()
    _C.print_info(device_id)


def paged_attention(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
) -> torch.Tensor:
    """Decode attention of q [B,Hq,D] over the paged KV cache; returns [B,Hq,D]."""
    return _C.ops.paged_attention(q, key_cache, value_cache, block_tables, context_lens)


_ROTARY_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


def rotary_frequencies(
    rotary_dim: int,
    base: float = 10000.0,
    scaling: str = "none",
    factor: float = 1.0,
    original_positions: int = 0,
    low: float | None = None,
    high: float | None = None,
) -> tuple[torch.Tensor, float]:
    """Rotary frequencies, optionally scaled for longer contexts: (float64 CPU [rotary_dim/2],
    amplitude), both for `rotary_tables`.  scaling: "none", "linear", "ntk", "yarn" (ramp between
    `low`=1 and `high`=32 turns over `original_positions`) or "bands" (`low`=1, `high`=4)."""
    if scaling not in _ROTARY_SCALINGS:
        raise RuntimeError(f"rotary_frequencies: scaling must be one of {sorted(_ROTARY_SCALINGS)}, got {scaling!r}")
    low = 1.0 if low is None else low
    high = (4.0 if scaling == "bands" else 32.0) if high is None else high
    return _C.ops.rotary_frequencies(
        rotary_dim, base, _ROTARY_SCALINGS[scaling], factor, original_positions, low, high
    )


def rotary_tables(
    frequencies: torch.Tensor,
    num_positions: int,
    amplitude: float = 1.0,
    start: int = 0,
    dtype: torch.dtype = torch.float16,
    device: torch.device | str | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin) tables [num_positions, len(frequencies)] of positions start, start+1, ... on the
    current CUDA device (or `device`), float16 (what `rope` takes) or float32."""
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    else:
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
    return _C.ops.rotary_tables(frequencies, num_positions, amplitude, start, dtype, device)


def rotary(
    q: torch.Tensor,
    k: torch.Tensor,
    position_ids: torch.Tensor,
    cos_table: torch.Tensor,
    sin_table: torch.Tensor,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotary embedding of q [T,Hq,D] and k [T,Hkv,D] with tables [max_pos, R/2], float16 or
    float32: pairs (j, j+R/2), or (2j, 2j+1) if `interleaved`, of the first R channels; the
    others are copied.  q and k may be views whose tokens are further apart than their heads."""
    return _C.ops.rotary(q, k, position_ids, cos_table, sin_table, interleaved)


def chunked_paged_attention(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    query_starts: torch.Tensor,
) -> torch.Tensor:
    """Causal attention of the sequences' new tokens, q [T,Hq,D], over the paged KV cache that already
    holds them.  Sequence b owns rows query_starts[b]..query_starts[b+1]-1 and has context_lens[b]
    tokens in the cache, the new ones last.  Returns [T,Hq,D]; rows of no sequence are not written."""
    return _C.ops.chunked_paged_attention(q, key_cache, value_cache, block_tables, context_lens, query_starts)


def _cache_list(caches, op: str) -> list[torch.Tensor]:
    if isinstance(caches, torch.Tensor):  # a sequence as well, of its pages
        raise RuntimeError(f"{op}: caches must be a list of tensors, got a tensor")
    return list(caches)


def copy_pages(caches: list[torch.Tensor], src_pages: torch.Tensor, dst_pages: torch.Tensor) -> None:
    """caches[i][dst_pages[j]] = caches[i][src_pages[j]] for j = 0, 1, ... in order, in place; pairs
    that name no page are skipped.  `caches`: contiguous [pages, ...] tensors of any type."""
    return _C.ops.copy_pages(_cache_list(caches, "copy_pages"), src_pages, dst_pages)


def compact_pages(
    caches: list[torch.Tensor], block_tables: torch.Tensor, page_counts: torch.Tensor
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Move the pages named by the first page_counts[b] entries of each row of block_tables to the
    front of every cache, in place.  Returns (new block tables, page_map [pages]: the new number of
    each live page, -1 for the others, num_live [1]).  Every column is looked at: hand over the columns
    in use of a wide table."""
    return _C.ops.compact_pages(_cache_list(caches, "compact_pages"), block_tables, page_counts)
