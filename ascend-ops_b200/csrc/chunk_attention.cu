// Attention of chunks of new tokens over the paged KV cache: C-ABI entry, the planning kernel and
// the general kernel (any cache layout, head_dim in {32, 64, 128, 256}, any page size and group).
//
//   out[t] = sum_s softmax_s(q[t] . k[s] / sqrt(D)) v[s],  s = 0 .. position(t),
// the softmax in one pass with running maximum and sum (fp32), base 2 with log2(e) folded into the
// scale.  Probabilities are rounded to fp16 for the second product, the type it multiplies; the sums they are divided by
// use the unrounded values.  The rounding moves each by at most 2^-11 of itself (half a step, like the rounding of the
// output itself, and of both signs, so the sum moves by less) as long as it is above 2^-14; a smaller one moves by up to
// 2^-25, and below 2^-25 it is lost, always in one direction.  So the exponents are lifted by 15 here (by 7 in the
// tcgen05 kernel, whose reference may be 2^8 below the maximum): the largest is 2^15, still fp16, and what rounding
// takes from a small one is at most 2^-40 (2^-32) of the largest.  The sums carry the same factor.
//
// Lengths are device data, so the work is planned on the device: a one-CTA launch cuts the batch
// into items (blocks of tokens x heads x ranges of kv tiles), longest ranges of a sequence first,
// and the attention kernel's CTAs draw items from a ticket counter.  A block whose context is long
// against the batch's work per SM is split; the CTA that finishes the last split merges them.
#include "chunk_attention.cuh"
#include "paged_attention_tile.cuh"

#include <cmath>

namespace b200ops {
namespace ca {
namespace {

// ---- plan -----------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

// Per-sequence plan, kept in the workspace behind the prefix array.
struct SeqPlan {
  int splits, row0, counter0;
};

__global__ void __launch_bounds__(kPlanThreads) chunk_attention_plan_kernel(Args a) {
  __shared__ long long sums[32];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x;
  const int heads = a.num_kv_heads * a.head_tiles;
  SeqPlan* plan = reinterpret_cast<SeqPlan*>(a.prefix + a.bs + 1);
  const int run = (a.bs + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * run, a.bs), b1 = min(b0 + run, a.bs);

  // 1. the batch's work in kv tiles, and the longest range an item gets
  long long work = 0, total;
  for (int b = b0; b < b1; ++b) {
    const Seq s = load_seq(a, b);
    if (s.blocks == 0) continue;
    const long long shorter = static_cast<long long>(s.blocks - 1) * a.block_tokens / a.kv_tile / 2;  // mean, causal
    work += s.blocks * max(s.tiles - shorter, 1LL);
  }
  block_prefix(work, sums, &total);
  const long long share = (total * heads + a.target - 1) / a.target;
  const int range = static_cast<int>(max(share, static_cast<long long>(a.min_tiles)));

  // 2. splits per sequence: none for one that has enough blocks by itself, and none past the
  //    workspace (the sums before the limit are those of the unlimited plan, so the kept ones fit)
  auto wanted = [&](const Seq& s) {
    if (s.blocks == 0) return 0;
    const int by_len = (s.tiles + range - 1) / range;
    const int by_blocks = a.target / (s.blocks * heads);
    return max(1, min(by_len, by_blocks));
  };
  long long rows = 0, split_items = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = load_seq(a, b);
    const int k = wanted(s);
    if (k > 1) {
      rows += static_cast<long long>(s.n) * a.group * heads * k;
      split_items += static_cast<long long>(s.blocks) * heads * k;
    }
  }
  long long row0 = block_prefix(rows, sums, &total);
  long long split0 = block_prefix(split_items, sums, &total);
  long long items = 0, counters = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = load_seq(a, b);
    int k = wanted(s);
    if (k > 1) {
      const long long r = static_cast<long long>(s.n) * a.group * heads * k, i = static_cast<long long>(s.blocks) * heads * k;
      const bool fits = row0 + r <= a.max_rows && split0 + i <= a.max_split_items;
      plan[b].row0 = fits ? static_cast<int>(row0) : 0;
      row0 += r;
      split0 += i;
      if (!fits) k = 1;
    }
    plan[b].splits = k;
    items += static_cast<long long>(s.blocks) * heads * k;
    if (k > 1) counters += static_cast<long long>(s.blocks) * heads;
  }
  long long total_items, total_counters;
  long long item0 = block_prefix(items, sums, &total_items);
  long long counter0 = block_prefix(counters, sums, &total_counters);
  for (int b = b0; b < b1; ++b) {
    const Seq s = load_seq(a, b);
    const int k = plan[b].splits;
    a.prefix[b] = static_cast<int>(min(item0, static_cast<long long>(a.max_items)));
    plan[b].counter0 = static_cast<int>(counter0);
    item0 += static_cast<long long>(s.blocks) * heads * k;
    if (k > 1) counter0 += static_cast<long long>(s.blocks) * heads;
  }
  // more items than tokens allow: query_starts overlap (an error the device cannot report); the rest is left out
  const int n_items = static_cast<int>(min(total_items, static_cast<long long>(a.max_items)));
  if (tid == 0) {
    a.prefix[a.bs] = n_items;
    a.header->n_items = n_items;
    a.header->ticket = 0;
  }
  for (int i = tid; i < total_counters && i < a.max_split_items; i += kPlanThreads) a.counters[i] = 0;
  __syncthreads();

  // 3. the items: per sequence the last block (the longest context) first, heads innermost
  for (int i = tid; i < n_items; i += kPlanThreads) {
    int lo = 0, hi = a.bs;  // the last sequence whose items start at or before i
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.prefix[mid] <= i) lo = mid; else hi = mid;
    }
    const Seq s = load_seq(a, lo);
    const SeqPlan p = plan[lo];
    const int rest = i - a.prefix[lo];
    const int head = rest % heads;
    const int bs_ = rest / heads;
    const int split = bs_ % p.splits;
    const int block = s.blocks - 1 - bs_ / p.splits;
    Item it;
    it.q_tok = s.start + block * a.block_tokens;
    it.n_tok = min(a.block_tokens, s.n - block * a.block_tokens);
    it.pos0 = s.len - s.n + block * a.block_tokens;
    it.seq = lo;
    it.head = head;
    const int tiles = (max(min(it.pos0 + it.n_tok, s.len), 0) + a.kv_tile - 1) / a.kv_tile;
    const int cut = p.splits > 1 ? max(1, min(p.splits, (tiles + range - 1) / range)) : 1;
    const int per = max((tiles + cut - 1) / cut, 1);
    it.n_splits = max((tiles + per - 1) / per, 1);  // no split is empty
    it.split = split;
    it.tile0 = min(split * per, tiles);
    it.tile1 = min(it.tile0 + per, tiles);
    const int rows_before = block * a.block_tokens * a.group * p.splits * heads;  // blocks before this one
    it.row0 = p.row0 + rows_before + head * it.n_tok * a.group * p.splits;
    it.counter = p.counter0 + block * heads + head;
    it.pad = 0;
    a.items[i] = it;
  }
}

// ---- general kernel ---------------------------------------------------------------------------
constexpr int kThreads = 128;
constexpr int kRows = 64;
constexpr float kLift = 15.f;  // a row's largest probability is 2^15: the small ones stay away from fp16's subnormals

template <int D>
struct GeneralShape {
  static constexpr int kTile = D == 256 ? 32 : 64;
  static constexpr int kLd = D + 8;  // 16-byte offset per row: ldmatrix without bank conflicts
  static constexpr size_t kSmem = static_cast<size_t>(kRows + 2 * kTile) * kLd * 2 + 3 * D * 4;
};

// Element offset of (page, off, head, d) in either cache layout (d a multiple of 8).
__device__ __forceinline__ size_t kv_offset(const Args& a, int page, int off, int head, int d) {
  if (a.layout == B200OPS_KV_LAYOUT_NHD)
    return ((static_cast<size_t>(page) * a.page_size + off) * a.num_kv_heads + head) * a.head_dim + d;
  const int e = head * a.head_dim + d;
  const size_t chunks = static_cast<size_t>(a.num_kv_heads) * a.head_dim / 16;
  return ((static_cast<size_t>(page) * chunks + (e >> 4)) * a.page_size + off) * 16 + (e & 15);
}

// Takes the non-finite halfs out of `v` (channels d .. d+7 of position t); `special` [3][head_dim].
constexpr int kNever = 0x7fffffff;

__device__ __noinline__ void take_nonfinite(uint4& v, int t, int d, int head_dim, int* special, int* flag) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
  for (int i = 0; i < 8; ++i) {
    const uint32_t h = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
    if ((h & 0x7c00u) != 0x7c00u) continue;
    const int kind = (h & 0x3ffu) ? 2 : ((h & 0x8000u) ? 1 : 0);
    atomicMin(&special[kind * head_dim + d + i], t);
    w[i >> 1] &= ~(0xffffu << (16 * (i & 1)));
    *flag = 1;
  }
  v = make_uint4(w[0], w[1], w[2], w[3]);
}

// What a row at position `pos` adds to channel d for the values taken out.
__device__ __forceinline__ float special_term(const int* special, int head_dim, int d, int pos) {
  float s = 0.f;
  if (special[d] <= pos) s += INFINITY;
  if (special[head_dim + d] <= pos) s -= INFINITY;
  if (special[2 * head_dim + d] <= pos) s = NAN;
  return s;
}

// Four warps, each 16 of the block's 64 rows; K and V tiles go through shared memory, the products
// run on warp-level tensor-core instructions (fp16 in, fp32 out).  The path for shapes the tcgen05
// kernel does not take (head_dim 32 or 256, pages that are not a multiple of 8 tokens, more than 128 query heads per kv
// head); bound by the load latency of its single-buffered tiles: 4096 new tokens at context 16384, 28 heads of 128, take
// 9.3 ms (0.09 PFLOP/s); 2048 at context 8192, 16 heads of 256 on 4, 2.6 ms, 32 heads of 32 on 8, 0.74 ms (0.09, 0.08).
template <int D>
__global__ void __launch_bounds__(kThreads) chunk_attention_general_kernel(Args a) {
  using G = GeneralShape<D>;
  constexpr int kTile = G::kTile, kLd = G::kLd;
  extern __shared__ __align__(16) uint8_t smem[];
  __half* sq = reinterpret_cast<__half*>(smem);
  __half* sk = sq + kRows * kLd;
  __half* sv = sk + kTile * kLd;
  int* special = reinterpret_cast<int*>(sv + kTile * kLd);
  __shared__ int s_ticket, s_special, s_last;
  __shared__ uint32_t s_mask[2];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int full_group = a.num_heads / a.num_kv_heads;
  const int n_items = a.header->n_items;

  while (true) {
    __syncthreads();
    if (tid == 0) s_ticket = atomicAdd(&a.header->ticket, 1);
    __syncthreads();
    if (s_ticket >= n_items) break;
    const Item it = a.items[s_ticket];
    if (it.split >= it.n_splits) continue;
    const int kvh = it.head / a.head_tiles;
    const int first = (it.head - kvh * a.head_tiles) * a.group;  // query heads of this tile
    const int heads_here = min(a.group, full_group - first);
    const int h0 = kvh * full_group + first;
    const int rows = it.n_tok * a.group;
    auto row_ok = [&](int r) { return r < rows && r % a.group < heads_here; };
    auto row_ptr = [&](int r) {
      return (static_cast<size_t>(it.q_tok + r / a.group) * a.num_heads + h0 + r % a.group) * D;
    };

    for (int i = tid; i < kRows * (D / 8); i += kThreads) {
      const int r = i / (D / 8), c = i - r * (D / 8);
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row_ok(r)) v = *reinterpret_cast<const uint4*>(a.q + row_ptr(r) + c * 8);
      *reinterpret_cast<uint4*>(sq + r * kLd + c * 8) = v;
    }
    for (int i = tid; i < 3 * D; i += kThreads) special[i] = kNever;
    if (tid == 0) s_special = 0;
    __syncthreads();

    uint32_t qa[D / 16][4];
    {
      const int r = warp * 16 + (lane & 15), c = (lane >> 4) * 8;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) pa::tile::ldmatrix_x4(qa[ks], static_cast<uint32_t>(__cvta_generic_to_shared(sq + r * kLd + ks * 16 + c)));
    }
    const int r_lo = warp * 16 + g, r_hi = r_lo + 8;
    const int pos_lo = it.pos0 + r_lo / a.group, pos_hi = it.pos0 + r_hi / a.group;
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;
    bool seen_lo = false, seen_hi = false;  // the row sees a key
    const int kv_len = it.pos0 + it.n_tok;
    const int32_t* table = a.block_tables + static_cast<size_t>(it.seq) * a.max_pages_per_seq;

    for (int tile = it.tile0; tile < it.tile1; ++tile) {
      const int t0 = tile * kTile;
      __syncthreads();
      if (tid < 64) {
        bool ok = false;
        if (tid < kTile && t0 + tid < kv_len) {
          const int page = table[(t0 + tid) / a.page_size];
          ok = page >= 0 && page < a.num_pages;
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) s_mask[warp] = mask;
      }
      for (int i = tid; i < kTile * (D / 8); i += kThreads) {
        const int r = i / (D / 8), c = i - r * (D / 8);
        uint4 kv = make_uint4(0, 0, 0, 0), vv = kv;
        if (t0 + r < kv_len) {
          const int page = table[(t0 + r) / a.page_size];
          if (page >= 0 && page < a.num_pages) {
            const size_t off = kv_offset(a, page, (t0 + r) % a.page_size, kvh, c * 8);
            kv = *reinterpret_cast<const uint4*>(a.k_cache + off);
            vv = *reinterpret_cast<const uint4*>(a.v_cache + off);
            if (t0 + r > it.pos0 && any_nonfinite(vv)) take_nonfinite(vv, t0 + r, c * 8, D, special, &s_special);
          }
        }
        *reinterpret_cast<uint4*>(sk + r * kLd + c * 8) = kv;
        *reinterpret_cast<uint4*>(sv + r * kLd + c * 8) = vv;
      }
      __syncthreads();
      if (warp * 16 >= rows) continue;  // a warp without rows only helps to load

      float s[kTile / 8][4];
#pragma unroll
      for (int nb = 0; nb < kTile / 8; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
        for (int nb = 0; nb < kTile / 8; nb += 2) {
          uint32_t kb[4];
          const int r = nb * 8 + ((lane >> 4) << 3) + (lane & 7), c = ks * 16 + ((lane >> 3) & 1) * 8;
          pa::tile::ldmatrix_x4(kb, static_cast<uint32_t>(__cvta_generic_to_shared(sk + r * kLd + c)));
          pa::tile::mma_16816(s[nb], qa[ks], kb[0], kb[1]);
          pa::tile::mma_16816(s[nb + 1], qa[ks], kb[2], kb[3]);
        }
      }
      const uint64_t mask = s_mask[0] | (static_cast<uint64_t>(s_mask[1]) << 32);
      const int lim_lo = pos_lo - t0, lim_hi = pos_hi - t0;  // last visible column
      auto visible = [&](int lim) { return lim < 0 ? 0 : mask & (lim >= 63 ? ~0ull : (2ull << lim) - 1); };
      seen_lo |= visible(lim_lo) != 0;
      seen_hi |= visible(lim_hi) != 0;
      float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
      for (int nb = 0; nb < kTile / 8; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int col = nb * 8 + 2 * t4 + (j & 1);
          const bool see = ((mask >> col) & 1) && col <= (j < 2 ? lim_lo : lim_hi);
          s[nb][j] = see ? s[nb][j] * a.scale_log2 : -INFINITY;
          if (j < 2) mx_lo = fmaxf(mx_lo, s[nb][j]); else mx_hi = fmaxf(mx_hi, s[nb][j]);
        }
#pragma unroll
      for (int x = 1; x <= 2; x <<= 1) {
        mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, x));
        mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, x));
      }
      const float n_lo = fmaxf(m_lo, mx_lo), n_hi = fmaxf(m_hi, mx_hi);
      const float u_lo = n_lo == -INFINITY ? 0.f : n_lo, u_hi = n_hi == -INFINITY ? 0.f : n_hi;
      const float f_lo = exp2f(m_lo - u_lo), f_hi = exp2f(m_hi - u_hi);
      const float z_lo = u_lo - kLift, z_hi = u_hi - kLift;
      m_lo = n_lo;
      m_hi = n_hi;
      l_lo *= f_lo;
      l_hi *= f_hi;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= f_lo;
        o[i][1] *= f_lo;
        o[i][2] *= f_hi;
        o[i][3] *= f_hi;
      }
#pragma unroll
      for (int kb = 0; kb < kTile / 16; ++kb) {  // 16 tokens: the first product's layout is the second one's operand
        uint32_t pf[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = exp2f(s[2 * kb + h][0] - z_lo), p1 = exp2f(s[2 * kb + h][1] - z_lo);
          const float p2 = exp2f(s[2 * kb + h][2] - z_hi), p3 = exp2f(s[2 * kb + h][3] - z_hi);
          l_lo += p0 + p1;
          l_hi += p2 + p3;
          pf[2 * h] = f2_to_h2(p0, p1);
          pf[2 * h + 1] = f2_to_h2(p2, p3);
        }
#pragma unroll
        for (int db = 0; db < D / 16; ++db) {
          uint32_t vb[4];
          const int r = kb * 16 + (((lane >> 3) & 1) << 3) + (lane & 7), c = db * 16 + (lane >> 4) * 8;
          pa::tile::ldmatrix_x4_trans(vb, static_cast<uint32_t>(__cvta_generic_to_shared(sv + r * kLd + c)));
          pa::tile::mma_16816(o[2 * db], pf, vb[0], vb[1]);
          pa::tile::mma_16816(o[2 * db + 1], pf, vb[2], vb[3]);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      l_lo += __shfl_xor_sync(0xffffffffu, l_lo, x);
      l_hi += __shfl_xor_sync(0xffffffffu, l_hi, x);
    }
    if (s_special) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[i][j] += special_term(special, D, i * 8 + 2 * t4 + (j & 1), j < 2 ? pos_lo : pos_hi);
    }
    if (seen_lo) m_lo = fmaxf(m_lo, kLowest);
    if (seen_hi) m_hi = fmaxf(m_hi, kLowest);
    if (it.n_splits == 1) {
      const float i_lo = row_factor(m_lo, l_lo), i_hi = row_factor(m_hi, l_hi);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = half ? r_hi : r_lo;
        if (!row_ok(r)) continue;
        __half* dst = a.out + row_ptr(r);
        const float inv = half ? i_hi : i_lo;
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<uint32_t*>(dst + i * 8 + 2 * t4) = f2_to_h2(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
      }
      continue;
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = half ? r_hi : r_lo;
      if (r >= rows) continue;
      const size_t pr = static_cast<size_t>(it.row0) + static_cast<size_t>(it.split) * rows + r;
      float* dst = a.part_o + pr * D;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<float2*>(dst + i * 8 + 2 * t4) = make_float2(o[i][2 * half], o[i][2 * half + 1]);
      if (t4 == 0) a.part_ml[pr] = half ? make_float2(m_hi, l_hi) : make_float2(m_lo, l_lo);
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) s_last = atomicAdd(&a.counters[it.counter], 1) == it.n_splits - 1;
    __syncthreads();
    if (s_last) {
      __threadfence();
      for (int r = warp; r < rows; r += kThreads / 32)
        if (row_ok(r)) merge_row(a, it.row0, rows, r, it.n_splits, a.out + row_ptr(r), lane);
    }
  }
}

template <int D>
int launch_general_d(const Args& a, cudaStream_t st) {
  auto kern = chunk_attention_general_kernel<D>;
  constexpr int smem = static_cast<int>(GeneralShape<D>::kSmem);
  if (smem > 48 * 1024) B200OPS_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int grid = a.max_items < 3 * sm_count() ? a.max_items : 3 * sm_count();
  B200OPS_CUDA(launch_kernel(kern, dim3(grid), dim3(kThreads), smem, st, a));
  return B200OPS_OK;
}

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// Everything of the plan that follows from the shape.
void plan_shape(Args* a, bool tc) {
  const int group = a->num_heads / a->num_kv_heads;
  if (tc) {  // two score tiles of 128 rows per block
    a->group = group;
    a->head_tiles = 1;
    a->block_tokens = 2 * (128 / group);
    a->kv_tile = 64;
    a->shares = sm_count() < kMaxShares ? sm_count() : kMaxShares;
    a->slot_rows = (a->block_tokens < a->num_tokens ? a->block_tokens : a->num_tokens) * group;
    // two records per stretch, unless no context is long enough to be cut
    const bool cut = a->shares > 1 && static_cast<int64_t>(a->max_pages_per_seq) * a->page_size > 5 * a->kv_tile;
    a->max_rows = cut ? 2 * a->shares * a->slot_rows : 0;
    return;
  } else {
    a->group = group < kRows ? group : kRows;
    a->head_tiles = (group + a->group - 1) / a->group;
    a->block_tokens = kRows / a->group;
    a->kv_tile = a->head_dim == 256 ? 32 : 64;
    a->min_tiles = 8;
    a->target = 3 * sm_count();
  }
  const int64_t heads = static_cast<int64_t>(a->num_kv_heads) * a->head_tiles;
  const int64_t blocks = (a->num_tokens / a->block_tokens + static_cast<int64_t>(a->bs < a->num_tokens ? a->bs : a->num_tokens)) * heads;
  const int64_t cap_tiles = (static_cast<int64_t>(a->max_pages_per_seq) * a->page_size + a->kv_tile - 1) / a->kv_tile;
  const int64_t splits = (cap_tiles + a->min_tiles - 1) / a->min_tiles;
  int64_t split_items = splits > 1 ? 4 * static_cast<int64_t>(a->target) : 0;
  if (split_items > blocks * splits) split_items = blocks * splits;
  int64_t rows = static_cast<int64_t>(a->num_tokens) * heads * a->group * splits;
  const int64_t most = static_cast<int64_t>(a->target) * a->block_tokens * a->group;
  if (rows > most) rows = most;
  if (splits <= 1) rows = 0;
  a->max_split_items = static_cast<int>(split_items);
  a->max_items = static_cast<int>(blocks + split_items);
  a->max_rows = static_cast<int>(rows);
}

// Lays the workspace out from `base` (may be null: only the size is wanted).  Callers align it to 16 bytes, the
// kernels' 32-byte stores need more: the parts begin at the next multiple of 256, and the size has room for that.
size_t lay_out(Args* a, char* base) {
  constexpr size_t kSlack = 256 - 16;
  base = reinterpret_cast<char*>(align256(reinterpret_cast<uintptr_t>(base)));
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char* p = base + off;
    off += align256(bytes);
    return p;
  };
  a->header = reinterpret_cast<Header*>(take(sizeof(Header)));
  if (a->shares > 0) {  // the tcgen05 kernel needs no plan
    a->cuts = take(a->max_rows > 0 ? cut_list_bytes(a->shares) : 0);
    a->part_ml = reinterpret_cast<float2*>(take(static_cast<size_t>(a->max_rows) * sizeof(float2)));
    a->part_o = reinterpret_cast<float*>(take(static_cast<size_t>(a->max_rows) * a->head_dim * sizeof(float)));
    return off + kSlack;
  }
  a->prefix = reinterpret_cast<int*>(take((static_cast<size_t>(a->bs) + 1) * sizeof(int) + static_cast<size_t>(a->bs) * sizeof(SeqPlan)));
  a->counters = reinterpret_cast<int*>(take(static_cast<size_t>(a->max_split_items) * sizeof(int)));
  a->items = reinterpret_cast<Item*>(take(static_cast<size_t>(a->max_items) * sizeof(Item)));
  a->part_ml = reinterpret_cast<float2*>(take(static_cast<size_t>(a->max_rows) * sizeof(float2)));
  a->part_o = reinterpret_cast<float*>(take(static_cast<size_t>(a->max_rows) * a->head_dim * sizeof(float)));
  return off + kSlack;
}

}  // namespace

int launch_plan(const Args& a, cudaStream_t st) {
  B200OPS_CUDA(launch_kernel(chunk_attention_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a));
  return B200OPS_OK;
}

int launch_general(const Args& a, cudaStream_t st) {
  switch (a.head_dim) {
    case 32: return launch_general_d<32>(a, st);
    case 64: return launch_general_d<64>(a, st);
    case 128: return launch_general_d<128>(a, st);
    default: return launch_general_d<256>(a, st);
  }
}

namespace {

int check_shape(int64_t num_tokens, int64_t bs, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                int64_t page_size, int64_t max_pages_per_seq) {
  B200OPS_REQUIRE(num_tokens >= 0 && bs >= 0 && num_heads > 0 && num_kv_heads > 0,
                  "chunked_paged_attention: bad shape tokens=%lld sequences=%lld heads=%lld kv_heads=%lld",
                  (long long)num_tokens, (long long)bs, (long long)num_heads, (long long)num_kv_heads);
  B200OPS_REQUIRE(num_heads % num_kv_heads == 0,
                  "chunked_paged_attention: num_heads %lld is not a multiple of num_kv_heads %lld",
                  (long long)num_heads, (long long)num_kv_heads);
  B200OPS_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256,
                  "chunked_paged_attention: head_dim must be 32, 64, 128 or 256, got %lld", (long long)head_dim);
  B200OPS_REQUIRE(page_size > 0 && max_pages_per_seq > 0,
                  "chunked_paged_attention: bad cache shape page_size=%lld max_pages_per_seq=%lld",
                  (long long)page_size, (long long)max_pages_per_seq);
  // row, item and position numbers are 32-bit on the device
  B200OPS_REQUIRE(bs <= 65535 && num_heads <= 4096 && num_tokens <= (1 << 24) && num_tokens * num_heads <= (1LL << 29) &&
                      page_size <= (1 << 20) && max_pages_per_seq <= (1 << 24) &&
                      max_pages_per_seq * page_size <= 0x3fffffffLL,
                  "chunked_paged_attention: shape too large");
  return B200OPS_OK;
}

Args shape_args(int64_t num_tokens, int64_t bs, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                int64_t page_size, int64_t max_pages_per_seq, bool tc) {
  Args a = {};
  a.num_tokens = (int)num_tokens;
  a.bs = (int)bs;
  a.num_heads = (int)num_heads;
  a.num_kv_heads = (int)num_kv_heads;
  a.head_dim = (int)head_dim;
  a.page_size = (int)page_size;
  a.max_pages_per_seq = (int)max_pages_per_seq;
  plan_shape(&a, tc);
  return a;
}

}  // namespace
}  // namespace ca
}  // namespace b200ops

extern "C" size_t b200ops_chunked_paged_attention_workspace_size(int64_t num_tokens, int64_t bs, int64_t num_heads,
                                                                 int64_t num_kv_heads, int64_t head_dim,
                                                                 int64_t page_size, int64_t max_pages_per_seq) {
  using namespace b200ops;
  if (ca::check_shape(num_tokens, bs, num_heads, num_kv_heads, head_dim, page_size, max_pages_per_seq) != B200OPS_OK ||
      num_tokens == 0 || bs == 0)
    return 0;
  ca::Args a = ca::shape_args(num_tokens, bs, num_heads, num_kv_heads, head_dim, page_size, max_pages_per_seq, false);
  size_t need = ca::lay_out(&a, nullptr);
  if (ca::tc_supported(head_dim, num_heads / num_kv_heads, page_size)) {
    a = ca::shape_args(num_tokens, bs, num_heads, num_kv_heads, head_dim, page_size, max_pages_per_seq, true);
    const size_t tc = ca::lay_out(&a, nullptr);
    if (tc > need) need = tc;  // enough for either kernel: the option may change
  }
  return need;
}

extern "C" int b200ops_chunked_paged_attention(const void* q, const void* key_cache, const void* value_cache,
                                               const int32_t* block_tables, const int32_t* context_lens,
                                               const int32_t* query_starts, void* out, int64_t num_tokens, int64_t bs,
                                               int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                                               int64_t num_pages, int64_t page_size, int64_t max_pages_per_seq,
                                               int layout, void* workspace, size_t workspace_size, void* stream) {
  using namespace b200ops;
  const int rc = ca::check_shape(num_tokens, bs, num_heads, num_kv_heads, head_dim, page_size, max_pages_per_seq);
  if (rc != B200OPS_OK) return rc;
  B200OPS_REQUIRE(num_pages > 0 && num_pages <= 0x7fffffffLL, "chunked_paged_attention: bad cache shape pages=%lld",
                  (long long)num_pages);
  B200OPS_REQUIRE(layout == B200OPS_KV_LAYOUT_NZ || layout == B200OPS_KV_LAYOUT_NHD,
                  "chunked_paged_attention: unknown cache layout %d", layout);
  if (num_tokens == 0 || bs == 0) return B200OPS_OK;
  B200OPS_REQUIRE(q && key_cache && value_cache && block_tables && context_lens && query_starts && out,
                  "chunked_paged_attention: null pointer");
  B200OPS_REQUIRE(aligned16(q) && aligned16(key_cache) && aligned16(value_cache) && aligned16(out),
                  "chunked_paged_attention: pointers must be 16-byte aligned");
  const bool tc = knob(kKnobPaMode, 0) != 2 && ca::tc_supported(head_dim, num_heads / num_kv_heads, page_size);
  ca::Args a = ca::shape_args(num_tokens, bs, num_heads, num_kv_heads, head_dim, page_size, max_pages_per_seq, tc);
  const size_t need = ca::lay_out(&a, static_cast<char*>(workspace));
  if (workspace == nullptr || workspace_size < need)
    return fail(B200OPS_EWORKSPACE, "chunked_paged_attention: workspace of %zu bytes needed, got %zu", need,
                workspace ? workspace_size : (size_t)0);
  B200OPS_REQUIRE(aligned16(workspace), "chunked_paged_attention: the workspace must be 16-byte aligned");
  a.q = static_cast<const __half*>(q);
  a.k_cache = static_cast<const __half*>(key_cache);
  a.v_cache = static_cast<const __half*>(value_cache);
  a.block_tables = block_tables;
  a.context_lens = context_lens;
  a.query_starts = query_starts;
  a.out = static_cast<__half*>(out);
  a.num_pages = (int)num_pages;
  a.layout = layout;
  a.scale_log2 = (1.0f / std::sqrt(static_cast<float>(head_dim))) * 1.44269504088896340736f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (tc) return ca::launch_tc(a, st);
  const int pr = ca::launch_plan(a, st);
  return pr != B200OPS_OK ? pr : ca::launch_general(a, st);
}
