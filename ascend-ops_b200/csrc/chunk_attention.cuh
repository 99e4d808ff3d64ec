// Shared definitions of the attention of chunks of new tokens over the paged KV cache: the work
// list, the partial records of split contexts and their merge.
//
// Rows.  The query heads that share a kv head are folded into the rows of one matrix: row r of a
// block is (token r / group, head r % group), so a key or value is read once for all of them and a
// block of few tokens still fills the tensor core's rows.  Position of token i of a sequence with
// n new tokens and L in its context: L - n + i; it sees the keys at positions 0 .. L - n + i.
#pragma once

#include "common.cuh"

namespace b200ops {
namespace ca {

// One unit of work: `n_tok` tokens of one sequence, one tile of heads, a range of kv tiles.
struct Item {
  int q_tok;           // first token (row of q and out)
  int n_tok;           // tokens of the block
  int pos0;            // position of the first token in its sequence (negative: it sees nothing)
  int seq;             // row of the block table
  int head;            // kv head * head_tiles + tile of its query heads
  int tile0, tile1;    // kv tiles; none if the block sees no key
  int split, n_splits; // this range among those of the block (split >= n_splits: nothing to do)
  int row0;            // partial rows of the block start here, those of split s at row0 + s * n_tok * group
  int counter;         // index of the block's arrival counter (n_splits > 1)
  int pad;
};

constexpr int kMaxShares = 160;

struct Header {
  int n_items;
  int ticket;  // next item to hand out
};

struct Args {
  const __half* q;
  const __half* k_cache;
  const __half* v_cache;
  const int32_t* block_tables;
  const int32_t* context_lens;
  const int32_t* query_starts;
  __half* out;
  // workspace
  Header* header;
  Item* items;
  int* counters;
  int* prefix;       // [bs + 1] items before each sequence, then the per-sequence plan
  float* part_o;     // [rows, head_dim] un-normalised sums of a split
  float2* part_ml;   // [rows] maximum (in base-2 units) and sum
  int num_tokens, bs, num_heads, num_kv_heads, head_dim;
  int num_pages, page_size, max_pages_per_seq, layout;
  float scale_log2;  // 1/sqrt(head_dim) * log2(e)
  // plan
  int block_tokens;  // tokens per block
  int kv_tile;       // tokens per kv tile
  int group;         // query heads per tile of heads (rows per token)
  int head_tiles;    // tiles of heads per kv head
  int min_tiles;     // a split is at least this many kv tiles
  int target;        // items wanted at least
  int max_items, max_split_items, max_rows;
  // tcgen05 kernel: CTAs, rows of a part's record, the cut units of the call (workspace)
  int shares, slot_rows;
  void* cuts;
};

#ifdef __CUDACC__
struct Seq {
  int start, n, len, blocks, tiles;  // first row, new tokens, context, blocks, kv tiles of the last block
};

__device__ __forceinline__ Seq load_seq(const Args& a, int b) {
  Seq s;
  const int lo = min(max(a.query_starts[b], 0), a.num_tokens), hi = min(max(a.query_starts[b + 1], 0), a.num_tokens);
  s.start = lo;
  s.n = max(hi - lo, 0);
  s.len = min(max(a.context_lens[b], 0), a.max_pages_per_seq * a.page_size);
  s.blocks = (s.n + a.block_tokens - 1) / a.block_tokens;
  s.tiles = (s.len + a.kv_tile - 1) / a.kv_tile;
  return s;
}

// Exclusive prefix sum over the block's threads (whole warps); *total gets the sum.  `sums`: 32 words
// of shared memory.
__device__ __forceinline__ long long block_prefix(long long v, long long* sums, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  __syncthreads();  // `sums` may still be read from the call before
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  const int warps = static_cast<int>(blockDim.x) >> 5;
  long long x = lane < warps ? sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += u;
  }
  *total = __shfl_sync(0xffffffffu, x, 31);
  const long long before = __shfl_sync(0xffffffffu, x, max(warp - 1, 0));
  return incl - v + (warp > 0 ? before : 0);
}

// Non-finite values among hidden keys.  A hidden key's probability is exactly 0, but the matrix
// product still forms 0 * v, which is NaN if v is infinite or NaN.  So the kernels take such values
// out of the V tiles at positions that some row of the block does not see, remember per channel the
// first position that holds +inf, -inf and NaN, and add them to the sums of the rows that do see them.
__device__ __forceinline__ uint32_t nonfinite_bits(const uint4& v) {  // a full exponent carries into the sign's place
  auto carry = [](uint32_t w) { return (w & 0x7c007c00u) + 0x04000400u; };
  return (carry(v.x) | carry(v.y) | carry(v.z) | carry(v.w)) & 0x80008000u;
}
__device__ __forceinline__ bool any_nonfinite(const uint4& v) { return nonfinite_bits(v) != 0; }

// Maximum of a row that sees keys, but none with a score above -inf: its softmax is 0 / 0.  Below any score that finite
// operands can have, so a part with such a key decides; -inf stays the maximum of a row that sees no key.
constexpr float kLowest = -1e38f;

// What a row's sums are multiplied with: sum 0 and nothing seen: zeros; a NaN sum stays NaN.
__device__ __forceinline__ float row_factor(float m, float l) { return l == 0.f ? (m == -INFINITY ? 0.f : NAN) : 1.0f / l; }

// Merges the splits of one row (one warp) and stores the fp16 row.  The records were written by
// other SMs of the same launch: ld.global.cg.  A part whose weight underflows is added like any other: if it
// holds an infinity or a NaN, the result must not be finite.
__device__ __forceinline__ void merge_row(const Args& a, int row0, int rows, int r, int n_splits, __half* out, int lane) {
  const float2* ml = a.part_ml + row0 + r;
  float m = -INFINITY;
  for (int s = lane; s < n_splits; s += 32) m = fmaxf(m, __ldcg(&ml[static_cast<size_t>(s) * rows].x));
  m = warp_max(m);
  const float m_use = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int s = lane; s < n_splits; s += 32) {
    const float2 v = __ldcg(&ml[static_cast<size_t>(s) * rows]);
    l += v.y * exp2f(v.x - m_use);
  }
  l = warp_sum(l);
  const float inv = row_factor(m, l);
  const int per = a.head_dim >> 5;  // channels lane, lane + 32, ...
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  for (int s = 0; s < n_splits; ++s) {
    const float w = exp2f(__ldcg(&ml[static_cast<size_t>(s) * rows].x) - m_use);
    const float* o = a.part_o + (static_cast<size_t>(row0) + static_cast<size_t>(s) * rows + r) * a.head_dim;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < per) acc[i] = fmaf(w, __ldcg(o + lane + 32 * i), acc[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < per) out[lane + 32 * i] = __float2half_rn(acc[i] * inv);
}
#endif

int launch_plan(const Args& a, cudaStream_t st);
int launch_general(const Args& a, cudaStream_t st);
bool tc_supported(int64_t head_dim, int64_t group, int64_t page_size);
int launch_tc(const Args& a, cudaStream_t st);
size_t cut_list_bytes(int shares);

}  // namespace ca
}  // namespace b200ops
