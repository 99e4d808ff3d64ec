// Attention of chunks of new tokens over the paged KV cache on the 5th-generation tensor cores:
// head_dim 64 or 128, caches of either layout with P a multiple of 8, up to 128 query heads per kv head.
//
// One persistent CTA per SM takes an equal share of the batch's work (below) and computes two 128-row
// score tiles at a time:  S_t = Q_t K^T and O_t += P_t V, t = 0, 1, both accumulators in TMEM (2 x 2 buffers of 64
// columns for S, 2 x D for O; P_t is written back over S_t as fp16 and read from TMEM as the second product's left
// operand).  While the tensor core works on one tile, a warpgroup takes the exponentials of the
// other.  The two tiles are
//   - the two halves of a block of more than 128 rows: both read the same K and V tile; or
//   - for a block of at most 128 rows (decoding, short chunks): the even and the odd kv tiles of its range,
//     two running softmaxes that are merged at the end.
// Roles: warps 0-3 and 4-7 softmax of tile 0 and 1 (a thread owns a row), warps 8 and 9
// issue the MMAs of tile 0 and 1, warp 10 goes through the CTA's work and announces every pair of kv tiles, warp 11
// guards the V tiles (below), warps 12-15 walk the block table and issue the TMA loads.
//
// Online softmax: a row's reference maximum is only raised when the new maximum would make a
// probability larger than 2^8 times that of the reference, so the accumulator in TMEM is rescaled a few times per item
// instead of once per tile.  The reference's own probability is taken as 2^7: the largest is then 2^15, still inside fp16,
// the small ones stay away from its subnormals, and the final division by the sum in fp32 makes up for any factor.
//
// Bounds.  With more than one score tile per block, a step (64 keys for both score tiles) takes about 2050 clocks at D = 128
// (4096 new tokens at context 16384, 28 heads of 128 on 4: 690 steps per SM in 725 us on a cool chip) and about 2200 at
// D = 64 (4096 tokens, 32 heads on 8: 112 steps in 129 us, with the starts of the units).  The tensor core needs 1280 and
// 640 of them, the special-function unit 1024, so neither is the limit, and half the products leave the step as long: it is
// the way of one softmax warp from a tile's scores to the next one's, with two such warps per scheduler to fill each
// other's gaps (issue slots 41 %, special functions 51 %, tensor pipe 60 % busy).  Clock stamps, which lengthen the step to
// 2550, give for either D: masks, maximum and the first half of the exponentials 800, the second half 750, the way of the
// probabilities to TMEM and their barrier 390, the barrier of the next scores 300, their way from TMEM 280.  725 us = 1.16
// PFLOP/s; 850 us = 0.99 PFLOP/s in a row under the power limit, where a large matrix product runs at 1.4.  Keys 64 at a
// time with two score buffers each, because 128 at a time leave TMEM room for one (770 us).
// Single tokens are bound by HBM: 37 contexts of 8192 take 101 us = 6.2 TB/s; a few short ones by a chain of latencies
// (19 us for four of 1300, of which the merge is 3; paged_attention, one launch, has the shorter chain: 14.4).
//
// V tiles: a hidden key has probability 0, but 0 * inf is NaN.  Slots past the context and pages that
// name nothing are filled with zeros (by TMA outside the tensor, by the guard warp inside a box), and
// the non-finite values of keys that some row of the block does not see are taken out and
// accounted for at the end (take_nonfinite).
#include "chunk_attention.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.cuh"

#include <algorithm>
#include <atomic>

namespace b200ops {
namespace ca {
namespace {

constexpr int kThreads = 512;
constexpr int kRows = 128;  // rows of a score tile
constexpr int kKeys = 64;   // keys of a kv tile
constexpr int kMaskRing = 16;
constexpr int kMmaWarp = 8, kPlanWarp = 10, kGuardWarp = 11, kLoadWarp = 12;  // MMA: 8 and 9, one per score tile
constexpr uint32_t kSoftmaxWarps = 8;
constexpr float kLift = 7.f, kWindow = 8.f;  // log2 of the reference's probability, and of what the largest is over it
constexpr int kErrBase = 21;  // 21 loads, 22 MMA, 23 softmax, 24 guard, 25 misaligned shared memory

__device__ int g_ca_status = 0;

// ---- shares of the work -------------------------------------------------------------------
// The batch is a line of units (sequence, kv head, block of tokens), each as long as the keys its
// last token sees plus a constant for its start and end; CTA c of S takes the stretch
// [c, c + 1) * total / S.  Every CTA finds its stretch from the lengths by itself (one pass over the
// sequences, arithmetic inside one), so there is no planning launch and no ticket counter.  A unit
// that a stretch boundary falls into is cut there, at a whole kv tile.  So at most S - 1 units are cut
// whatever the batch, and all CTAs finish together.  The parts of a cut unit are written un-normalised
// and merged by a second launch, which spreads the rows over all SMs (the last part's CTA merging alone
// was measured too: 5 us more per prefill, and far slower where one unit has dozens of parts).
constexpr int kOverheadTokens = 256;
// Length per key of a block of two score tiles and of one.  Alone on the chip the one takes 1.0 us per kv tile, the
// other 0.75 us (bound by HBM, so less beside the first): a mixed batch of 64 sequences took 265 us at 2 : 1,
// 271 us at 3 : 2, 277 us at 5 : 4.  Measured there only (28 heads of 128 on 4, caches [pages, P, Hkv, D]); head dimension
// 64 and the other layout use the same lengths, which cost balance at most, never the result.
constexpr int kTwoTiles = 2, kOneTile = 1;

struct Line {
  long long total, share;
};

__device__ __forceinline__ long long unit_base(const Seq& s) { return max(s.len - s.n, 0) + kOverheadTokens; }
// Only the last block of a sequence can be one of a single score tile.
__device__ __forceinline__ int unit_weight(const Args& a, const Seq& s, int block) {
  return s.n - block * a.block_tokens > a.block_tokens / 2 ? kTwoTiles : kOneTile;
}
__device__ __forceinline__ long long unit_length(const Args& a, const Seq& s, int block) {
  return unit_weight(a, s, block) * (unit_base(s) + static_cast<long long>(a.block_tokens) * (block + 1));
}
// Length of the first m blocks of one head.
__device__ __forceinline__ long long blocks_length(const Args& a, const Seq& s, long long m) {
  if (m <= 0) return 0;
  const long long k = m - 1;  // blocks of two tiles, then one of either kind
  return kTwoTiles * (k * unit_base(s) + a.block_tokens * (k * (k + 1) / 2)) + unit_length(a, s, static_cast<int>(k));
}

struct Unit {
  Seq s;
  int seq, head, block;
  long long at;  // where it starts on the line
  int n_tok, pos0, tiles;
  long long length;
};

__device__ __forceinline__ void set_block(const Args& a, Unit& u) {
  u.n_tok = min(a.block_tokens, u.s.n - u.block * a.block_tokens);
  u.pos0 = u.s.len - u.s.n + u.block * a.block_tokens;
  u.tiles = (max(u.pos0 + u.n_tok, 0) + kKeys - 1) / kKeys;
  u.length = unit_length(a, u.s, u.block);
}

// Tile at which a boundary `x` behind the unit's start cuts it; 0 or `tiles`: it does not.
__device__ __forceinline__ int cut_tile(const Unit& u, long long x, long long share) {
  if (x <= 0) return 0;
  if (x >= u.length) return u.tiles;
  // Short shares (small batches): parts of eight tiles, or the merge costs more than the parts save.
  const bool is_short = share < 4096 * kOneTile;
  const int grain = is_short ? 8 : 1, least = is_short ? 8 : 3;
  // fp32 with each operation rounded by itself: cheaper than a 64-bit division, the same in both
  // kernels, and it never decreases in x
  int k = min(static_cast<int>(__fdiv_rn(__fmul_rn(static_cast<float>(x), static_cast<float>(u.tiles)),
                                         static_cast<float>(u.length))), u.tiles);
  k -= k % grain;
  return k < least ? 0 : (u.tiles - k < least ? u.tiles : k);
}

struct Found {
  int seq;
  long long at;
};

// Whole block: the line, and the sequence that holds position index * share (left in *found by the
// thread that meets it; seq = bs if the position lies behind the end).
__device__ __forceinline__ Line find_share(const Args& a, int shares, long long index, long long* sums, Found* found) {
  const int run = (a.bs + static_cast<int>(blockDim.x) - 1) / static_cast<int>(blockDim.x);
  const int b0 = min(static_cast<int>(threadIdx.x) * run, a.bs), b1 = min(b0 + run, a.bs);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = load_seq(a, b);
    mine += a.num_kv_heads * blocks_length(a, s, s.blocks);
  }
  if (threadIdx.x == 0) found->seq = a.bs;
  Line line;
  long long at = block_prefix(mine, sums, &line.total);
  line.share = max((line.total + shares - 1) / shares, 1LL);
  const long long x = index * line.share;
  if (at <= x && x < at + mine) {
    for (int b = b0; b < b1; ++b) {
      long long len = mine;
      if (run > 1) {
        const Seq s = load_seq(a, b);
        len = a.num_kv_heads * blocks_length(a, s, s.blocks);
      }
      if (x < at + len) {
        found->seq = b;
        found->at = at;
        break;
      }
      at += len;
    }
  }
  __syncthreads();
  return line;
}

// The unit that holds position x of the line, inside sequence f.seq.
__device__ __forceinline__ Unit unit_at(const Args& a, const Found& f, long long x) {
  Unit u;
  u.seq = f.seq;
  u.s = load_seq(a, f.seq);
  const long long per_head = blocks_length(a, u.s, u.s.blocks);
  u.head = min(static_cast<int>(static_cast<float>(x - f.at) / static_cast<float>(per_head)), a.num_kv_heads - 1);
  long long y = x - f.at - u.head * per_head;
  while (y < 0) y += per_head, --u.head;  // the quotient was rounded
  while (y >= per_head) y -= per_head, ++u.head;
  int lo = 0, hi = u.s.blocks;  // the last block that starts at or before y
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (blocks_length(a, u.s, mid) <= y) lo = mid; else hi = mid;
  }
  u.block = lo;
  u.at = f.at + u.head * per_head + blocks_length(a, u.s, lo);
  set_block(a, u);
  return u;
}

// The next unit of the line; false behind the last.
__device__ __forceinline__ bool next_unit(const Args& a, Unit& u) {
  u.at += u.length;
  if (++u.block == u.s.blocks) {
    u.block = 0;
    if (++u.head == a.num_kv_heads) {
      u.head = 0;
      do {
        if (++u.seq >= a.bs) return false;
        u.s = load_seq(a, u.seq);
      } while (u.s.blocks == 0);
    }
  }
  set_block(a, u);
  return true;
}

// What the CTA's roles are told of a unit or its part.
struct Work {
  int q_tok, n_tok, pos0, seq, head;
  int tile0, tile1;
  int part;  // record to write (see part_of); -1: the unit is whole, write the result
  int once;  // the only block of its sequence: its keys are read once
};

// One box of keys of a tile, tile after tile: its page (num_pages: nothing there, TMA fills zeros) and its
// place in it.
struct Walk {
  const int32_t* table;
  int key, end, index, offset, page;
  __device__ __forceinline__ Walk(const Args& a, const Work& it, int box_tokens, int box, bool active) {
    table = a.block_tables + static_cast<size_t>(it.seq) * a.max_pages_per_seq;
    end = active ? min(it.pos0 + it.n_tok, it.tile1 * kKeys) : 0;
    key = it.tile0 * kKeys + box * box_tokens;
    index = key / a.page_size;
    offset = key - index * a.page_size;
    look(a);
  }
  __device__ __forceinline__ void look(const Args& a) {
    page = a.num_pages;
    if (key < end) {
      const int pg = table[index];
      if (pg >= 0 && pg < a.num_pages) page = pg;
    }
  }
  __device__ __forceinline__ void forward(const Args& a) {
    key += kKeys;
    offset += kKeys;
    while (offset >= a.page_size) {
      offset -= a.page_size;
      ++index;
    }
    look(a);
  }
};

// A cut unit, as the merge needs it; left by the CTA that has its first part (n = 0: none).
struct CutUnit {
  int n, q_tok, n_tok, head;
  int parts[kMaxShares];
};

// Record of the part of a cut unit that CTA c has: 2 c + 1 for the unit's first part (the end of c's
// stretch), else 2 c (its start); -1: c has none.
__device__ __forceinline__ int part_of(const Unit& u, int c, long long share) {
  const int lo = cut_tile(u, c * share - u.at, share), hi = cut_tile(u, (c + 1) * share - u.at, share);
  return lo >= hi ? -1 : (lo > 0 ? 2 * c : 2 * c + 1);
}

// Q and, from caches [pages, P, Hkv, D], the kv tiles lie in shared memory as sub-tiles of 64 channels with
// the 128-byte swizzle: a copy brings `box_tokens` keys of a sub-tile.  From caches [pages, Hkv * D / 16, P, 16] a
// copy brings all channels of 8 keys, [D / 16][8 keys][16 halfs] with the 32-byte swizzle: such pieces are the same
// distance apart whatever the page size, as the products' descriptors need (one channel row of 16 keys per copy,
// 32 copies a tile, took 1.5 times as long for a mixed batch on pages of 16).
template <int D, bool NZ>
struct Shape {
  static constexpr int kHalves = D / 64;                    // 64-channel sub-tiles of Q
  static constexpr int kQSub = kRows * 128;                 // [128 rows][64 halfs]
  static constexpr int kQBytes = kHalves * kQSub;
  static constexpr int kPieces = NZ ? 1 : D / 64;           // copies per box of keys
  static constexpr int kGroup = D * 16;                     // NZ: 8 keys
  static constexpr int kSub = kKeys * 128;                  // [64 keys][64 halfs]
  static constexpr int kTileBytes = kKeys * D * 2;          // one K or V tile
  // Byte of the tile at which 16-byte chunk c of key r is.
  __device__ static int chunk(int r, int c) {
    return NZ ? (r >> 3) * kGroup + (c >> 1) * 256 + (r & 7) * 32 + (((c ^ (r >> 2)) & 1) << 4)
              : (c >> 3) * kSub + r * 128 + (((c ^ r) & 7) << 4);
  }
  static constexpr int kPairBytes = 2 * kTileBytes;         // a V tile, then the K tile that goes with it
  static constexpr int kStages = D == 128 ? 5 : 10;         // pairs in the ring
  static constexpr int kQ = 0;
  static constexpr int kRing = 2 * kQBytes;
  static constexpr int kMeta = kRing + kStages * kPairBytes;
};

struct Meta {
  uint64_t item_full[2], item_empty[2];
  uint64_t q_full, q_empty;
  uint64_t pair_full[10], pair_ok[10], pair_empty[10];  // landed; looked over by the guard; used up
  uint64_t s_full[2][2], p_full[2][2];  // [score tile][buffer]
  uint64_t pv_done[2], o_full[2];        // after an item's last but one and last second product
  uint64_t exchange;  // the softmax warps' barrier (bounded, unlike bar.sync)
  uint32_t tmem_base;
  int abort_flag;
  int special_flag[2];
  Work items[2];
  Found found;
  long long sums[32];
  uint32_t valid[kMaskRing];     // per kv tile: bit i = keys 8i .. 8i+7 lie in a page that exists
  float swap[2][kRows];          // per tile and row: maxima, then sums, of a block of one score tile
  uint32_t special[2][128];      // per item slot and channel: packed positions, see guard
};

template <int D>  // the same for both layouts
constexpr size_t smem_bytes() { return Shape<D, false>::kMeta + sizeof(Meta); }
static_assert(smem_bytes<128>() <= 232448 && smem_bytes<64>() <= 232448, "shared memory");

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Pairs of floats in one 64-bit register: one instruction for both.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void split(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float v;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}

// Special positions of one channel: three 10-bit fields (+inf, -inf, NaN), the first position
// minus `base`, 1023 = never.  base = the block's first hidden position, and a block spans at most
// 256 tokens, so offsets fit.
constexpr uint32_t kNoSpecial = 0x3fffffffu;

__device__ __noinline__ void guard_take(uint4& v, uint32_t off, uint32_t* special, int* flag) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
  for (int i = 0; i < 8; ++i) {
    const uint32_t h = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
    if ((h & 0x7c00u) != 0x7c00u) continue;
    const int shift = 10 * ((h & 0x3ffu) ? 2 : ((h & 0x8000u) ? 1 : 0));
    uint32_t seen = special[i];
    while (((seen >> shift) & 1023u) > off) {
      const uint32_t next = (seen & ~(1023u << shift)) | (off << shift);
      const uint32_t was = atomicCAS(&special[i], seen, next);
      if (was == seen) break;
      seen = was;
    }
    w[i >> 1] &= ~(0xffffu << (16 * (i & 1)));
    *flag = 1;
  }
  v = make_uint4(w[0], w[1], w[2], w[3]);
}

// What a row adds to a channel; `seen` = row position - base (negative: sees none of them).
__device__ __forceinline__ float guard_term(uint32_t special, int seen) {
  float s = 0.f;
  if (static_cast<int>(special & 1023u) <= seen) s += INFINITY;
  if (static_cast<int>((special >> 10) & 1023u) <= seen) s -= INFINITY;
  if (static_cast<int>(special >> 20) <= seen) s = NAN;
  return s;
}

// 32 channels of a row.  A thread owns a row, so the lanes of a store lie a row apart: whole 32-byte
// sectors per lane keep the number of store instructions and the traffic to L2 down (16-byte stores
// took 3 us per block).
__device__ __forceinline__ void store_part(float* p, const float (&v)[32]) {
#pragma unroll
  for (int k = 0; k < 32; k += 8) {
    Vec256 w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w.r[i] = __float_as_uint(v[k + i]);
    st256(p + k, w);
  }
}

__device__ __forceinline__ void store_row(__half* p, const float (&v)[32], float f, bool wide) {
  uint32_t h[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) h[k] = f2_to_h2(v[2 * k] * f, v[2 * k + 1] * f);
  if (wide) {
#pragma unroll
    for (int k = 0; k < 16; k += 8) {
      Vec256 w;
#pragma unroll
      for (int i = 0; i < 8; ++i) w.r[i] = h[k + i];
      st256(p + 2 * k, w);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 16; k += 4) *reinterpret_cast<uint4*>(p + 2 * k) = make_uint4(h[k], h[k + 1], h[k + 2], h[k + 3]);
  }
}

template <int D, bool NZ>
__global__ void __launch_bounds__(kThreads, 1)
chunk_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const Args a, const int box_tokens) {
  using Sh = Shape<D, NZ>;
  constexpr int kStages = Sh::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  Meta& sm = *reinterpret_cast<Meta*>(smem + Sh::kMeta);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (ptx::smem_u32(smem) & 1023u) {  // the swizzled tiles need it; never the case without static shared memory
    if (threadIdx.x == 0) atomicCAS(&g_ca_status, 0, kErrBase + 4);
    return;
  }
  pdl_trigger();
  if (warp == kMmaWarp) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        ptx::mbar_init(&sm.item_full[i], 1);
        // and two MMA warps, the guard, the loading warps that have a box
        ptx::mbar_init(&sm.item_empty[i], kSoftmaxWarps + 3 + (kKeys / box_tokens * Sh::kPieces > 1 ? 4 : 2));
        for (int b = 0; b < 2; ++b) {
          ptx::mbar_init(&sm.s_full[i][b], 1);
          ptx::mbar_init(&sm.p_full[i][b], 4);
        }
        ptx::mbar_init(&sm.pv_done[i], 1);
        ptx::mbar_init(&sm.o_full[i], 1);
        sm.special_flag[i] = 0;
      }
      ptx::mbar_init(&sm.q_full, 1);
      ptx::mbar_init(&sm.q_empty, 2);
      for (int i = 0; i < kStages; ++i) {
        ptx::mbar_init(&sm.pair_full[i], 1);
        ptx::mbar_init(&sm.pair_ok[i], 1);
        ptx::mbar_init(&sm.pair_empty[i], 2);
      }
      ptx::mbar_init(&sm.exchange, kSoftmaxWarps);
      sm.abort_flag = 0;
      ptx::fence_barrier_init();
    }
    __syncwarp();
    ptx::tmem_alloc(&sm.tmem_base, 512);
    ptx::tmem_relinquish_alloc_permit();
    ptx::tcgen05_fence_before();
  } else if (warp == kGuardWarp) {
    for (int i = lane; i < 2 * 128; i += 32) sm.special[i >> 7][i & 127] = kNoSpecial;
  } else if (warp == kPlanWarp && lane == 0) {
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
  }
  __syncthreads();
  ptx::tcgen05_fence_after();
  pdl_wait();
  const uint32_t tmem = sm.tmem_base;
  const Line line = find_share(a, gridDim.x, blockIdx.x, sm.sums, &sm.found);

  const int group = a.group;
  const int tile_tokens = a.block_tokens / 2;  // tokens per score tile
  const int slot_rows = a.slot_rows;

  // A wait that runs out (a broken pipeline) is recorded and every later wait of the CTA gives up
  // at once, so that all roles run through to the end.
  bool dead = false;
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (dead) return;
    if (!ptx::mbar_wait(bar, parity, &sm.abort_flag)) {
      dead = true;
      *reinterpret_cast<volatile int*>(&sm.abort_flag) = 1;
      atomicCAS(&g_ca_status, 0, kErrBase + code);
    }
  };

  // Pair p of an item: K tile p and V tile p - ahead, the two that one step of the MMA loop reads (the
  // first `ahead` pairs have no V, the last ones no K).  The pairs of all items go round one ring of stages.
  int stage = 0;
  uint32_t phase = 0;
  auto next_stage = [&]() {
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1u;
    }
  };

  // Items arrive through a two-slot ring.
  int slot = 0;
  uint32_t slot_phase = 0;
  auto next_item = [&](Work& it, int code) {
    wait(&sm.item_full[slot], slot_phase, code);
    it = sm.items[slot];
    return !dead && it.n_tok > 0;
  };
  auto release_item = [&]() {
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(&sm.item_empty[slot]);
    slot ^= 1;
    if (slot == 0) slot_phase ^= 1u;
  };

  if (warp < static_cast<int>(kSoftmaxWarps)) {
    // =============================== softmax ===============================
    // 256 threads x 176 + 256 x 80 = the launch's 512 x 128 registers
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    const int t = warp >> 2;                    // score tile
    const int row = (warp & 3) * 32 + lane;     // row of the tile = TMEM lane
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_col = lanes + t * 2 * kKeys;
    const uint32_t o_col = lanes + 4 * kKeys + t * D;
    uint32_t s_phase = 0, o_phase = 0, x_phase = 0, o_other = 0;  // s_phase: a bit per half
    uint32_t pv_phase = 0;
    uint32_t k_count = 0;  // kv tiles before this item
    const int tok = row / group, head = row - tok * group;
    const float scale = a.scale_log2;
    const bool wide = (reinterpret_cast<uintptr_t>(a.out) & 31u) == 0;
    auto exchange = [&]() {
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sm.exchange);
      wait(&sm.exchange, x_phase, 2);
      x_phase ^= 1u;
    };

    Work it;
    while (next_item(it, 2)) {
      const int n = it.tile1 - it.tile0;
      const bool dual = it.n_tok > tile_tokens;
      const int my_tok = dual ? t * tile_tokens + tok : tok;  // token of the block
      const bool valid = tok < tile_tokens && my_tok < it.n_tok;
      const int pos = it.pos0 + my_tok;
      const int kvh = it.head;
      __half* dst = a.out + (static_cast<size_t>(it.q_tok + my_tok) * a.num_heads + kvh * group + head) * D;
      if (n <= 0) {  // a block that sees no key
        if ((dual || t == 0) && valid)
          for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0, 0, 0, 0);
        release_item();
        continue;
      }
      const int steps = dual ? n : (n + 1 - t) / 2;  // kv tiles of this warpgroup
      float m = -INFINITY, l = 0.f;  // reference maximum (raw scores) and sum
      float limit = -INFINITY;       // scores up to here keep the reference
      uint32_t seen = 0;             // the row sees a key
      const int row_pos = pos - it.tile0 * kKeys;                 // this row's position behind the first key
      const int warp_pos = __shfl_sync(0xffffffffu, row_pos, 0);  // the least of the warp's
      int off = dual ? 0 : t * kKeys;                             // first key of the tile
      auto await_scores = [&](int b) {
        wait(&sm.s_full[t][b], (s_phase >> b) & 1u, 2);
        s_phase ^= 1u << b;
        ptx::tcgen05_fence_after();
      };
      uint32_t ok = 0;  // groups of eight keys of the tile that lie in a page that exists
      // Tile i, whose scores are in s; leaves those of the next tile there.
      auto step = [&](int i, uint32_t (&s)[2][32]) {
        const int b = i & 1;
        if (ok != 0xffu || warp_pos - off < kKeys - 1) {
          const int last_col = row_pos - off;  // last visible key of the tile
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int vis = min(max(last_col + 1 - g * 32, 0), 32);
            // a bit per column: visible by position, and its group of eight keys in a page that exists
            const uint32_t bits = (vis == 32 ? 0xffffffffu : (1u << vis) - 1u) &
                                  ((((ok >> (4 * g)) & 15u) * 0x00204081u & 0x01010101u) * 0xffu);
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!((bits >> c) & 1u)) s[g][c] = __float_as_uint(-INFINITY);
            seen |= bits;
          }
        } else {
          seen = 1;
        }
        off += dual ? kKeys : 2 * kKeys;
        uint32_t p[32];
        const uint64_t scale2 = pair(scale, scale);
        uint64_t sum2[2];
        auto exponentials = [&](int from, int to) {
          const float shift = m == -INFINITY ? 0.f : kLift - m * scale;
          const uint64_t shift2 = pair(shift, shift);
          if (from == 0) sum2[0] = sum2[1] = 0;
#pragma unroll
          for (int c = from; c < to; ++c) {
            const int g = c >> 4, k = 2 * (c & 15);
            const uint64_t x2 = fma2(pair(__uint_as_float(s[g][k]), __uint_as_float(s[g][k + 1])), scale2, shift2);
            float p0, p1;
            split(x2, p0, p1);
            p0 = ex2(p0);
            p1 = ex2(p1);
            sum2[c & 1] = add2(sum2[c & 1], pair(p0, p1));
            p[c] = f2_to_h2(p0, p1);
          }
        };
        // The reference maximum is nearly always still good: the first exponentials are taken with it while
        // the tile's own maximum is being found, and again in the rare case that it was not.
        exponentials(0, 16);
        float mx[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          mx[g] = __uint_as_float(s[g][0]);
#pragma unroll
          for (int c = 2; c < 32; c += 2) mx[g] = max3_nan(mx[g], __uint_as_float(s[g][c]), __uint_as_float(s[g][c - 1]));
        }
        const float top = max3_nan(max3_nan(mx[0], mx[1], __uint_as_float(s[0][31])), __uint_as_float(s[1][31]), mx[0]);
        // (Rows that are nobody's have scores of whatever was in shared memory, NaN included; with them here a warp
        // took 2.5 times as long, and its CTA 1.7 times.)
        const bool raise = valid && !(top <= limit);
        if (__any_sync(0xffffffffu, raise)) {
          float f = 1.f;
          if (raise && !(top < INFINITY)) {
            l = NAN;  // a visible score is +inf or NaN: so is the softmax
          } else if (raise) {
            f = ex2((m - top) * scale);  // from -inf: 0
            m = top;
            limit = top + kWindow / scale;
            l *= f;
          }
          if (i > 0) {
            // The accumulator follows, once the product before this one is in it: the next tile's scores are
            // computed behind that product; behind the last tile, its own barrier tells.
            if (i + 1 < steps)
              wait(&sm.s_full[t][b ^ 1], (s_phase >> (b ^ 1)) & 1u, 2);
            else
              wait(&sm.pv_done[t], pv_phase, 2);
            ptx::tcgen05_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 8) {  // a few columns at a time: the scores stay in registers
              uint32_t o[8];
              ptx::tmem_ld_32x32b_x8(o_col + c, o);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              ptx::tmem_st_32x32b_x8(o_col + c, o);
            }
          }
          exponentials(0, 16);
        }
        const bool more = i + 1 < steps;
        exponentials(16, 32);
        ptx::tmem_st_32x32b_x32(s_col + b * kKeys, p);
        float x, y;
        split(add2(sum2[0], sum2[1]), x, y);
        l += x + y;
        ptx::tmem_st_wait();
        ptx::tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sm.p_full[t][b]);
        // (Taking the next scores before this tile's probabilities are out, to hide the way from TMEM, makes the two
        // products wait for one another: 3 to 5 % more time.)
        if (more) {
          await_scores(b ^ 1);
          ptx::tmem_ld_32x32b_x32(s_col + (b ^ 1) * kKeys, s[0]);
          ptx::tmem_ld_32x32b_x32(s_col + (b ^ 1) * kKeys + 32, s[1]);
          ok = sm.valid[(k_count + off / kKeys) & (kMaskRing - 1)];
        }
        ptx::tmem_ld_wait();
      };
      if (!__any_sync(0xffffffffu, valid)) {  // no row of this warp is anybody's: its P may be anything
        for (int i = 0; i < steps; ++i) {
          await_scores(i & 1);
          if (lane == 0) ptx::mbar_arrive(&sm.p_full[t][i & 1]);
        }
      } else if (steps > 0) {
        uint32_t s[2][32];
        await_scores(0);
        ptx::tmem_ld_32x32b_x32(s_col, s[0]);
        ptx::tmem_ld_32x32b_x32(s_col + 32, s[1]);
        ok = sm.valid[(k_count + off / kKeys) & (kMaskRing - 1)];
        ptx::tmem_ld_wait();
#pragma unroll 1
        for (int i = 0; i < steps; ++i) step(i, s);
      }
      if (seen) m = fmaxf(m, kLowest);
      if (steps > 1) pv_phase ^= 1u;
      k_count += n;

      // ------------------------------ the item's result ------------------------------
      const int base = it.pos0 + 1;  // first hidden position of the block
      uint32_t* special = sm.special[slot];
      // The row's sums are f0 * O_0 + f1 * O_1 over channels [c0, c1): of a block of two score tiles its own
      // accumulator; else the even and the odd kv tiles' accumulators (a warp may read its 32 lanes of
      // either), each warpgroup taking half of the channels after both learned both maxima and sums.
      float f0 = 1.f, f1 = 0.f;
      uint32_t col0 = o_col, col1 = 0;
      int c0 = 0, c1 = D;
      bool both = false;
      if (dual) {
        wait(&sm.o_full[t], o_phase, 2);
        o_phase ^= 1u;
        o_other ^= 1u;
      } else {
        sm.swap[t][row] = m;
        exchange();
        const float m_other = sm.swap[t ^ 1][row];
        const float m_all = fmaxf(m, m_other);
        const float f = m == -INFINITY ? 0.f : ex2((m - m_all) * scale);
        exchange();
        l *= f;
        sm.swap[t][row] = l;
        exchange();
        const float l_other = sm.swap[t ^ 1][row];
        l = t == 0 ? l + l_other : l_other + l;  // the same order on both sides
        const float f_other = m_other == -INFINITY ? 0.f : ex2((m_other - m_all) * scale);
        m = m_all;
        f0 = t == 0 ? f : f_other;
        f1 = t == 0 ? f_other : f;
        both = n > 1;
        wait(&sm.o_full[0], t == 0 ? o_phase : o_other, 2);
        if (both) wait(&sm.o_full[1], t == 0 ? o_other : o_phase, 2);
        if (t == 0 || both) o_phase ^= 1u;
        if (t == 1 || both) o_other ^= 1u;
        col0 = lanes + 4 * kKeys;
        col1 = col0 + D;
        c0 = t * (D / 2);
        c1 = c0 + D / 2;
      }
      ptx::tcgen05_fence_after();
      const bool fix = *reinterpret_cast<volatile int*>(&sm.special_flag[slot]) != 0;  // values were taken out of V
      auto load_sums = [&](int c, float (&v)[32]) {
        uint32_t o0[32];
        ptx::tmem_ld_32x32b_x32(col0 + c, o0);
        if (both) {
          uint32_t o1[32];
          ptx::tmem_ld_32x32b_x32(col1 + c, o1);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = fmaf(__uint_as_float(o1[k]), f1, __uint_as_float(o0[k]) * f0);
        } else {
          ptx::tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(o0[k]) * f0;
        }
        if (fix) {
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] += guard_term(special[c + k], pos - base);
        }
      };
      const size_t record = static_cast<size_t>(it.part) * slot_rows + my_tok * group + head;
      const float inv = row_factor(m, l);
#pragma unroll 1
      for (int c = c0; c < c1; c += 32) {
        float v[32];
        load_sums(c, v);
        if (valid) {
          if (it.part >= 0)
            store_part(a.part_o + record * D + c, v);
          else
            store_row(dst + c, v, inv, wide);
        }
        __syncwarp();  // the next load needs the whole warp
      }
      if (it.part >= 0 && valid && (dual || t == 0)) a.part_ml[record] = make_float2(m == -INFINITY ? m : m * scale, l);
      if (!dual) {
        ptx::tcgen05_fence_before();
        exchange();  // both accumulators have been read: either warpgroup may start the next item
      }
      if (fix) {  // every warp has read the record: clear it for the slot's next item
        exchange();
        for (int i = threadIdx.x; i < D; i += 32 * kSoftmaxWarps) special[i] = kNoSpecial;
        if (threadIdx.x == 0) sm.special_flag[slot] = 0;
      }
      release_item();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == kMmaWarp || warp == kMmaWarp + 1) {
      // =============================== MMA issue ===============================
      constexpr uint32_t idesc_qk = ptx::make_f16_idesc(kRows, kKeys);
      constexpr uint32_t idesc_pv = ptx::make_f16_idesc(kRows, D) | ptx::kIdescBMnMajor;
      // One warp per score tile.  The tensor core takes instructions a few deep only, so whatever a warp does
      // between two groups of products leaves it idle unless the other warp has products for it (one
      // warp for both tiles took 1.5 times as long), and a single warp executes slowly: the loop is kept
      // short -- one wait per pair of tiles, one per half -- and uniform over the warp (lengths broadcast, one
      // elected lane issues), because MMA descriptors come from uniform registers.
      const int t = warp - kMmaWarp;
      const uint32_t v_ring = ptx::smem_u32(smem + Sh::kRing), k_ring = v_ring + Sh::kTileBytes;
      const uint64_t v_desc = NZ ? ptx::make_sw32_desc(v_ring, Sh::kGroup, 256) : ptx::make_sw128_mnmajor_desc(v_ring, Sh::kSub);
      const uint64_t k_desc = NZ ? ptx::make_sw32_desc(k_ring, Sh::kGroup) : ptx::make_sw128_kmajor_desc(k_ring);
      const uint32_t utmem = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t s_tmem = utmem + t * 2 * kKeys, o_tmem = utmem + 4 * kKeys + t * D;
      uint32_t q_phase = 0, p_phase = 0;  // p_phase: a bit per buffer
      Work it;
      while (next_item(it, 1)) {
        const int n = __shfl_sync(0xffffffffu, it.tile1 - it.tile0, 0);
        if (n <= 0) {
          release_item();
          continue;
        }
        const bool dual = __shfl_sync(0xffffffffu, static_cast<int>(it.n_tok > tile_tokens), 0) != 0;
        const int every = dual ? 1 : 2;  // of the kv tiles, this warp has each, or those of its parity
        const int ahead = 2 * every;     // two score buffers
        const uint64_t q_desc = ptx::make_sw128_kmajor_desc(ptx::smem_u32(smem + Sh::kQ)) +
                                (dual ? t * Sh::kQBytes >> 4 : 0);
        wait(&sm.q_full, q_phase, 1);
        q_phase ^= 1u;
        if (!dual && t >= n) {  // no kv tile for this warp, and no use of Q
          if (lane == 0) ptx::mbar_arrive(&sm.q_empty);
          __syncwarp();
        }
        uint32_t b = 0;  // score buffer
        for (int p = 0; p < n + ahead; ++p, next_stage()) {
          wait(&sm.pair_ok[stage], phase, 1);
          if (!dual && (p & 1) != t) {  // the other warp's
            if (lane == 0) ptx::mbar_arrive(&sm.pair_empty[stage]);
            __syncwarp();
            continue;
          }
          // Two tiles' scores are under way at any time: while the softmax works on one, the tensor core adds
          // the one before to the output and computes the one after it.
          if (p >= ahead) {
            wait(&sm.p_full[t][b], (p_phase >> b) & 1u, 1);
            p_phase ^= 1u << b;
          }
          ptx::tcgen05_fence_after();
          if (ptx::elect_one()) {
            if (p >= ahead) {  // O_t += P_t V
              const uint64_t v = v_desc + (stage * Sh::kPairBytes >> 4);
#pragma unroll
              for (int k = 0; k < kKeys / 16; ++k)
                ptx::umma_f16_ts(o_tmem, s_tmem + b * kKeys + k * 8, v + (k * (NZ ? 2 * Sh::kGroup : 2048) >> 4), idesc_pv,
                                 p >= ahead + every || k > 0);
            }
            if (p < n) {  // S_t = Q_t K^T
              const uint64_t k = k_desc + (stage * Sh::kPairBytes >> 4);
#pragma unroll
              for (int ks = 0; ks < D / 16; ++ks)
                ptx::umma_f16(s_tmem + b * kKeys, q_desc + (((ks >> 2) * Sh::kQSub + (ks & 3) * 32) >> 4),
                              k + ((NZ ? ks * 256 : (ks >> 2) * Sh::kSub + (ks & 3) * 32) >> 4), idesc_qk,
                              ks > 0);
              ptx::umma_commit(&sm.s_full[t][b]);
            }
            ptx::umma_commit(&sm.pair_empty[stage]);
            if (p < n && p + every >= n) ptx::umma_commit(&sm.q_empty);
            if (p >= n && p >= ahead) ptx::umma_commit(p + every >= n + ahead ? &sm.o_full[t] : &sm.pv_done[t]);
          }
          __syncwarp();
          b ^= 1u;
        }
        release_item();
      }
    } else if (warp == kPlanWarp) {
      // =============================== the CTA's work ===============================
      uint32_t q_phase = 0, k_count = 0;
      const long long x0 = blockIdx.x * line.share, x1 = x0 + line.share;
      CutUnit* cut = a.max_rows > 0 ? static_cast<CutUnit*>(a.cuts) + blockIdx.x : nullptr;
      bool listed = false;
      Unit u;
      bool more = sm.found.seq < a.bs;
      if (more) u = unit_at(a, sm.found, x0);
      for (; more && u.at < x1 && !dead; more = next_unit(a, u)) {
        Work it;
        it.q_tok = u.s.start + u.block * a.block_tokens;
        it.n_tok = u.n_tok;
        it.pos0 = u.pos0;
        it.seq = u.seq;
        it.head = u.head;
        it.once = u.s.blocks == 1;
        it.tile0 = cut_tile(u, x0 - u.at, line.share);
        it.tile1 = cut_tile(u, x1 - u.at, line.share);
        // a block without keys (zeros) belongs to the stretch that it starts in
        if (u.tiles == 0 ? u.at < x0 : it.tile0 >= it.tile1) continue;
        it.part = it.tile0 == 0 && it.tile1 == u.tiles ? -1 : part_of(u, static_cast<int>(blockIdx.x), line.share);
        wait(&sm.item_empty[slot], slot_phase ^ 1u, 0);
        if (lane == 0) {
          sm.items[slot] = it;
          ptx::mbar_arrive(&sm.item_full[slot]);
        }
        __syncwarp();
        slot ^= 1;
        if (slot == 0) slot_phase ^= 1u;
        const int n = it.tile1 - it.tile0;
        if (n <= 0) continue;
        const bool dual = it.n_tok > tile_tokens;
        const int ahead = dual ? 2 : 4;
        // a lane per box of keys: does its page exist?
        Walk walk(a, it, box_tokens, lane, lane < kKeys / box_tokens);
        // Q: rows (token, head) of this kv head's group
        wait(&sm.q_empty, q_phase ^ 1u, 0);
        q_phase ^= 1u;
        if (!dead && lane == 0) {
          const uint32_t bytes = static_cast<uint32_t>(tile_tokens * group) * 128u * Sh::kHalves;
          ptx::mbar_arrive_expect_tx(&sm.q_full, dual ? 2 * bytes : bytes);
          for (int t = 0; t < (dual ? 2 : 1); ++t)
            for (int h = 0; h < Sh::kHalves; ++h)
              ptx::tma_load_3d(smem + Sh::kQ + t * Sh::kQBytes + h * Sh::kQSub, &map_q, &sm.q_full, h * 64,
                               it.head * group, it.q_tok + t * tile_tokens);
        }
        __syncwarp();
        for (int p = 0; p < n + ahead; ++p, next_stage()) {
          const bool has_k = p < n, has_v = p >= ahead;
          if (has_k) {
            // which keys lie in a page that exists, for the softmax; published by the pair's barrier
            const uint32_t per_box = box_tokens / 8;
            const uint32_t bits = walk.page < a.num_pages ? ((1u << per_box) - 1u) << (lane * per_box) : 0u;
            const uint32_t all = __reduce_or_sync(0xffffffffu, bits);
            if (lane == 0) sm.valid[(k_count + p) & (kMaskRing - 1)] = all;
            walk.forward(a);
          }
          wait(&sm.pair_empty[stage], phase ^ 1u, 0);
          // (bytes may arrive before they are announced: the phase ends with this arrival at the earliest)
          if (!dead && lane == 0) ptx::mbar_arrive_expect_tx(&sm.pair_full[stage], (has_k + has_v) * Sh::kTileBytes);
          __syncwarp();
        }
        k_count += n;
        if (it.tile0 == 0 && it.tile1 < u.tiles) {  // first part of a cut unit: list the parts for the merge
          int n = 0;
          for (int c = blockIdx.x; c * line.share < u.at + u.length; c += 32) {
            const int part = (c + lane) * line.share < u.at + u.length ? part_of(u, c + lane, line.share) : -1;
            const uint32_t has = __ballot_sync(0xffffffffu, part >= 0);
            if (part >= 0) cut->parts[n + __popc(has & ((1u << lane) - 1u))] = part;
            n += __popc(has);
          }
          if (lane == 0) {
            cut->n = n;
            cut->q_tok = it.q_tok;
            cut->n_tok = it.n_tok;
            cut->head = it.head;
          }
          listed = true;
        }
      }
      if (cut != nullptr && !listed && lane == 0) cut->n = 0;
      if (!dead) {  // the end mark
        wait(&sm.item_empty[slot], slot_phase ^ 1u, 0);
        if (lane == 0) {
          sm.items[slot].n_tok = 0;
          ptx::mbar_arrive(&sm.item_full[slot]);
        }
      }
    } else if (warp >= kLoadWarp) {
      // =============================== loads ===============================
      // A warp issues the copies of its lanes one after the other, 58 clocks each whatever their size (and runs
      // the code around them slowly), and small pages make many: hence four warps, two for K and two for V, a lane
      // per copy (with one warp for all, pages of 16 keys took 1.4 times as long).
      const int boxes = kKeys / box_tokens;
      const bool is_v = (warp & 1) != 0;
      const int first = (warp - kLoadWarp) >> 1, box = 2 * lane + first;  // of the tile
      const int my_box = box / Sh::kPieces, my_piece = box - my_box * Sh::kPieces;
      const bool loads = my_box < boxes;
      const CUtensorMap* map = is_v ? &map_v : &map_k;
      uint8_t* ring = smem + Sh::kRing + (is_v ? 0 : Sh::kTileBytes) +
                      (NZ ? my_box * Sh::kGroup : my_piece * Sh::kSub + my_box * box_tokens * 128);
      const uint64_t policy = ptx::l2_evict_first();
      Work it;
      while (first < boxes * Sh::kPieces && next_item(it, 0)) {
        const int n = it.tile1 - it.tile0;
        const int ahead = n <= 0 ? 0 : (it.n_tok > tile_tokens ? 2 : 4);
        Walk walk(a, it, box_tokens, my_box, loads);
        const int c0 = NZ ? 0 : my_piece * 64, c2 = it.head * (D / 16);
        for (int p = 0; p < n + ahead; ++p, next_stage()) {
          // A pair without a tile for this warp is passed over; one with a tile cannot complete without it, so no
          // phase of its barrier is missed.
          if (is_v ? p < ahead : p >= n) continue;
          wait(&sm.pair_empty[stage], phase ^ 1u, 0);
          if (!dead && loads) {
            uint8_t* dst = ring + stage * Sh::kPairBytes;
            const int x1 = NZ ? walk.offset : it.head, x2 = NZ ? c2 : walk.offset;
            // Keys that are read once make room in L2 for those that other blocks read again.
            if (it.once)
              ptx::tma_load_4d_hint(dst, map, &sm.pair_full[stage], c0, x1, x2, walk.page, policy);
            else
              ptx::tma_load_4d(dst, map, &sm.pair_full[stage], c0, x1, x2, walk.page);
          }
          __syncwarp();
          walk.forward(a);
        }
        release_item();
      }
    } else {
      // =============================== V guard ===============================
      Work it;
      while (next_item(it, 3)) {
        const int n = it.tile1 - it.tile0;
        const int ahead = it.n_tok > tile_tokens ? 2 : 4;
        const int kv_len = it.pos0 + it.n_tok;
        uint32_t* special = sm.special[slot];
        for (int p = 0; n > 0 && p < n + ahead; ++p, next_stage()) {
          wait(&sm.pair_full[stage], phase, 3);
          // (a pair without a V tile: nothing lies at or behind hid)
          const int t0 = p < ahead ? -0x40000000 : (it.tile0 + p - ahead) * kKeys;
          uint8_t* tile = smem + Sh::kRing + stage * Sh::kPairBytes;
          // rows behind the context: zeros (whole rows, so the swizzle does not matter)
          const int end = min(max(kv_len - t0, 0), kKeys);
          // rows that some row of the block does not see: no infinities, no NaN
          const int hid = min(max(it.pos0 + 1 - t0, 0), end);
          if (hid < kKeys) {
            // A lane looks after one 16-byte column.  One test per eight chunks: one by one, a tile took 6000 clocks,
            // and blocks of short contexts, nearly all of whose tiles are looked over, waited for it.
            constexpr int kChunks = D / 8, kStep = 32 / kChunks, kAhead = 8;  // loads under way per lane
            const int c = lane % kChunks, mine = lane / kChunks;
            auto at = [&](int r) { return reinterpret_cast<uint4*>(tile + Sh::chunk(r, c)); };
            for (int r0 = hid + mine; r0 < end; r0 += kStep * kAhead) {
              uint4 v[kAhead];
              uint32_t hit = 0;
#pragma unroll
              for (int u = 0; u < kAhead; ++u) v[u] = *at(min(r0 + u * kStep, end - 1));
#pragma unroll
              for (int u = 0; u < kAhead; ++u) hit |= nonfinite_bits(v[u]);
              if (hit != 0) {
#pragma unroll 1
                for (int r = r0; r < min(r0 + kStep * kAhead, end); r += kStep) {
                  uint4 w = *at(r);
                  if (!any_nonfinite(w)) continue;
                  guard_take(w, static_cast<uint32_t>(t0 + r - (it.pos0 + 1)), special + c * 8, &sm.special_flag[slot]);
                  *at(r) = w;
                }
              }
            }
            for (int r = end + mine; r < kKeys; r += kStep) *at(r) = make_uint4(0, 0, 0, 0);
            ptx::fence_proxy_async();
          }
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&sm.pair_ok[stage]);
        }
        release_item();
      }
    }
  }

  // All roles are through; nothing of this CTA is in flight unless a wait ran out, in which case its
  // copies and products get a moment to land before the memory goes away.
  if (dead) {
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 1000000ull) {
    }
  }
  __syncwarp();
  ptx::tcgen05_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    ptx::tcgen05_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// ---- merge of cut units ---------------------------------------------------------------------
constexpr int kMergeThreads = 256;
constexpr int kMergeRows = 2;  // rows that eight lanes take at once: their loads overlap
constexpr int kMergeCtas = 4;  // CTAs per unit at most

// CTA (c, y): a share of the rows of the unit whose first part CTA c of the attention had.  Every row is
// sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over its parts.  Eight lanes take two rows of a part; the four such
// groups of a warp take four parts of the same rows, or two parts of four rows where a unit has no more (one
// part at a time, 16 parts took 12 us more).  The groups' sums are added in a fixed order.  A chain of three
// L2 round trips (the list, the maxima, the sums); bound by reading the records (D + 2 floats per row and part).
template <int D>
__global__ void __launch_bounds__(kMergeThreads) chunk_attention_merge_kernel(const Args a) {
  constexpr int kPer = D / 32;  // times four channels per lane
  pdl_trigger();
  pdl_wait();
  const CutUnit& cut = static_cast<const CutUnit*>(a.cuts)[blockIdx.x];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = cut.n, rows = cut.n_tok * a.group;
  if (n == 0) return;
  const int parts = n > 2 ? 4 : 2, warp_rows = kMergeRows * 4 / parts;
  const int sub = (lane >> 3) & (parts - 1), row = (lane >> 3) / parts * kMergeRows, channel = (lane & 7) * 4;
  const int step = gridDim.y * (kMergeThreads / 32) * warp_rows;
  for (int r_warp = (blockIdx.y * (kMergeThreads / 32) + warp) * warp_rows; r_warp < rows; r_warp += step) {
    const int r0 = r_warp + row;
    float m[kMergeRows], top[kMergeRows], l[kMergeRows], acc[kMergeRows][kPer * 4];
#pragma unroll
    for (int j = 0; j < kMergeRows; ++j) {
      m[j] = -INFINITY;
      l[j] = 0.f;
#pragma unroll
      for (int k = 0; k < kPer * 4; ++k) acc[j][k] = 0.f;
    }
    for (int i = lane & 7; i < n; i += 8) {
      const float2* ml = a.part_ml + static_cast<size_t>(cut.parts[i]) * a.slot_rows;
#pragma unroll
      for (int j = 0; j < kMergeRows; ++j) m[j] = fmaxf(m[j], ml[min(r0 + j, rows - 1)].x);
    }
#pragma unroll
    for (int j = 0; j < kMergeRows; ++j) {
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) m[j] = fmaxf(m[j], __shfl_xor_sync(0xffffffffu, m[j], o));
      top[j] = m[j];
      if (m[j] == -INFINITY) m[j] = 0.f;
    }
    for (int i = sub; i < n; i += parts) {
      const size_t pr = static_cast<size_t>(cut.parts[i]) * a.slot_rows;
#pragma unroll
      for (int j = 0; j < kMergeRows; ++j) {
        const int r = min(r0 + j, rows - 1);
        const float2 ml = a.part_ml[pr + r];
        const float w = exp2f(ml.x - m[j]);
        l[j] += ml.y * w;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const float4 x = *reinterpret_cast<const float4*>(a.part_o + (pr + r) * D + k * 32 + channel);
          const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][4 * k + e] = fmaf(w, v[e], acc[j][4 * k + e]);  // 0 * inf: see merge_row
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kMergeRows; ++j) {
#pragma unroll
      for (int o = 8; o < 32; o <<= 1) {
        if (o >= 8 * parts) break;
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
#pragma unroll
        for (int k = 0; k < kPer * 4; ++k) acc[j][k] += __shfl_xor_sync(0xffffffffu, acc[j][k], o);
      }
      const int r = r0 + j;
      if (r >= rows) continue;
      const float inv = row_factor(top[j], l[j]);
      const int tok = r / a.group;
      __half* dst = a.out + (static_cast<size_t>(cut.q_tok + tok) * a.num_heads + cut.head * a.group + r - tok * a.group) * D + channel;
#pragma unroll
      for (int k = 0; k < kPer; ++k)
        if (k % parts == sub)
          *reinterpret_cast<uint2*>(dst + k * 32) = make_uint2(f2_to_h2(acc[j][4 * k] * inv, acc[j][4 * k + 1] * inv),
                                                               f2_to_h2(acc[j][4 * k + 2] * inv, acc[j][4 * k + 3] * inv));
    }
  }
}

int box_tokens_of(int64_t page_size) {
  for (int b = kKeys; b >= 8; b >>= 1)
    if (page_size % b == 0) return b;
  return 0;
}

template <int D, bool NZ>
int launch_tc_d(const Args& a, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  const uint64_t e = 2;
  const int box = NZ ? 8 : box_tokens_of(a.page_size);  // keys per copy
  {
    const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a.num_heads), static_cast<uint64_t>(a.num_tokens)};
    const uint64_t strides[2] = {D * e, static_cast<uint64_t>(a.num_heads) * D * e};
    const uint32_t b[3] = {64, static_cast<uint32_t>(a.group), static_cast<uint32_t>(a.block_tokens / 2)};
    const int rc = encode_f16_map(&mq, a.q, 3, dims, strides, b, "chunked_paged_attention(q)");
    if (rc != B200OPS_OK) return rc;
  }
  {
    const uint64_t hkv = a.num_kv_heads, page = a.page_size, pages = static_cast<uint64_t>(a.num_pages);
    const uint64_t groups = hkv * D / 16;  // of 16 channels
    const uint64_t dims[2][4] = {{static_cast<uint64_t>(D), hkv, page, pages}, {16, page, groups, pages}};
    const uint64_t strides[2][3] = {{D * e, hkv * D * e, page * hkv * D * e}, {16 * e, page * 16 * e, page * hkv * D * e}};
    const uint32_t rows = static_cast<uint32_t>(box), b[2][4] = {{64, 1, rows, 1}, {16, rows, D / 16, 1}};
    const CUtensorMapSwizzle swizzle = NZ ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_128B;
    int rc = encode_f16_map(&mk, a.k_cache, 4, dims[NZ], strides[NZ], b[NZ], "chunked_paged_attention(key_cache)", swizzle);
    if (rc != B200OPS_OK) return rc;
    rc = encode_f16_map(&mv, a.v_cache, 4, dims[NZ], strides[NZ], b[NZ], "chunked_paged_attention(value_cache)", swizzle);
    if (rc != B200OPS_OK) return rc;
  }
  auto kern = chunk_attention_tc_kernel<D, NZ>;
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  B200OPS_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
    B200OPS_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_bytes<D>())));
    if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
  }
  B200OPS_CUDA(launch_kernel(kern, dim3(a.shares), dim3(kThreads), smem_bytes<D>(), st, mq, mk, mv, a, box));
  if (a.max_rows > 0) {  // some context may be long enough to be cut
    constexpr int kRowsPerCta = kMergeThreads / 32 * 2 * kMergeRows;  // of a unit of two parts
    const int y = std::min((a.slot_rows + kRowsPerCta - 1) / kRowsPerCta, kMergeCtas);
    B200OPS_CUDA(launch_kernel(chunk_attention_merge_kernel<D>, dim3(a.shares, y), dim3(kMergeThreads), 0, st, a));
  }
  return B200OPS_OK;
}

}  // namespace

size_t cut_list_bytes(int shares) { return static_cast<size_t>(shares) * sizeof(CutUnit); }

bool tc_supported(int64_t head_dim, int64_t group, int64_t page_size) {
  return (head_dim == 64 || head_dim == 128) && group <= 128 && page_size % 8 == 0;
}

int launch_tc(const Args& a, cudaStream_t st) {
  if (a.layout == B200OPS_KV_LAYOUT_NZ) return a.head_dim == 64 ? launch_tc_d<64, true>(a, st) : launch_tc_d<128, true>(a, st);
  return a.head_dim == 64 ? launch_tc_d<64, false>(a, st) : launch_tc_d<128, false>(a, st);
}

int status_take() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_ca_status, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_ca_status, &zero, sizeof(int));
  }
  return v;
}

}  // namespace ca
}  // namespace b200ops
