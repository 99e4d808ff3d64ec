// Attention of chunks of new tokens over the paged KV cache on the 5th-generation tensor cores:
// head_dim 64 or 128, caches [pages, P, Hkv, D] with P a multiple of 8, up to 128 query heads per kv head.
//
// One persistent CTA per SM draws items (chunk_attention.cuh) and works on two 128-row score tiles
// at a time:  S_t = Q_t K^T and O_t += P_t V, t = 0, 1, both accumulators in TMEM (2 x 128 columns for
// S, 2 x D for O; P_t is written back over S_t as fp16 and read from TMEM as the second product's left
// operand).  While the tensor core works on one tile, a warpgroup takes the exponentials of the
// other.  The two tiles are
//   - the two halves of a block of more than 128 rows: both read the same K and V tile; or
//   - for a block of at most 128 rows (decoding, short chunks): the even and the odd kv tiles of its range,
//     two running softmaxes that are merged at the end.
// Roles: warps 0-3 and 4-7 softmax of tile 0 and 1 (a thread owns a row), warp 8 issues the MMAs,
// warp 9 walks the block table and issues the TMA loads, warps 10-11 guard the V tiles (below).
//
// Online softmax: a row's reference maximum is only raised when the new maximum exceeds it by more
// than 2^8 in the exponential, so the accumulator in TMEM is rescaled a few times per item instead of
// once per tile; probabilities are then up to 256, well inside fp16, and the final division
// by the sum in fp32 makes up for any reference.
//
// V tiles: a hidden key has probability 0, but 0 * inf is NaN.  Slots past the context and pages that
// name nothing are filled with zeros (by TMA outside the tensor, by the guard warps inside a box), and
// the non-finite values of keys that some row of the block does not see are taken out and
// accounted for at the end (take_nonfinite).
#include "chunk_attention.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.cuh"

#include <atomic>

namespace b200ops {
namespace ca {
namespace {

constexpr int kThreads = 384;
constexpr int kTile = 128;  // keys per kv tile, rows per score tile
constexpr int kMaskRing = 16;
constexpr int kMmaWarp = 8, kProducerWarp = 9, kGuardWarp = 10;
constexpr uint32_t kSoftmaxWarps = 8;
constexpr int kErrBase = 21;  // 21 producer, 22 MMA, 23 softmax, 24 guard, 25 misaligned shared memory

__device__ int g_ca_status = 0;

template <int D>
struct Shape {
  static constexpr int kHalves = D / 64;                    // 64-channel sub-tiles
  static constexpr int kSubBytes = kTile * 128;             // [128 rows][64 halfs]
  static constexpr int kTileBytes = kHalves * kSubBytes;    // one Q, K or V tile
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr int kQ = 0;
  static constexpr int kRing = 2 * kTileBytes;
  static constexpr int kMeta = kRing + kStages * kTileBytes;
};

struct Meta {
  uint64_t item_full[2], item_empty[2];
  uint64_t q_full, q_empty;
  // A stage holds a K or a V tile in turn.  Each kind has arrival barriers of its own, because the guard
  // warps follow the V tiles alone and a copy may land long after ones issued behind it: with one
  // barrier per stage they could take the tile before theirs for theirs.
  uint64_t k_full[10], v_full[10], kv_empty[10], v_ok[10];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t exchange;  // the softmax warps' barrier (bounded, unlike bar.sync)
  uint32_t tmem_base;
  int abort_flag;
  int last;
  int special_flag[2];
  Item items[2];
  uint32_t valid[kMaskRing];     // per kv tile: bit i = keys 8i .. 8i+7 lie in a page that exists
  float swap[2][kTile];          // per tile and row: maxima, then sums, of a block of one score tile
  uint32_t special[2][128];      // per item slot and channel: packed positions, see guard
};

template <int D>
constexpr size_t smem_bytes() { return Shape<D>::kMeta + sizeof(Meta); }
static_assert(smem_bytes<128>() <= 232448 && smem_bytes<64>() <= 232448, "shared memory");

struct Ring {
  int stage = 0;
  uint32_t phase = 0;
};
template <int kStages>
__device__ __forceinline__ void advance(Ring& r) {
  if (++r.stage == kStages) {
    r.stage = 0;
    r.phase ^= 1u;
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
chunk_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const Args a, const int box_tokens) {
  using Sh = Shape<D>;
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
        ptx::mbar_init(&sm.item_empty[i], kSoftmaxWarps + 3);
        ptx::mbar_init(&sm.s_full[i], 1);
        ptx::mbar_init(&sm.p_full[i], 4);
        ptx::mbar_init(&sm.o_full[i], 1);
        sm.special_flag[i] = 0;
      }
      ptx::mbar_init(&sm.q_full, 1);
      ptx::mbar_init(&sm.q_empty, 1);
      for (int i = 0; i < kStages; ++i) {
        ptx::mbar_init(&sm.k_full[i], 1);
        ptx::mbar_init(&sm.v_full[i], 1);
        ptx::mbar_init(&sm.kv_empty[i], 1);
        ptx::mbar_init(&sm.v_ok[i], 2);
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
  } else if (warp == kProducerWarp && lane == 0) {
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
  }
  __syncthreads();
  ptx::tcgen05_fence_after();
  pdl_wait();
  const uint32_t tmem = sm.tmem_base;

  const int group = a.group;
  const int tile_tokens = a.block_tokens / 2;  // tokens per score tile

  // A wait that runs out (a broken pipeline) is recorded and every later wait of the CTA gives up
  // at once, so that all roles run through to the end.
  bool dead = false;
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (dead) return;
    if (!__all_sync(0xffffffffu, ptx::mbar_wait(bar, parity, &sm.abort_flag))) {  // the warp stays together
      dead = true;
      *reinterpret_cast<volatile int*>(&sm.abort_flag) = 1;
      atomicCAS(&g_ca_status, 0, kErrBase + code);
    }
  };

  // Items arrive through a two-slot ring.
  int slot = 0;
  uint32_t slot_phase = 0;
  auto next_item = [&](Item& it, int code) {
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int t = warp >> 2;                    // score tile
    const int row = (warp & 3) * 32 + lane;     // row of the tile = TMEM lane
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_col = lanes + t * kTile;
    const uint32_t o_col = lanes + 2 * kTile + t * D;
    uint32_t s_phase = 0, o_phase = 0, x_phase = 0, o_other = 0;
    uint32_t k_count = 0;  // kv tiles before this item
    const int tok = row / group, head = row - tok * group;
    const float scale = a.scale_log2;
    auto exchange = [&]() {
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sm.exchange);
      wait(&sm.exchange, x_phase, 2);
      x_phase ^= 1u;
    };

    Item it;
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
      const int my_n = dual ? n : (n + 1 - t) / 2;
      float m = -INFINITY, l = 0.f;  // reference maximum (raw scores) and sum
      for (int j = 0; j < my_n; ++j) {
        const int idx = dual ? j : 2 * j + t;
        const int last_col = pos - (it.tile0 + idx) * kTile;  // last visible key of the tile
        wait(&sm.s_full[t], s_phase, 2);
        s_phase ^= 1u;
        ptx::tcgen05_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) ptx::tmem_ld_32x32b_x32(s_col + i * 32, s[i]);
        const uint32_t ok = sm.valid[(k_count + idx) & (kMaskRing - 1)];
        ptx::tmem_ld_wait();
        if (ok != 0xffffu || __any_sync(0xffffffffu, last_col < kTile - 1)) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const int col = i * 32 + c;
              if (col > last_col || !((ok >> (col >> 3)) & 1u)) s[i][c] = __float_as_uint(-INFINITY);
            }
        }
        float mx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mx[i] = __uint_as_float(s[i][0]);
#pragma unroll
          for (int c = 1; c < 32; ++c) mx[i] = fmaxf(mx[i], __uint_as_float(s[i][c]));
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const bool raise = top > m && (m == -INFINITY || (top - m) * scale > 8.f);
        if (__any_sync(0xffffffffu, raise)) {
          const float f = raise ? ex2((m - top) * scale) : 1.f;  // m = -inf: 0
          if (raise) m = top;
          l *= f;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              ptx::tmem_ld_32x32b_x32(o_col + c, o);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              ptx::tmem_st_32x32b_x32(o_col + c, o);
            }
          }
        }
        const float shift = m == -INFINITY ? 0.f : -m * scale;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t p[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const int i = 2 * h + (c >> 4), k = 2 * (c & 15);
            const float p0 = ex2(fmaf(__uint_as_float(s[i][k]), scale, shift));
            const float p1 = ex2(fmaf(__uint_as_float(s[i][k + 1]), scale, shift));
            sum[c & 1] += p0;
            sum[2 + (c & 1)] += p1;
            p[c] = f2_to_h2(p0, p1);
          }
          ptx::tmem_st_32x32b_x32(s_col + h * 32, p);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        ptx::tmem_st_wait();
        ptx::tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sm.p_full[t]);
      }
      k_count += n;

      // ------------------------------ the item's result ------------------------------
      const int rows = it.n_tok * group;
      const int base = it.pos0 + 1;  // first hidden position of the block
      uint32_t* special = sm.special[slot];
      bool fix;  // some value was taken out of this item's V tiles
      if (dual) {
        wait(&sm.o_full[t], o_phase, 2);
        o_phase ^= 1u;
        o_other ^= 1u;
        ptx::tcgen05_fence_after();
        fix = *reinterpret_cast<volatile int*>(&sm.special_flag[slot]) != 0;
        const float inv = it.n_splits > 1 ? 1.f : (l == 0.f ? 0.f : 1.0f / l);
        const size_t pr = static_cast<size_t>(it.row0) + static_cast<size_t>(it.split) * rows + my_tok * group + head;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          ptx::tmem_ld_32x32b_x32(o_col + c, o);
          ptx::tmem_ld_wait();
          if (valid) {
            float v[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(o[k]);
            if (fix) {
#pragma unroll
              for (int k = 0; k < 32; ++k) v[k] += guard_term(special[c + k], pos - base);
            }
            if (it.n_splits > 1) {
#pragma unroll
              for (int k = 0; k < 32; k += 4)
                *reinterpret_cast<float4*>(a.part_o + pr * D + c + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
            } else {
#pragma unroll
              for (int k = 0; k < 32; k += 8)
                *reinterpret_cast<uint4*>(dst + c + k) =
                    make_uint4(f2_to_h2(v[k] * inv, v[k + 1] * inv), f2_to_h2(v[k + 2] * inv, v[k + 3] * inv),
                               f2_to_h2(v[k + 4] * inv, v[k + 5] * inv), f2_to_h2(v[k + 6] * inv, v[k + 7] * inv));
            }
          }
          __syncwarp();  // the next load needs the whole warp
        }
        if (it.n_splits > 1 && valid) a.part_ml[pr] = make_float2(m == -INFINITY ? m : m * scale, l);
      } else {
        // Even and odd kv tiles: both warpgroups learn both maxima and sums, then each takes half of
        // the channels of both accumulators (a warp may read its 32 lanes of either).
        sm.swap[t][row] = my_n > 0 ? m : -INFINITY;
        exchange();
        const float m_other = sm.swap[t ^ 1][row];
        const float m_all = fmaxf(m, m_other);
        const float f = m == -INFINITY ? 0.f : ex2((m - m_all) * scale);
        exchange();
        sm.swap[t][row] = l * f;
        exchange();
        const float l_all = l * f + sm.swap[t ^ 1][row];
        const float f_other = m_other == -INFINITY ? 0.f : ex2((m_other - m_all) * scale);
        const float f0 = t == 0 ? f : f_other, f1 = t == 0 ? f_other : f;
        wait(&sm.o_full[0], t == 0 ? o_phase : o_other, 2);
        if (n > 1) wait(&sm.o_full[1], t == 0 ? o_other : o_phase, 2);
        if (t == 0) {
          o_phase ^= 1u;
          if (n > 1) o_other ^= 1u;
        } else {
          o_other ^= 1u;
          if (n > 1) o_phase ^= 1u;
        }
        ptx::tcgen05_fence_after();
        fix = *reinterpret_cast<volatile int*>(&sm.special_flag[slot]) != 0;
        const float inv = it.n_splits > 1 ? 1.f : (l_all == 0.f ? 0.f : 1.0f / l_all);
        const size_t pr = static_cast<size_t>(it.row0) + static_cast<size_t>(it.split) * rows + tok * group + head;
#pragma unroll 1
        for (int c = t * (D / 2); c < (t + 1) * (D / 2); c += 32) {
          uint32_t o0[32], o1[32];
          ptx::tmem_ld_32x32b_x32(lanes + 2 * kTile + c, o0);
          if (n > 1) ptx::tmem_ld_32x32b_x32(lanes + 2 * kTile + D + c, o1);
          ptx::tmem_ld_wait();
          if (valid) {
            float v[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              v[k] = __uint_as_float(o0[k]) * f0;
              if (n > 1) v[k] = fmaf(__uint_as_float(o1[k]), f1, v[k]);
            }
            if (fix) {
#pragma unroll
              for (int k = 0; k < 32; ++k) v[k] += guard_term(special[c + k], pos - base);
            }
            if (it.n_splits > 1) {
#pragma unroll
              for (int k = 0; k < 32; k += 4)
                *reinterpret_cast<float4*>(a.part_o + pr * D + c + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
            } else {
#pragma unroll
              for (int k = 0; k < 32; k += 8)
                *reinterpret_cast<uint4*>(dst + c + k) =
                    make_uint4(f2_to_h2(v[k] * inv, v[k + 1] * inv), f2_to_h2(v[k + 2] * inv, v[k + 3] * inv),
                               f2_to_h2(v[k + 4] * inv, v[k + 5] * inv), f2_to_h2(v[k + 6] * inv, v[k + 7] * inv));
            }
          }
          __syncwarp();  // the next load needs the whole warp
        }
        if (it.n_splits > 1 && valid && t == 0)
          a.part_ml[pr] = make_float2(m_all == -INFINITY ? m_all : m_all * scale, l_all);
        ptx::tcgen05_fence_before();
        exchange();  // both accumulators have been read: either warpgroup may start the next item
      }
      if (it.n_splits > 1) {
        __threadfence();
        exchange();
        if (threadIdx.x == 0) sm.last = atomicAdd(&a.counters[it.counter], 1) == it.n_splits - 1;
        exchange();
        if (*reinterpret_cast<volatile int*>(&sm.last)) {
          __threadfence();
          for (int r = warp; r < rows; r += kSoftmaxWarps) {
            const int rt = r / group;
            merge_row(a, it.row0, rows, r, it.n_splits,
                      a.out + (static_cast<size_t>(it.q_tok + rt) * a.num_heads + kvh * group + r - rt * group) * D, lane);
          }
        }
        exchange();  // `last` may be overwritten from here on
      }
      if (fix) {  // every warp has read the record: clear it for the slot's next item
        exchange();
        for (int i = threadIdx.x; i < D; i += 32 * kSoftmaxWarps) special[i] = kNoSpecial;
        if (threadIdx.x == 0) sm.special_flag[slot] = 0;
      }
      release_item();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == kMmaWarp) {
      // =============================== MMA issue ===============================
      constexpr uint32_t idesc_qk = ptx::make_f16_idesc(kTile, kTile);
      constexpr uint32_t idesc_pv = ptx::make_f16_idesc(kTile, D) | ptx::kIdescBMnMajor;
      Ring ring;
      uint32_t q_phase = 0, p_phase[2] = {0, 0};
      const uint32_t q_base = ptx::smem_u32(smem + Sh::kQ), kv_base = ptx::smem_u32(smem + Sh::kRing);
      auto issue_qk = [&](int t, int qt, int stage) {
        if (ptx::elect_one()) {
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = (ks >> 2) * Sh::kSubBytes + (ks & 3) * 32;
            ptx::umma_f16(tmem + t * kTile, ptx::make_sw128_kmajor_desc(q_base + qt * Sh::kTileBytes + off),
                          ptx::make_sw128_kmajor_desc(kv_base + stage * Sh::kTileBytes + off), idesc_qk, ks > 0);
          }
          ptx::umma_commit(&sm.s_full[t]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int t, int stage, bool accumulate) {
        if (ptx::elect_one()) {
#pragma unroll
          for (int ks = 0; ks < kTile / 16; ++ks)
            ptx::umma_f16_ts(tmem + 2 * kTile + t * D, tmem + t * kTile + ks * 8,
                             ptx::make_sw128_mnmajor_desc(kv_base + stage * Sh::kTileBytes + ks * 2048, Sh::kSubBytes),
                             idesc_pv, accumulate || ks > 0);
        }
        __syncwarp();
      };
      uint32_t k_phase = 0, v_phase = 0;  // a bit per stage: the barriers of a kind only count that kind's tiles
      auto wait_k = [&]() {
        const int ks = ring.stage;
        wait(&sm.k_full[ks], (k_phase >> ks) & 1u, 1);
        k_phase ^= 1u << ks;
        advance<kStages>(ring);
        return ks;
      };
      auto wait_v = [&]() {
        const int vs = ring.stage;
        wait(&sm.v_ok[vs], (v_phase >> vs) & 1u, 1);
        v_phase ^= 1u << vs;
        advance<kStages>(ring);
        return vs;
      };
      auto commit = [&](uint64_t* bar) {
        if (ptx::elect_one()) ptx::umma_commit(bar);
        __syncwarp();
      };
      auto wait_p = [&](int t) {
        wait(&sm.p_full[t], p_phase[t], 1);
        p_phase[t] ^= 1u;
        ptx::tcgen05_fence_after();
      };
      Item it;
      while (next_item(it, 1)) {
        const int n = it.tile1 - it.tile0;
        if (n <= 0) {
          release_item();
          continue;
        }
        const bool dual = it.n_tok > tile_tokens;
        wait(&sm.q_full, q_phase, 1);
        q_phase ^= 1u;
        const int first = wait_k();
        ptx::tcgen05_fence_after();
        issue_qk(0, 0, first);
        if (dual) issue_qk(1, 1, first);
        commit(&sm.kv_empty[first]);
        if (!dual && n > 1) {
          const int second = wait_k();
          issue_qk(1, 0, second);
          commit(&sm.kv_empty[second]);
        }
        if (n <= (dual ? 1 : 2)) commit(&sm.q_empty);
        if (dual) {
          for (int j = 0; j < n; ++j) {
            const int vs = wait_v();
            wait_p(0);
            issue_pv(0, vs, j > 0);
            int ks = 0;
            if (j + 1 < n) {
              ks = wait_k();
              issue_qk(0, 0, ks);
            } else {
              commit(&sm.o_full[0]);
            }
            wait_p(1);
            issue_pv(1, vs, j > 0);
            commit(&sm.kv_empty[vs]);
            if (j + 1 < n) {
              issue_qk(1, 1, ks);
              commit(&sm.kv_empty[ks]);
              if (j + 2 == n) commit(&sm.q_empty);
            } else {
              commit(&sm.o_full[1]);
            }
          }
        } else {
          for (int i = 0; i < n; ++i) {
            const int t = i & 1;
            const int vs = wait_v();
            wait_p(t);
            issue_pv(t, vs, i > 1);
            commit(&sm.kv_empty[vs]);
            if (i + 2 < n) {
              const int ks = wait_k();
              issue_qk(t, 0, ks);
              commit(&sm.kv_empty[ks]);
              if (i + 3 == n) commit(&sm.q_empty);
            } else {
              commit(&sm.o_full[t]);
            }
          }
        }
        release_item();
      }
    } else if (warp == kProducerWarp) {
      // =============================== loads ===============================
      const int n_items = a.header->n_items;
      const int boxes = kTile / box_tokens;          // per 64-channel sub-tile
      const int my_box = lane / Sh::kHalves, my_half = lane - my_box * Sh::kHalves;
      const bool loads = my_box < boxes;
      Ring ring;
      uint32_t q_phase = 0, k_count = 0;
      int idx = blockIdx.x;
      while (idx < n_items && !dead) {
        const Item it = a.items[idx];
        if (lane == 0) idx = gridDim.x + atomicAdd(&a.header->ticket, 1);
        idx = __shfl_sync(0xffffffffu, idx, 0);
        if (it.split >= it.n_splits) continue;
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
        const int ahead = dual ? 1 : 2;
        const int kv_len = it.pos0 + it.n_tok;
        const int32_t* table = a.block_tables + static_cast<size_t>(it.seq) * a.max_pages_per_seq;
        // Page of this lane's box of kv tile i (num_pages: nothing there, TMA fills zeros).
        auto page_of = [&](int i) {
          const int first = (it.tile0 + i) * kTile + my_box * box_tokens;
          if (!loads || i >= n || first >= kv_len) return a.num_pages;
          const int pg = table[first / a.page_size];
          return pg >= 0 && pg < a.num_pages ? pg : a.num_pages;
        };
        auto load = [&](const CUtensorMap* map, uint64_t* full, int i, int page) {
          wait(&sm.kv_empty[ring.stage], ring.phase ^ 1u, 0);
          if (!dead) {
            if (lane == 0) ptx::mbar_arrive_expect_tx(&full[ring.stage], Sh::kTileBytes);
            __syncwarp();
            if (loads)
              ptx::tma_load_4d(smem + Sh::kRing + ring.stage * Sh::kTileBytes + my_half * Sh::kSubBytes +
                                   my_box * box_tokens * 128,
                               map, &full[ring.stage], my_half * 64, it.head,
                               ((it.tile0 + i) * kTile + my_box * box_tokens) % a.page_size, page);
          }
          __syncwarp();
          advance<kStages>(ring);
        };
        auto load_k = [&](int i, int page) {
          // which keys lie in a page that exists, for the softmax; published by the K tile's barrier
          const uint32_t per_box = box_tokens / 8;
          uint32_t bits = 0;
          if (loads && my_half == 0 && page < a.num_pages)
            bits = ((1u << per_box) - 1u) << (my_box * per_box);
          bits = __reduce_or_sync(0xffffffffu, bits);
          if (lane == 0) sm.valid[(k_count + i) & (kMaskRing - 1)] = bits;
          load(&map_k, sm.k_full, i, page);
        };
        int p0 = page_of(0), p1 = page_of(1), p2;  // pages of the next tiles, read ahead of their use
        // Q: rows (token, head) of this kv head's group
        wait(&sm.q_empty, q_phase ^ 1u, 0);
        q_phase ^= 1u;
        if (!dead && lane == 0) {
          const uint32_t bytes = static_cast<uint32_t>(tile_tokens * group) * 128u * Sh::kHalves;
          ptx::mbar_arrive_expect_tx(&sm.q_full, dual ? 2 * bytes : bytes);
          for (int t = 0; t < (dual ? 2 : 1); ++t)
            for (int h = 0; h < Sh::kHalves; ++h)
              ptx::tma_load_3d(smem + Sh::kQ + t * Sh::kTileBytes + h * Sh::kSubBytes, &map_q, &sm.q_full, h * 64,
                               it.head * group, it.q_tok + t * tile_tokens);
        }
        __syncwarp();
        load_k(0, p0);
        if (ahead == 2) {
          p2 = page_of(2);
          if (n > 1) load_k(1, p1);
        } else {
          p2 = 0;
        }
        for (int i = 0; i < n; ++i) {
          load(&map_v, sm.v_full, i, p0);
          const int next = i + ahead;
          if (ahead == 2) {
            const int p3 = page_of(next + 1);
            if (next < n) load_k(next, p2);
            p0 = p1;
            p1 = p2;
            p2 = p3;
          } else {
            const int p3 = page_of(next + 1);
            if (next < n) load_k(next, p1);
            p0 = p1;
            p1 = p3;
          }
        }
        k_count += n;
      }
      if (!dead) {  // the end mark
        wait(&sm.item_empty[slot], slot_phase ^ 1u, 0);
        if (lane == 0) {
          sm.items[slot].n_tok = 0;
          ptx::mbar_arrive(&sm.item_full[slot]);
        }
      }
    } else {
      // =============================== V guard ===============================
      const int part = warp - kGuardWarp;  // this warp's half of the rows
      uint32_t v_phase = 0;
      Ring ring;
      Item it;
      while (next_item(it, 3)) {
        const int n = it.tile1 - it.tile0;
        const bool dual = it.n_tok > tile_tokens;
        const int kv_len = it.pos0 + it.n_tok;
        uint32_t* special = sm.special[slot];
        if (n > 0) advance<kStages>(ring);  // over the K tiles
        if (!dual && n > 1) advance<kStages>(ring);
        for (int i = 0; i < n; ++i) {
          wait(&sm.v_full[ring.stage], (v_phase >> ring.stage) & 1u, 3);
          v_phase ^= 1u << ring.stage;
          const int t0 = (it.tile0 + i) * kTile;
          uint8_t* tile = smem + Sh::kRing + ring.stage * Sh::kTileBytes;
          // rows behind the context: zeros (whole rows, so the swizzle does not matter)
          const int end = min(max(kv_len - t0, 0), kTile);
          // rows that some row of the block does not see: no infinities, no NaN
          const int hid = min(max(it.pos0 + 1 - t0, 0), end);
          if (hid < kTile) {
            const int lo = max(hid, part * (kTile / 2)), hi = (part + 1) * (kTile / 2);
            for (int k = lo * (D / 8) + lane; k < hi * (D / 8); k += 32) {
              const int r = k / (D / 8), c = k - r * (D / 8);
              uint4* p = reinterpret_cast<uint4*>(tile + (c >> 3) * Sh::kSubBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4));
              if (r >= end) {
                *p = make_uint4(0, 0, 0, 0);
              } else {
                uint4 v = *p;
                if (any_nonfinite(v)) {
                  guard_take(v, static_cast<uint32_t>(t0 + r - (it.pos0 + 1)), special + c * 8, &sm.special_flag[slot]);
                  *p = v;
                }
              }
            }
            ptx::fence_proxy_async();
          }
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&sm.v_ok[ring.stage]);
          advance<kStages>(ring);
          if (i + (dual ? 1 : 2) < n) advance<kStages>(ring);
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

int box_tokens_of(int page_size) {
  for (int b = 128; b >= 8; b >>= 1)
    if (page_size % b == 0) return b;
  return 0;
}

template <int D>
int launch_tc_d(const Args& a, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  const uint64_t e = 2;
  const int box = box_tokens_of(a.page_size);
  {
    const uint64_t dims[3] = {D, static_cast<uint64_t>(a.num_heads), static_cast<uint64_t>(a.num_tokens)};
    const uint64_t strides[2] = {D * e, static_cast<uint64_t>(a.num_heads) * D * e};
    const uint32_t b[3] = {64, static_cast<uint32_t>(a.group), static_cast<uint32_t>(a.block_tokens / 2)};
    const int rc = encode_f16_map(&mq, a.q, 3, dims, strides, b, "chunked_paged_attention(q)");
    if (rc != B200OPS_OK) return rc;
  }
  {
    const uint64_t hkv = a.num_kv_heads, page = a.page_size;
    const uint64_t dims[4] = {D, hkv, page, static_cast<uint64_t>(a.num_pages)};
    const uint64_t strides[3] = {D * e, hkv * D * e, page * hkv * D * e};
    const uint32_t b[4] = {64, 1, static_cast<uint32_t>(box), 1};
    int rc = encode_f16_map(&mk, a.k_cache, 4, dims, strides, b, "chunked_paged_attention(key_cache)");
    if (rc != B200OPS_OK) return rc;
    rc = encode_f16_map(&mv, a.v_cache, 4, dims, strides, b, "chunked_paged_attention(value_cache)");
    if (rc != B200OPS_OK) return rc;
  }
  auto kern = chunk_attention_tc_kernel<D>;
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  B200OPS_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
    B200OPS_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_bytes<D>())));
    if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
  }
  const int grid = a.max_items < sm_count() ? a.max_items : sm_count();
  B200OPS_CUDA(launch_kernel(kern, dim3(grid), dim3(kThreads), smem_bytes<D>(), st, mq, mk, mv, a, box));
  return B200OPS_OK;
}

}  // namespace

bool tc_supported(int64_t head_dim, int64_t group, int64_t page_size, int layout) {
  return (head_dim == 64 || head_dim == 128) && group <= 128 && page_size % 8 == 0 && layout == B200OPS_KV_LAYOUT_NHD;
}

int launch_tc(const Args& a, cudaStream_t st) {
  return a.head_dim == 64 ? launch_tc_d<64>(a, st) : launch_tc_d<128>(a, st);
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
