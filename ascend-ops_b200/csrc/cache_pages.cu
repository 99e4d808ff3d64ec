// Moving pages of the paged KV cache: copy_pages carries out a list of page copies, compact_pages
// closes the holes that ended sequences leave, so that the live pages are the cache's first ones.
// Both treat a page as bytes (any layout and element type whose pages are contiguous) and take
// all the tensors that share one page numbering -- keys and values of every layer -- in one launch.
//
// Bound: HBM, every moved byte read once and written once: 572 MB of pages copied in 208 us = 5.5 TB/s, 515 MB
// compacted in 178 us = 5.8 TB/s.  Four 16-byte loads under way per thread (eight: 2 % faster there, 5 % slower for a few
// pages; evict-first hints on the loads: 2 to 4 % slower).
#include "common.cuh"

#include <algorithm>
#include <type_traits>

namespace b200ops {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kMaxTensors = 256;    // tensors per launch (their addresses travel by value)
constexpr int kMaxListed = 1024;    // tensors per call
constexpr int kMaxPairs = 4096;     // pairs per launch of copy_pages
constexpr int kUnroll = 4;          // loads in flight per thread

struct TensorTable {
  char* base[kMaxTensors];
};

// Copies `n` vectors, kUnroll in flight per thread.  (No __restrict__ on inputs in this file: it would let them be
// read as constants, but the kernels may be resident while the launch that writes them still runs.)
template <typename V>
__device__ __forceinline__ void copy_slice(const V* src, V* dst, int n) {
  for (int i0 = threadIdx.x; i0 < n; i0 += kCopyThreads * kUnroll) {
    V v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i0 + u * kCopyThreads < n) v[u] = src[i0 + u * kCopyThreads];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i0 + u * kCopyThreads < n) dst[i0 + u * kCopyThreads] = v[u];
  }
}

// All pairs' copies, none of whose sources is another pair's destination, spread over the grid:
// unit = (pair, tensor, slice of the page).
template <typename V>
__device__ __forceinline__ void copy_disjoint(const TensorTable& tt, int tensors, const int32_t* src, const int32_t* dst,
                                              int pairs, int num_pages, long long page_vecs) {
  constexpr int kSlice = kCopyThreads * kUnroll;
  const long long slices = (page_vecs + kSlice - 1) / kSlice;
  const long long units = static_cast<long long>(pairs) * tensors * slices;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const long long pt = u / slices;
    const long long sl = u - pt * slices;
    const int pair = static_cast<int>(pt / tensors);
    const int tensor = static_cast<int>(pt - static_cast<long long>(pair) * tensors);
    const int s = src[pair], d = dst[pair];
    if (s < 0 || d < 0 || s >= num_pages || d >= num_pages || s == d) continue;
    V* base = reinterpret_cast<V*>(tt.base[tensor]);
    const long long off = sl * kSlice;
    copy_slice(base + s * page_vecs + off, base + d * page_vecs + off,
               static_cast<int>(min(static_cast<long long>(kSlice), page_vecs - off)));
  }
}

// copy_pages: the result is that of a loop over the pairs in order.  Pairs are independent unless
// one pair's destination is also a source or the destination of another; every CTA finds that out
// for itself with a hash set of the destinations in shared memory (about 1 us for 1000 pairs,
// hidden by the first copies' latency; a planning launch of its own would cost more).  Independent
// pairs are spread over the grid.  Otherwise every thread walks the whole list for its own 16-byte
// columns of the page, which keeps the order without any exchange between threads, at one load and store
// at a time: 600 pairs of 128 KB in 8 tensors take 205 us if they are independent and 408 us if a single pair is not.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads)
copy_pages_kernel(const TensorTable tt, int tensors, const int32_t* src, const int32_t* dst,
                  int pairs, int num_pages, long long page_vecs, int hash_mask) {
  extern __shared__ int table[];  // hash_mask + 1 destinations, -1 = free
  __shared__ int conflict;
  pdl_trigger();
  for (int i = threadIdx.x; i <= hash_mask; i += kCopyThreads) table[i] = -1;
  if (threadIdx.x == 0) conflict = 0;
  __syncthreads();
  pdl_wait();
  auto hash = [&](int p) { return static_cast<int>((static_cast<uint32_t>(p) * 2654435761u) >> 16) & hash_mask; };
  auto live = [&](int s, int d) { return s >= 0 && d >= 0 && s < num_pages && d < num_pages && s != d; };
  for (int i = threadIdx.x; i < pairs; i += kCopyThreads) {
    const int s = src[i], d = dst[i];
    if (!live(s, d)) continue;
    for (int h = hash(d);; h = (h + 1) & hash_mask) {  // at most half full: a free slot always turns up
      const int was = atomicCAS(&table[h], -1, d);
      if (was == -1) break;
      if (was == d) {
        conflict = 1;
        break;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += kCopyThreads) {
    const int s = src[i], d = dst[i];
    if (!live(s, d)) continue;
    for (int h = hash(s); table[h] != -1; h = (h + 1) & hash_mask)
      if (table[h] == s) {
        conflict = 1;
        break;
      }
  }
  __syncthreads();
  if (conflict == 0) {
    copy_disjoint<V>(tt, tensors, src, dst, pairs, num_pages, page_vecs);
    return;
  }
  const long long columns = page_vecs * tensors;
  for (long long c = static_cast<long long>(blockIdx.x) * kCopyThreads + threadIdx.x; c < columns;
       c += static_cast<long long>(gridDim.x) * kCopyThreads) {
    const int tensor = static_cast<int>(c / page_vecs);
    V* column = reinterpret_cast<V*>(tt.base[tensor]) + (c - tensor * page_vecs);
    for (int i = 0; i < pairs; ++i) {
      const int s = src[i], d = dst[i];
      if (live(s, d)) column[d * page_vecs] = column[s * page_vecs];
    }
  }
}

// compact_pages, first launch: one CTA finds the live pages and where each goes.  Its time goes with the size of
// the tables, used or not (an entry costs its row's count, then itself, from L2): 28 us for 256 rows of 128
// entries, 130 us for 64 of 8192, 500 us for 256 of 8192, with 100 entries of each row in use (both launches, nothing to
// move).  A caller with wide tables hands over the columns in use.
// Workspace: move count, then the sources and the destinations of the moves.
constexpr int kPlanThreads = 1024;
constexpr int kMaxCompactPages = 1 << 19;  // bitmap and prefix counts in shared memory: 128 KB

__global__ void __launch_bounds__(kPlanThreads)
compact_plan_kernel(const int32_t* tables, const int32_t* page_counts, long long seqs, int width,
                    int num_pages, int32_t* __restrict__ page_map, int32_t* __restrict__ num_live,
                    int32_t* __restrict__ moves, int32_t* __restrict__ move_src, int32_t* __restrict__ move_dst) {
  extern __shared__ uint32_t sm[];
  const int words = (num_pages + 31) >> 5;
  uint32_t* bits = sm;                                  // live pages
  int* before = reinterpret_cast<int*>(sm + words);     // live pages before each word
  __shared__ int warp_sums[32];
  __shared__ int total, low;
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < words; i += kPlanThreads) bits[i] = 0;
  __syncthreads();
  pdl_wait();
  const int entries = static_cast<int>(seqs * width);  // at most 2^26
  for (int i0 = tid; i0 < entries; i0 += kPlanThreads * kUnroll) {
    int page[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = i0 + u * kPlanThreads, b = i / width;
      page[u] = i < entries && i - b * width < page_counts[b] ? tables[i] : -1;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (page[u] >= 0 && page[u] < num_pages) atomicOr(&bits[page[u] >> 5], 1u << (page[u] & 31));
  }
  __syncthreads();
  // exclusive prefix of the words' live counts: a run of words per thread, then over the threads
  const int run = (words + kPlanThreads - 1) / kPlanThreads;
  const int w0 = min(tid * run, words), w1 = min(w0 + run, words);
  int mine = 0;
  for (int w = w0; w < w1; ++w) mine += __popc(bits[w]);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int v = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    warp_sums[lane] = v;
    if (lane == 31) total = v;
  }
  __syncthreads();
  int acc = incl - mine + (warp > 0 ? warp_sums[warp - 1] : 0);
  for (int w = w0; w < w1; ++w) {
    before[w] = acc;
    acc += __popc(bits[w]);
  }
  __syncthreads();
  const int m = total;
  auto live_before = [&](int p) { return before[p >> 5] + __popc(bits[p >> 5] & ((1u << (p & 31)) - 1u)); };
  if (tid == 0) {
    low = m < num_pages ? live_before(m) : m;  // live pages that stay
    *num_live = m;
    *moves = m - low;
  }
  for (int p = tid; p < m; p += kPlanThreads)  // holes, ascending
    if (((bits[p >> 5] >> (p & 31)) & 1u) == 0) move_dst[p - live_before(p)] = p;
  __syncthreads();
  for (int p = tid; p < num_pages; p += kPlanThreads) {
    int to = -1;
    if ((bits[p >> 5] >> (p & 31)) & 1u) {
      to = p;
      if (p >= m) {
        const int rank = live_before(p) - low;
        move_src[rank] = p;
        to = move_dst[rank];
      }
    }
    page_map[p] = to;
  }
}

// compact_pages, second launch: the moves (sources lie above, destinations below the new end, so
// they never meet) and the tables under the new numbers.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads)
compact_move_kernel(const TensorTable tt, int tensors, const int32_t* moves, const int32_t* move_src,
                    const int32_t* move_dst, const int32_t* tables, const int32_t* page_counts,
                    const int32_t* page_map, int32_t* new_tables, long long seqs, int width, int num_pages,
                    long long page_vecs) {
  pdl_trigger();
  pdl_wait();
  if (new_tables != nullptr) {
    const long long entries = seqs * width;
    for (long long i = static_cast<long long>(blockIdx.x) * kCopyThreads + threadIdx.x; i < entries;
         i += static_cast<long long>(gridDim.x) * kCopyThreads) {
      const long long b = i / width;
      int p = tables[i];
      if (i - b * width < page_counts[b] && p >= 0 && p < num_pages) p = page_map[p];
      new_tables[i] = p;
    }
  }
  copy_disjoint<V>(tt, tensors, move_src, move_dst, *moves, num_pages, page_vecs);
}

// Widest vector that a page of this size at these addresses can be copied in.
int vector_bytes(void* const* tensors, int64_t n, int64_t page_bytes) {
  uintptr_t bits = static_cast<uintptr_t>(page_bytes);
  for (int64_t i = 0; i < n; ++i) bits |= reinterpret_cast<uintptr_t>(tensors[i]);
  if ((bits & 15) == 0) return 16;
  if ((bits & 3) == 0) return 4;
  return 1;
}

int check_tensors(const char* op, void* const* tensors, int64_t n, int64_t num_pages, int64_t page_bytes) {
  B200OPS_REQUIRE(n >= 1 && n <= kMaxListed && tensors, "%s: one to %d cache tensors, got %lld", op, kMaxListed,
                  (long long)n);
  constexpr int64_t kMaxBytes = 1LL << 48;  // of a tensor: more than can be addressed, and the sums below cannot wrap
  B200OPS_REQUIRE(num_pages >= 1 && num_pages <= 0x7fffffffLL && page_bytes >= 1 && page_bytes <= kMaxBytes / num_pages,
                  "%s: bad cache shape pages=%lld page_bytes=%lld", op, (long long)num_pages, (long long)page_bytes);
  // Two tensors that share memory would be written through both: refuse instead of racing.
  uintptr_t sorted[kMaxListed];
  for (int64_t i = 0; i < n; ++i) {
    B200OPS_REQUIRE(tensors[i], "%s: null pointer", op);
    sorted[i] = reinterpret_cast<uintptr_t>(tensors[i]);
  }
  std::sort(sorted, sorted + n);
  const uintptr_t span = static_cast<uintptr_t>(num_pages) * static_cast<uintptr_t>(page_bytes);
  for (int64_t i = 1; i < n; ++i)
    B200OPS_REQUIRE(sorted[i] - sorted[i - 1] >= span, "%s: two of the cache tensors overlap", op);
  return B200OPS_OK;
}

unsigned copy_grid(int64_t units) {
  const int64_t limit = static_cast<int64_t>(sm_count()) * 8;
  return static_cast<unsigned>(units < 1 ? 1 : (units < limit ? units : limit));
}

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

template <typename V>
int launch_copy(const TensorTable& tt, int tensors, const int32_t* src, const int32_t* dst, int pairs, int num_pages,
                int64_t page_bytes, cudaStream_t st) {
  const int64_t vecs = page_bytes / static_cast<int64_t>(sizeof(V));
  int slots = 64;
  while (slots < 2 * pairs) slots *= 2;
  const int64_t units = pairs * static_cast<int64_t>(tensors) * ((vecs + kCopyThreads * kUnroll - 1) / (kCopyThreads * kUnroll));
  B200OPS_CUDA(launch_kernel(copy_pages_kernel<V>, dim3(copy_grid(units)), dim3(kCopyThreads), slots * sizeof(int), st,
                             tt, tensors, src, dst, pairs, num_pages, (long long)vecs, slots - 1));
  return B200OPS_OK;
}

}  // namespace
}  // namespace b200ops

extern "C" int b200ops_copy_pages(void* const* tensors, int64_t num_tensors, int64_t num_pages, int64_t page_bytes,
                                  const int32_t* src_pages, const int32_t* dst_pages, int64_t num_pairs, void* stream) {
  using namespace b200ops;
  const int rc = check_tensors("copy_pages", tensors, num_tensors, num_pages, page_bytes);
  if (rc != B200OPS_OK) return rc;
  B200OPS_REQUIRE(num_pairs >= 0 && num_pairs <= 0x7fffffffLL, "copy_pages: bad number of pairs %lld",
                  (long long)num_pairs);
  if (num_pairs == 0) return B200OPS_OK;
  B200OPS_REQUIRE(src_pages && dst_pages, "copy_pages: null pointer");
  const int vec = vector_bytes(tensors, num_tensors, page_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int64_t t0 = 0; t0 < num_tensors; t0 += kMaxTensors) {
    TensorTable tt;
    const int n = static_cast<int>(num_tensors - t0 < kMaxTensors ? num_tensors - t0 : kMaxTensors);
    for (int i = 0; i < n; ++i) tt.base[i] = static_cast<char*>(tensors[t0 + i]);
    for (int64_t p0 = 0; p0 < num_pairs; p0 += kMaxPairs) {  // launches of one stream: the order of the pairs is kept
      const int pairs = static_cast<int>(num_pairs - p0 < kMaxPairs ? num_pairs - p0 : kMaxPairs);
      const int r = vec == 16  ? launch_copy<uint4>(tt, n, src_pages + p0, dst_pages + p0, pairs, (int)num_pages, page_bytes, st)
                    : vec == 4 ? launch_copy<uint32_t>(tt, n, src_pages + p0, dst_pages + p0, pairs, (int)num_pages, page_bytes, st)
                               : launch_copy<uint8_t>(tt, n, src_pages + p0, dst_pages + p0, pairs, (int)num_pages, page_bytes, st);
      if (r != B200OPS_OK) return r;
    }
  }
  return B200OPS_OK;
}

extern "C" size_t b200ops_compact_pages_workspace_size(int64_t num_pages) {
  using namespace b200ops;
  if (num_pages <= 0) return 0;
  return 256 + 2 * align256(static_cast<size_t>(num_pages) * sizeof(int32_t));
}

extern "C" int b200ops_compact_pages(void* const* tensors, int64_t num_tensors, int64_t num_pages, int64_t page_bytes,
                                     const int32_t* block_tables, const int32_t* page_counts, int64_t num_seqs,
                                     int64_t max_pages_per_seq, int32_t* new_block_tables, int32_t* page_map,
                                     int32_t* num_live, void* workspace, size_t workspace_size, void* stream) {
  using namespace b200ops;
  const int rc = check_tensors("compact_pages", tensors, num_tensors, num_pages, page_bytes);
  if (rc != B200OPS_OK) return rc;
  B200OPS_REQUIRE(num_seqs >= 0 && max_pages_per_seq >= 0 && num_seqs <= (1 << 26) && max_pages_per_seq <= (1 << 26) &&
                      num_seqs * max_pages_per_seq <= (1 << 26),
                  "compact_pages: bad table shape [%lld, %lld]", (long long)num_seqs, (long long)max_pages_per_seq);
  if (num_pages > kMaxCompactPages)
    return fail(B200OPS_EUNSUPPORTED, "compact_pages: at most %d pages, got %lld", kMaxCompactPages, (long long)num_pages);
  const bool empty = num_seqs == 0 || max_pages_per_seq == 0;
  B200OPS_REQUIRE(page_map && num_live && (empty || (block_tables && page_counts && new_block_tables)),
                  "compact_pages: null pointer");
  B200OPS_REQUIRE(empty || new_block_tables != block_tables,
                  "compact_pages: the new tables need memory of their own");
  const size_t need = b200ops_compact_pages_workspace_size(num_pages);
  if (workspace == nullptr || workspace_size < need)
    return fail(B200OPS_EWORKSPACE, "compact_pages: workspace of %zu bytes needed, got %zu", need,
                workspace ? workspace_size : (size_t)0);
  B200OPS_REQUIRE(aligned16(workspace), "compact_pages: the workspace must be 16-byte aligned");
  int32_t* moves = static_cast<int32_t*>(workspace);
  int32_t* move_src = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + 256);
  int32_t* move_dst = reinterpret_cast<int32_t*>(reinterpret_cast<char*>(move_src) +
                                                 align256(static_cast<size_t>(num_pages) * sizeof(int32_t)));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t smem = static_cast<size_t>((num_pages + 31) / 32) * 8;
  if (smem > 48 * 1024)  // set on every such call: the attribute belongs to the device, and the call is cheap
    B200OPS_CUDA(cudaFuncSetAttribute(compact_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      kMaxCompactPages / 32 * 8));
  B200OPS_CUDA(launch_kernel(compact_plan_kernel, dim3(1), dim3(kPlanThreads), smem, st, block_tables, page_counts,
                             (long long)(empty ? 0 : num_seqs), (int)(empty ? 1 : max_pages_per_seq), (int)num_pages,
                             page_map, num_live, moves, move_src, move_dst));
  const int vec = vector_bytes(tensors, num_tensors, page_bytes);
  for (int64_t t0 = 0; t0 < num_tensors; t0 += kMaxTensors) {
    TensorTable tt;
    const int n = static_cast<int>(num_tensors - t0 < kMaxTensors ? num_tensors - t0 : kMaxTensors);
    for (int i = 0; i < n; ++i) tt.base[i] = static_cast<char*>(tensors[t0 + i]);
    int32_t* out = t0 == 0 && !empty ? new_block_tables : nullptr;
    const dim3 grid(copy_grid(0x7fffffff));
    auto launch = [&](auto* v) {
      using V = std::remove_pointer_t<decltype(v)>;
      return launch_kernel(compact_move_kernel<V>, grid, dim3(kCopyThreads), 0, st, tt, n, moves, move_src, move_dst,
                           block_tables, page_counts, page_map, out, (long long)(empty ? 0 : num_seqs),
                           (int)(empty ? 1 : max_pages_per_seq), (int)num_pages,
                           (long long)(page_bytes / static_cast<int64_t>(sizeof(V))));
    };
    B200OPS_CUDA(vec == 16  ? launch(static_cast<uint4*>(nullptr))
                 : vec == 4 ? launch(static_cast<uint32_t*>(nullptr))
                            : launch(static_cast<uint8_t*>(nullptr)));
  }
  return B200OPS_OK;
}
