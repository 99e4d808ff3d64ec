// Rotary position embedding in the forms rope.cu does not cover -- interleaved pairs, a rotated
// part of the head, fp32 tables -- and the tables themselves, with the frequency scalings used to
// stretch a model's context.
//
// Frequencies (host, double): f_j = base^(-2j/R), j < R/2, R the rotated channels, then
//   linear  f_j / s                                  (positions interpolated)
//   ntk     base replaced by base * s^(R/(R-2))      (the lowest frequency is divided by s, the highest kept)
//   yarn    f_j / s for the low frequencies, f_j for the high ones, a linear ramp over the index j
//           between those that turn `high` and `low` times over the original context; amplitude 0.1 ln s + 1
//   bands   the same idea with the blend linear in the number of turns
// Tables: cos_t[p, j] = amplitude * cos((start + p) * f_j), sin_t likewise.
//
// Rotary: pair (a, b) of a head becomes (a cos - b sin, b cos + a sin); pairs are (x[j], x[j + R/2])
// or, interleaved, (x[2j], x[2j+1]); channels from R on are copied.  fp32 arithmetic, one rounding.
#include "common.cuh"

#include <cmath>

namespace b200ops {
namespace {

constexpr int kMaxHalf = 256;
constexpr double kTwoPi = 6.283185307179586476925286766559;
constexpr double kTwoPiRest = 2.4492935982947064e-16;  // 2 pi - kTwoPi

// Frequencies, by value in the launch.
struct FrequencyTable {
  double f[kMaxHalf];
};

// Turns (periods) per position, f / 2 pi, as the sum of two doubles: by itself the first is off by 2^-54 of itself, and so
// is a position's angle, which at position 2^31 is more than the last bit of an fp32 table.
struct Turns {
  double high, low;
};

__device__ __forceinline__ Turns turns_of(double f) {
  Turns t;
  t.high = f / kTwoPi;
  t.low = (fma(-t.high, kTwoPi, f) - t.high * kTwoPiRest) / kTwoPi;
  return t;
}

// position * t less whole turns, in turns: the product's rounding error is kept (fma), so what is left are a few
// roundings of numbers below one.
__device__ __forceinline__ double reduced(double position, Turns t) {
  const double p = position * t.high;
  return (p - rint(p)) + fma(position, t.low, fma(position, t.high, -p));
}

__device__ __forceinline__ void store_pair(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_pair(__half* p, float v) { *p = __float2half_rn(v); }

constexpr int kTableThreads = 256;

// One thread = one frequency over `rows` consecutive positions.  The angle of the first one is
// reduced to 2^-50 at any position (fp32 would lose every digit past position 10^7, a plain double product
// one more with every doubling); the others follow by rotating (cos, sin) by one step's angle, four double operations per
// entry.  A step adds an error of at most 2^-50, so all 64 stay below 2^-43 of the amplitude: 2^-18 of half a step of an
// fp32 entry between 1/2 and 1.
// Bound: writing the tables.  Neighbouring threads hold neighbouring frequencies of one row, so a
// warp stores whole sectors: 262144 positions x 64 frequencies in fp32 (134 MB) take 23 us = 5.8 TB/s, in fp16 (67 MB, in
// L2 when the call is repeated) 14.4 us.
template <typename T>
__global__ void __launch_bounds__(kTableThreads)
rotary_tables_kernel(const FrequencyTable ft, T* __restrict__ cos_t, T* __restrict__ sin_t, long long start,
                     long long num_positions, int half, int rows, double amplitude) {
  __shared__ Turns turns[kMaxHalf];
  pdl_trigger();
  for (int i = threadIdx.x; i < half; i += kTableThreads) turns[i] = turns_of(ft.f[i]);
  __syncthreads();
  pdl_wait();
  const long long item = static_cast<long long>(blockIdx.x) * kTableThreads + threadIdx.x;
  const long long group = item / half;
  const int j = static_cast<int>(item - group * half);
  const long long p0 = group * rows;
  if (p0 >= num_positions) return;
  const int n = static_cast<int>(min(static_cast<long long>(rows), num_positions - p0));
  const Turns t = turns[j];
  double c, s, cs, ss;
  sincospi(2.0 * reduced(static_cast<double>(start + p0), t), &s, &c);
  sincospi(2.0 * reduced(1.0, t), &ss, &cs);
  c *= amplitude;
  s *= amplitude;
  T* pc = cos_t + p0 * half + j;
  T* ps = sin_t + p0 * half + j;
  for (int r = 0; r < n; ++r) {
    store_pair(pc, static_cast<float>(c));
    store_pair(ps, static_cast<float>(s));
    pc += half;
    ps += half;
    const double nc = c * cs - s * ss;
    s = s * cs + c * ss;
    c = nc;
  }
}

// ---- rotation ---------------------------------------------------------------------------
constexpr int kRotThreads = 256;

struct RotArgs {
  const __half* q;
  const __half* k;
  const int32_t* position_ids;
  const void* cos_t;
  const void* sin_t;
  __half* out_q;
  __half* out_k;
  long long q_stride, k_stride;  // elements between tokens of the inputs (the outputs are dense)
  long long tokens;
  int num_heads, num_kv_heads, head_dim, half, max_pos;
  bool interleaved;
};

// Plain (coherent) loads: the kernel may be resident while the launch that writes its inputs still runs, so they
// are not constant for its whole life, as the non-coherent path wants.
__device__ __forceinline__ uint4 load_piece(const __half* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// Four neighbouring table entries, 8- (fp16) or 16-byte aligned.
__device__ __forceinline__ void table4(const __half* t, float* v) {
  const uint2 u = *reinterpret_cast<const uint2*>(t);
  const float2 x = h2_to_f2(u.x), y = h2_to_f2(u.y);
  v[0] = x.x, v[1] = x.y, v[2] = y.x, v[3] = y.y;
}
__device__ __forceinline__ void table4(const float* t, float* v) {
  const float4 u = *reinterpret_cast<const float4*>(t);
  v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
}

__device__ __forceinline__ float table_at(const __half* t, long long i) { return __half2float(t[i]); }
__device__ __forceinline__ float table_at(const float* t, long long i) { return t[i]; }

// Any size and alignment: one thread per pair (or per copied channel).  Two-byte accesses and 64-bit index arithmetic bound
// it: 8192 tokens of 32 + 8 heads of 96, 24 channels rotated (pieces that do not end on 16 bytes), take 176 us = 0.7 TB/s
// (floor 19); 48 channels, which the vector kernel takes, 24 us.
template <typename T>
__global__ void __launch_bounds__(kRotThreads) rotary_scalar_kernel(const RotArgs a) {
  pdl_trigger();
  pdl_wait();
  const int slots = a.head_dim - a.half;  // half pairs, then head_dim - 2*half copied channels
  const int heads = a.num_heads + a.num_kv_heads;
  const long long total = a.tokens * heads * slots;
  for (long long i = static_cast<long long>(blockIdx.x) * kRotThreads + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * kRotThreads) {
    const int slot = static_cast<int>(i % slots);
    const long long rest = i / slots;
    const int head = static_cast<int>(rest % heads);
    const long long t = rest / heads;
    const bool is_q = head < a.num_heads;
    const int hh = is_q ? head : head - a.num_heads;
    const __half* in = (is_q ? a.q + t * a.q_stride : a.k + t * a.k_stride) + static_cast<long long>(hh) * a.head_dim;
    __half* out = (is_q ? a.out_q + (t * a.num_heads + hh) * a.head_dim
                        : a.out_k + (t * a.num_kv_heads + hh) * a.head_dim);
    const int pos = a.position_ids[t];
    const bool ok = pos >= 0 && pos < a.max_pos;
    if (slot >= a.half) {
      const int d = slot + a.half;
      out[d] = ok ? in[d] : __float2half(0.f);
      continue;
    }
    const int d0 = a.interleaved ? 2 * slot : slot, d1 = a.interleaved ? 2 * slot + 1 : slot + a.half;
    if (!ok) {
      out[d0] = out[d1] = __float2half(0.f);
      continue;
    }
    const long long e = static_cast<long long>(pos) * a.half + slot;
    const float c = table_at(static_cast<const T*>(a.cos_t), e), s = table_at(static_cast<const T*>(a.sin_t), e);
    const float x = __half2float(in[d0]), y = __half2float(in[d1]);
    out[d0] = __float2half_rn(x * c - y * s);
    out[d1] = __float2half_rn(y * c + x * s);
  }
}

// One thread takes two 16-byte pieces of a head -- eight pairs (x[j], x[j + half]), or four interleaved pairs
// each, or channels to copy -- in `Heads` heads of one token, so that cos and sin are read and converted once for
// all of them and 32 * Heads bytes are under way per thread before the first is used.  Bound by HBM: 16384 tokens
// of 32 + 8 heads of 128 (335 MB in and out) take 60 us = 5.6 TB/s; element by element they took 365 us.
template <typename T, bool Interleaved, int Heads>
__global__ void __launch_bounds__(kRotThreads) rotary_vector_kernel(const RotArgs a, const int pair_items,
                                                                    const int items, const int spans) {
  pdl_trigger();
  const long long i = static_cast<long long>(blockIdx.x) * kRotThreads + threadIdx.x;
  const unsigned per_token = static_cast<unsigned>(items) * spans;
  const long long t = i / per_token;
  if (t >= a.tokens) return;
  const unsigned in_token = static_cast<unsigned>(i - t * per_token);
  const int span = in_token / items, item = in_token - span * items;
  const int heads = a.num_heads + a.num_kv_heads;
  // The item's pieces begin at channels d0 and d1; d1 = head_dim: there is no second one.
  const bool rotates = item < pair_items;
  int d0, d1;
  if (rotates) {
    d0 = 8 * item;
    d1 = Interleaved ? d0 + 8 * pair_items : d0 + a.half;
    if (Interleaved && d1 >= 2 * a.half) d1 = a.head_dim;
  } else {
    d0 = 2 * a.half + 8 * (item - pair_items);
    d1 = d0 + 8 * (items - pair_items);
  }
  const bool second = d1 < a.head_dim;
  pdl_wait();
  uint4 v[Heads][2];
#pragma unroll
  for (int n = 0; n < Heads; ++n) {
    const int head = span + n * spans;
    if (head < heads) {
      const __half* in = head < a.num_heads ? a.q + t * a.q_stride + static_cast<long long>(head) * a.head_dim
                                            : a.k + t * a.k_stride + static_cast<long long>(head - a.num_heads) * a.head_dim;
      v[n][0] = load_piece(in + d0);
      if (second) v[n][1] = load_piece(in + d1);
    }
  }
  const int pos = a.position_ids[t];
  const bool ok = pos >= 0 && pos < a.max_pos;
  float c[8], s[8];
  if (ok && rotates) {
    const long long e = static_cast<long long>(pos) * a.half;
    const T* ct = static_cast<const T*>(a.cos_t) + e;
    const T* st = static_cast<const T*>(a.sin_t) + e;
    if constexpr (Interleaved) {
      table4(ct + d0 / 2, c);
      table4(st + d0 / 2, s);
      if (second) {
        table4(ct + d1 / 2, c + 4);
        table4(st + d1 / 2, s + 4);
      }
    } else {
      table4(ct + d0, c);
      table4(ct + d0 + 4, c + 4);
      table4(st + d0, s);
      table4(st + d0 + 4, s + 4);
    }
  }
#pragma unroll
  for (int n = 0; n < Heads; ++n) {
    const int head = span + n * spans;
    if (head >= heads) break;
    uint32_t x[2][4] = {{v[n][0].x, v[n][0].y, v[n][0].z, v[n][0].w}, {v[n][1].x, v[n][1].y, v[n][1].z, v[n][1].w}};
    if (!ok) {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[0][k] = x[1][k] = 0;
    } else if (rotates) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 p = h2_to_f2(x[0][k]), r = h2_to_f2(x[1][k]);
        if constexpr (Interleaved) {
          x[0][k] = f2_to_h2(p.x * c[k] - p.y * s[k], p.y * c[k] + p.x * s[k]);
          x[1][k] = f2_to_h2(r.x * c[4 + k] - r.y * s[4 + k], r.y * c[4 + k] + r.x * s[4 + k]);
        } else {
          x[0][k] = f2_to_h2(p.x * c[2 * k] - r.x * s[2 * k], p.y * c[2 * k + 1] - r.y * s[2 * k + 1]);
          x[1][k] = f2_to_h2(r.x * c[2 * k] + p.x * s[2 * k], r.y * c[2 * k + 1] + p.y * s[2 * k + 1]);
        }
      }
    }
    __half* out = head < a.num_heads ? a.out_q + (t * a.num_heads + head) * a.head_dim
                                     : a.out_k + (t * a.num_kv_heads + head - a.num_heads) * a.head_dim;
    const uint4 y0 = make_uint4(x[0][0], x[0][1], x[0][2], x[0][3]), y1 = make_uint4(x[1][0], x[1][1], x[1][2], x[1][3]);
    if constexpr (Heads == 4) {  // outputs beyond the L2's size leave it first (60 us, else 64)
      st_stream(out + d0, y0);
      if (second) st_stream(out + d1, y1);
    } else {
      *reinterpret_cast<uint4*>(out + d0) = y0;
      if (second) *reinterpret_cast<uint4*>(out + d1) = y1;
    }
  }
}

template <typename T>
cudaError_t launch_rotary(const RotArgs& a, bool vector, cudaStream_t st) {
  const long long heads = a.num_heads + a.num_kv_heads;
  auto grid = [](long long threads) { return dim3(static_cast<unsigned>((threads + kRotThreads - 1) / kRotThreads)); };
  if (vector) {
    const int pair_items = a.interleaved ? (a.half / 4 + 1) / 2 : a.half / 8;
    const int items = pair_items + ((a.head_dim - 2 * a.half) / 8 + 1) / 2;
    // More heads per thread as the work grows; a small call is spread over as many threads as it can.  With one,
    // two and four (28 + 4 heads of 128): 64 tokens 1.7, 2.0, 2.4 us; 2048 tokens 5.8, 5.2, 5.5 us; 16384 tokens
    // 53, 51, 44 us.
    const long long threads = a.tokens * heads * items, chip = 1024LL * sm_count();
    const int per = threads < chip ? 1 : (threads < 8 * chip ? 2 : 4);
    const int spans = static_cast<int>((heads + per - 1) / per);
    const dim3 g = grid(a.tokens * spans * items);
    auto go = [&](auto kern) { return launch_kernel(kern, g, dim3(kRotThreads), 0, st, a, pair_items, items, spans); };
    if (a.interleaved)
      return per == 1 ? go(rotary_vector_kernel<T, true, 1>)
                      : (per == 2 ? go(rotary_vector_kernel<T, true, 2>) : go(rotary_vector_kernel<T, true, 4>));
    return per == 1 ? go(rotary_vector_kernel<T, false, 1>)
                    : (per == 2 ? go(rotary_vector_kernel<T, false, 2>) : go(rotary_vector_kernel<T, false, 4>));
  }
  const long long total = a.tokens * heads * (a.head_dim - a.half);
  const long long most = 0x7fffffffLL * kRotThreads;
  return launch_kernel(rotary_scalar_kernel<T>, grid(total < most ? total : most), dim3(kRotThreads), 0, st, a);
}

}  // namespace
}  // namespace b200ops

extern "C" int b200ops_rotary_frequencies(int64_t rotary_dim, double base, int scaling, double factor,
                                          int64_t original_positions, double low, double high,
                                          double* frequencies, double* amplitude) {
  using namespace b200ops;
  B200OPS_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= 2 * kMaxHalf,
                  "rotary_frequencies: rotary_dim must be even and at most %d, got %lld", 2 * kMaxHalf,
                  (long long)rotary_dim);
  B200OPS_REQUIRE(base > 1.0 && std::isfinite(base), "rotary_frequencies: base must be finite and above 1, got %g", base);
  B200OPS_REQUIRE(scaling >= B200OPS_ROTARY_NONE && scaling <= B200OPS_ROTARY_BANDS,
                  "rotary_frequencies: unknown scaling %d", scaling);
  B200OPS_REQUIRE(frequencies && amplitude, "rotary_frequencies: null pointer");
  const bool ramped = scaling == B200OPS_ROTARY_YARN || scaling == B200OPS_ROTARY_BANDS;
  B200OPS_REQUIRE(scaling == B200OPS_ROTARY_NONE || (factor >= 1.0 && std::isfinite(factor)),
                  "rotary_frequencies: factor must be finite and at least 1, got %g", factor);
  B200OPS_REQUIRE(scaling != B200OPS_ROTARY_NTK || rotary_dim > 2,
                  "rotary_frequencies: ntk scaling needs a rotary_dim above 2");
  B200OPS_REQUIRE(!ramped || (original_positions > 0 && low > 0.0 && high > low && std::isfinite(high)),
                  "rotary_frequencies: this scaling needs original_positions > 0 and 0 < low < high, got %lld, %g, %g",
                  (long long)original_positions, low, high);
  const double dim = static_cast<double>(rotary_dim);
  const int half = static_cast<int>(rotary_dim / 2);
  if (scaling == B200OPS_ROTARY_NTK) base *= std::pow(factor, dim / (dim - 2.0));
  *amplitude = 1.0;
  double ramp_lo = 0.0, ramp_hi = 0.0;
  if (scaling == B200OPS_ROTARY_YARN) {
    // index whose frequency turns n times over the original context
    auto index_of = [&](double n) {
      return dim * std::log(original_positions / (n * kTwoPi)) / (2.0 * std::log(base));
    };
    ramp_lo = std::fmax(std::floor(index_of(high)), 0.0);
    ramp_hi = std::fmin(std::ceil(index_of(low)), dim - 1.0);
    *amplitude = 0.1 * std::log(factor) + 1.0;
  }
  for (int j = 0; j < half; ++j) {
    double f = std::pow(base, -2.0 * j / dim);
    double keep = 1.0;  // share of the unscaled frequency
    if (scaling == B200OPS_ROTARY_LINEAR) {
      keep = 0.0;
    } else if (scaling == B200OPS_ROTARY_YARN) {
      const double r = (j - ramp_lo) / std::fmax(ramp_hi - ramp_lo, 1e-3);
      keep = 1.0 - std::fmin(std::fmax(r, 0.0), 1.0);
    } else if (scaling == B200OPS_ROTARY_BANDS) {
      const double r = (original_positions * f / kTwoPi - low) / (high - low);
      keep = std::fmin(std::fmax(r, 0.0), 1.0);
    }
    frequencies[j] = keep == 1.0 ? f : f / factor * (1.0 - keep) + f * keep;
  }
  return B200OPS_OK;
}

extern "C" int b200ops_rotary_tables(const double* frequencies, int64_t half, double amplitude, int64_t start,
                                     int64_t num_positions, void* cos_table, void* sin_table, int table_type,
                                     void* stream) {
  using namespace b200ops;
  B200OPS_REQUIRE(half >= 1 && half <= kMaxHalf, "rotary_tables: 1 to %d frequencies, got %lld", kMaxHalf,
                  (long long)half);
  B200OPS_REQUIRE(start >= 0 && num_positions >= 0 && start <= 0x7fffffffLL && num_positions <= 0x7fffffffLL,
                  "rotary_tables: bad range of positions, start=%lld count=%lld", (long long)start,
                  (long long)num_positions);
  B200OPS_REQUIRE(table_type == B200OPS_TABLE_F16 || table_type == B200OPS_TABLE_F32,
                  "rotary_tables: unknown table type %d", table_type);
  B200OPS_REQUIRE(std::isfinite(amplitude), "rotary_tables: amplitude must be finite");
  B200OPS_REQUIRE(frequencies, "rotary_tables: null pointer");
  FrequencyTable ft;
  for (int64_t j = 0; j < half; ++j) {
    B200OPS_REQUIRE(std::isfinite(frequencies[j]) && std::fabs(frequencies[j]) <= 1e6,
                    "rotary_tables: frequency %lld is %g", (long long)j, frequencies[j]);
    ft.f[j] = frequencies[j];
  }
  if (num_positions == 0) return B200OPS_OK;
  B200OPS_REQUIRE(cos_table && sin_table, "rotary_tables: null pointer");
  int64_t rows = num_positions * half / (static_cast<int64_t>(sm_count()) * 1024);
  rows = rows < 4 ? 4 : (rows > 64 ? 64 : rows);
  const int64_t items = (num_positions + rows - 1) / rows * half;
  const dim3 grid(static_cast<unsigned>((items + kTableThreads - 1) / kTableThreads));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (table_type == B200OPS_TABLE_F32)
    B200OPS_CUDA(launch_kernel(rotary_tables_kernel<float>, grid, dim3(kTableThreads), 0, st, ft,
                               static_cast<float*>(cos_table), static_cast<float*>(sin_table), (long long)start,
                               (long long)num_positions, (int)half, (int)rows, amplitude));
  else
    B200OPS_CUDA(launch_kernel(rotary_tables_kernel<__half>, grid, dim3(kTableThreads), 0, st, ft,
                               static_cast<__half*>(cos_table), static_cast<__half*>(sin_table), (long long)start,
                               (long long)num_positions, (int)half, (int)rows, amplitude));
  return B200OPS_OK;
}

extern "C" int b200ops_rotary(const void* q, const void* k, const int32_t* position_ids, const void* cos_table,
                              const void* sin_table, int table_type, void* out_q, void* out_k, int64_t num_tokens,
                              int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t rotary_dim,
                              int64_t q_stride, int64_t k_stride, int64_t max_pos, int interleaved, void* stream) {
  using namespace b200ops;
  B200OPS_REQUIRE(num_tokens >= 0 && num_heads >= 0 && num_kv_heads >= 0 && head_dim > 0 && max_pos >= 0,
                  "rotary: bad shape tokens=%lld heads=%lld kv_heads=%lld head_dim=%lld max_pos=%lld",
                  (long long)num_tokens, (long long)num_heads, (long long)num_kv_heads, (long long)head_dim,
                  (long long)max_pos);
  B200OPS_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
                  "rotary: rotary_dim must be even and at most head_dim %lld, got %lld", (long long)head_dim,
                  (long long)rotary_dim);
  B200OPS_REQUIRE(table_type == B200OPS_TABLE_F16 || table_type == B200OPS_TABLE_F32, "rotary: unknown table type %d",
                  table_type);
  B200OPS_REQUIRE(max_pos <= 0x7fffffffLL && head_dim <= 65536 && num_heads <= 65536 && num_kv_heads <= 65536 &&
                      num_tokens <= 0x7fffffffLL,
                  "rotary: shape too large");
  if (num_tokens == 0 || num_heads + num_kv_heads == 0) return B200OPS_OK;
  B200OPS_REQUIRE(q_stride >= num_heads * head_dim && k_stride >= num_kv_heads * head_dim,
                  "rotary: token strides %lld and %lld are shorter than a token's heads", (long long)q_stride,
                  (long long)k_stride);
  B200OPS_REQUIRE(position_ids && cos_table && sin_table, "rotary: null pointer");
  B200OPS_REQUIRE((num_heads == 0 || (q && out_q)) && (num_kv_heads == 0 || (k && out_k)), "rotary: null pointer");
  RotArgs a;
  a.q = static_cast<const __half*>(q);
  a.k = static_cast<const __half*>(k);
  a.position_ids = position_ids;
  a.cos_t = cos_table;
  a.sin_t = sin_table;
  a.out_q = static_cast<__half*>(out_q);
  a.out_k = static_cast<__half*>(out_k);
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.tokens = num_tokens;
  a.num_heads = (int)num_heads;
  a.num_kv_heads = (int)num_kv_heads;
  a.head_dim = (int)head_dim;
  a.half = (int)(rotary_dim / 2);
  a.max_pos = (int)max_pos;
  a.interleaved = interleaved != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // 16-byte pieces need aligned heads, tokens and table rows, and rotated channels that end with a piece.
  const bool vector = head_dim % 8 == 0 && a.half % (interleaved ? 4 : 8) == 0 && q_stride % 8 == 0 &&
                      k_stride % 8 == 0 && aligned16(q) && aligned16(k) && aligned16(out_q) && aligned16(out_k) &&
                      aligned16(cos_table) && aligned16(sin_table);
  B200OPS_CUDA(table_type == B200OPS_TABLE_F32 ? launch_rotary<float>(a, vector, st) : launch_rotary<__half>(a, vector, st));
  return B200OPS_OK;
}
