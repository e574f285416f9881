// Sampling a token from each row of logits: temperature, top-k, top-p, min-p and a given random number (include/dspark.h).
//
// A token's weight exp((z - max) / T) is a whole number w = rint((2^44 - 2^24) exp(..)), computed in 64 bits, so that every sum of
// weights is one too whatever the order it is taken in: histograms by atomic adds, partial sums of workgroups and the
// draw itself give the same bits always, and sums of 2^20 weights, the longest row, reach 2^64 - 2^44 at most. (Sums of fp32
// weights move the borders between tokens by 2^-24 of the whole, more than most of a vocabulary's tokens have; one draw in a
// thousand then falls to another token than the definition's.)
//
// Top-k and top-p both keep a prefix of the tokens ranked by (z descending, index), min-p one by z alone: what is kept is
// "key above key*, or equal to it and index up to idx*" and z at least the min-p bound. The cut is found without sorting:
//   1 sample_max    a part of a row each: the largest key, and about the part's weight; clears the row's histogram
//   2 sample_hist   a part each: tokens by bins of max - z, logarithmic (128 an octave), counts (top-k) or weights too (top-p)
//                   by LDS atomics, added to the row's; the last part to finish finds the bin in which the cut lies
//   3 sample_pick   a part each: that bin's tokens into the row's list, and the weight above it by chunks of 512 tokens (top-k of few:
//                   all tokens down to the bin into the list); the last part finds the cut in the list, then the token. SP_SMALL
//                   tokens are ranked by comparing all with all, more narrowed to that by a second division of the bin.
// Rows that need no cut take no histogram but sums by chunks, and one workgroup then the draw. A row whose bin alone passes
// SP_LIST tokens (equal logits by thousands, as bfloat16 has far from zero) takes two passes of one workgroup more (sp_crowded: 9 rows
// of 128000 tokens around 40, top-p 0.9, 0.57 -> 0.12 ms). One whose top-k passes a list with top-p behind it is finished by one
// workgroup from the row itself, some fifteen passes (the same rows, top-k 5000 with top-p 0.9: 0.88 ms against 0.06 with top-k 3000).
//
// What bounds it: few rows, the three launches' chains of dependent reads (one row of 65536 tokens 3.8 + 7.4 + 11.5 us, each beginning
// with ~2.5 of launch and first load and ending in round trips to memory of ~1 us: arrivals, list, sums, the drawn chunk). Many
// rows, 64-bit multiply-adds: 256 rows of 128000 fp16 tokens read 65.5 MB three times, 20 us for the maximum (3.4 TB/s), 38 for
// the histogram, 60-66 for the third launch, most of which is the CUs whose rows keep a third of their tokens: each of those
// has its weight worked out again. Measured and not kept: the weights of kept tokens alone, one a lane at a time (71 -> 69 us at
// top-p 0.9); 2048 parts instead of 1024 (mixed settings 61 -> 58 us, top-k 32 -> 37, none 10 -> 16).
#include <algorithm>
#include <type_traits>

#include "batch.h"
#include "dspark.h"

namespace dspark {

// Tokens of a thread and of a workgroup at a time. The second and third launch have workgroups of 512 threads: adds of many workgroups to
// one word go one after the other, some 50 ns each (9 rows of 128000 tokens: with 256 threads and a word a wave 45 us a call, with
// 512 and a word a workgroup 29).
constexpr int SP_UNIT = 8, SP_MAX_THREADS = 256, SP_THREADS = 512, SP_STEP = SP_THREADS * SP_UNIT;
// Waves of a SIMD in the second launch, so that four workgroups a CU run at once: left alone the compiler takes over 96 scalar registers,
// which leaves room for three (256 rows of 128000 tokens 43 -> 38.5 us). The third launch keeps to three: the fourth goes where one is
// done first, and rows that keep many tokens lie on more CUs (top-p 0.9 71 us, with four at once 87).
constexpr int SP_WAVES = 8;
constexpr int SP_CHUNK = 64 * SP_UNIT;
constexpr int SP_BINS = 2048, SP_LIST = 3584, SP_SMALL = 256, SP_PARTS = 256, SP_CHUNKS = 2048;
constexpr uint64_t SP_ONE = ((uint64_t)1 << 44) - ((uint64_t)1 << 24);  // the largest weight: 2^20 of them are under 2^64
constexpr uint32_t SP_BIN0 = (127 - 9) << 7;  // bin 1 begins at max - z = 2^-9, the last one at 2^7

enum : uint32_t { SP_EMPTY, SP_GREEDY, SP_ALL, SP_LISTED, SP_BELOW, SP_ROW };

__device__ __forceinline__ float sp_value(float z) { return z != z ? -INFINITY : z == 0.f ? 0.f : z; }  // (-0 is 0)
// What an argmax key was made of.
__device__ __forceinline__ float sp_logit(uint32_t ord) { return __uint_as_float(ord & 0x80000000u ? ord ^ 0x80000000u : ~ord); }
__device__ __forceinline__ uint32_t sp_index(uint64_t key) { return 0xffffffffu - (uint32_t)key; }
// max - z, rounded but in the order of z. (s.inf is the same in every lane: the other side of its branches costs nothing.)
__device__ __forceinline__ float sp_dist(float z, const SampleLocals& s) {
  if (s.inf) return z == INFINITY ? 0.f : INFINITY;
  return s.m - z;
}

// Eight logits from `at` as they are (those from `end` on are -inf), and as numbers.
template <typename T>
struct SampleUnit {
  T x[SP_UNIT];
  __device__ __forceinline__ void load(const T* row, int at, int end, bool wide) {
    if (wide && at + SP_UNIT <= end) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(x) / 16; ++i) {
        const u32x4 u = ldg(reinterpret_cast<const u32x4*>(row + at) + i);
        __builtin_memcpy(reinterpret_cast<char*>(x) + 16 * i, &u, 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i) x[i] = at + i < end ? row[at + i] : (T)-INFINITY;
    }
  }
  __device__ __forceinline__ void values(float (&z)[SP_UNIT]) const {
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i) z[i] = sp_value((float)x[i]);
  }
};
// f(at, z) for this thread's units of [begin, end), a step of the workgroup at a time, the next step's loads in flight meanwhile. Every
// wave that has a unit there calls it with all its lanes (at >= end: -inf).
template <typename T, int THREADS = SP_THREADS, typename F>
__device__ __forceinline__ void sp_units(const T* row, int begin, int end, bool wide, F f) {
  const int lane0 = (threadIdx.x & ~63) * SP_UNIT;
  int at = begin + threadIdx.x * SP_UNIT;
  SampleUnit<T> now, next;
  now.load(row, at, end, wide);
  constexpr int STEP = THREADS * SP_UNIT;
  for (int wave = begin + lane0; wave < end; wave += STEP, at += STEP) {
    if (wave + STEP < end) next.load(row, at + STEP, end, wide);
    f(at, now);
    now = next;
  }
}

// The bin of d = max - z >= 0 (rounded, but the bins stay in the order of z).
__device__ __forceinline__ uint32_t sp_bin(float d) {
  const int b = (int)(__float_as_uint(d) >> 16);
  return (uint32_t)(min(max(b, (int)SP_BIN0 - 1), (int)SP_BIN0 + SP_BINS - 2) - ((int)SP_BIN0 - 1));
}
// Bins up to b hold what is not at least this (the last bin: everything).
__device__ __forceinline__ float sp_edge(uint32_t b) { return b >= SP_BINS - 1 ? NAN : __uint_as_float((SP_BIN0 + b) << 16); }

// a b + c for a constant c that stays in scalar registers (the compiler copies it into the accumulator of a two-address form
// instead: a third of a weight's instructions).
__device__ __forceinline__ double sp_fma(double a, double b, double c) {
  double d;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
  return d;
}
// (2^44 - 2^24) exp((z - m) / T) as a whole number, m finite: 2^x by its whole part and a polynomial of (1 - 2^-20) 2^f, |f| <= 1/2, of
// degree 10 (through the Chebyshev nodes; off by 2^-51; its first term is exact: a token at the maximum weighs SP_ONE). -inf and NaN
// weigh nothing: they end as x = -46, a quarter of a unit.
__device__ __forceinline__ uint64_t sp_weight_finite(float z, const SampleLocals& s) {
  const double x = fmax(((double)z - (double)s.m) * s.inv_t2, -46.0);
  const double k = rint(x), f = x - k;
  double e = sp_fma(f, 7.072579204325653e-09, 1.0208680564192563e-07);
  e = sp_fma(e, f, 1.3215429984693514e-06);
  e = sp_fma(e, f, 1.5252642714133351e-05);
  e = sp_fma(e, f, 0.00015403515751784687);
  e = sp_fma(e, f, 0.0013333545514292945);
  e = sp_fma(e, f, 0.009618119935044186);
  e = sp_fma(e, f, 0.055504055731604836);
  e = sp_fma(e, f, 0.24022627786125117);
  e = sp_fma(e, f, 0.6931465195232863);
  e = sp_fma(e, f, 1.0 - 0x1p-20);
  // in units of one and rounded to a whole number by the unit of 2^52
  const double y = __builtin_ldexp(e, (int)k + 44) + 4503599627370496.0;
  return (uint64_t)__double_as_longlong(y) & 0xfffffffffffffull;
}
__device__ __forceinline__ uint64_t sp_weight(float z, const SampleLocals& s) {
  if (s.inf) return z == INFINITY ? SP_ONE : 0;
  return sp_weight_finite(z, s);
}
__device__ __forceinline__ bool sp_high(float z, const SampleLocals& s) {  // min-p
  if (s.inf) return !s.cut_low || z == INFINITY;
  return !s.cut_low || ((double)z - (double)s.m) * s.inv_t >= s.low;
}

// Sums of whole numbers over a wave, inclusive in lane order (by row moves, no LDS: 16, then across the rows), and the whole.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t wave_moved_u64(uint64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
  return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
  v += wave_moved_u64<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
  v += wave_moved_u64<0x112, 0xf>(v);
  v += wave_moved_u64<0x114, 0xf>(v);
  v += wave_moved_u64<0x118, 0xf>(v);
  v += wave_moved_u64<0x142, 0xa>(v);  // lane 15 of rows 0 and 2 to rows 1 and 3
  v += wave_moved_u64<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
  return v;
}
__device__ __forceinline__ uint64_t wave_last_u64(uint64_t v) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
}
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) { return wave_last_u64(wave_scan_u64(v)); }
// The same over a workgroup in thread order (*total the whole), and the whole alone: eight lanes add the eight waves' sums.
static_assert(SP_THREADS / 64 == 8, "a wave's sum a lane of half a row");
__device__ __forceinline__ uint64_t row_sum_u64(uint64_t v) {  // of values that repeat after eight lanes
  v += wave_moved_u64<0x124, 0xf>(v);  // row_ror:4, 2, 1
  v += wave_moved_u64<0x122, 0xf>(v);
  return v + wave_moved_u64<0x121, 0xf>(v);
}
__device__ __forceinline__ uint64_t block_scan_u64(uint64_t v, uint64_t* scratch, uint64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan_u64(v);
  if (lane == 63) scratch[wave] = v;
  __syncthreads();
  const uint64_t w = scratch[lane & 7];
  *total = row_sum_u64(w);
  v += row_sum_u64((lane & 7) < wave ? w : 0);
  __syncthreads();  // (the scratch is free again)
  return v;
}
__device__ __forceinline__ uint64_t block_sum_u64(uint64_t v, uint64_t* scratch) {
  v = wave_sum_u64(v);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  v = row_sum_u64(scratch[threadIdx.x & 7]);
  __syncthreads();
  return v;
}
__device__ __forceinline__ void sp_add(uint64_t* to, uint64_t v) {
  atomicAdd(reinterpret_cast<unsigned long long*>(to), (unsigned long long)v);
}

template <typename T>
__device__ __forceinline__ const T* sp_row(const SampleParams& p, int row) {
  return static_cast<const T*>(p.logits) + (size_t)row * p.stride;
}
__device__ __forceinline__ uint64_t sp_limit(float p, uint64_t whole) {  // of weight in front of a kept token: less than this
  return max((uint64_t)ceil((double)p * (double)whole), (uint64_t)1);
}

// The row's settings without its maximum.
__device__ __forceinline__ SampleLocals sp_settings(const SampleParams& p, int row) {
  SampleLocals s = {};
  const float t = p.temperature ? ldc(p.temperature + row) : p.temperature_all;
  s.greedy = !(t > 0.f);
  s.inv_t = s.greedy ? 1.0 : 1.0 / (double)t;
  s.inv_t2 = s.inv_t * 1.4426950408889634074;
  s.k = p.top_k ? ldc(p.top_k + row) : p.top_k_all;
  if (s.k <= 0 || s.k >= p.V) s.k = 0;
  s.p = p.top_p ? ldc(p.top_p + row) : p.top_p_all;
  if (!(s.p < 1.f)) s.p = 1.f;
  s.p = fmaxf(s.p, 0.f);
  const float low = p.min_p ? ldc(p.min_p + row) : p.min_p_all;
  s.cut_low = low > 0.f;
  s.low = s.cut_low ? log((double)fminf(low, 1.f)) : 0.0;
  return s;
}
// Sets the row's maximum (after sample_max; every lane of a wave together, the same in all).
__device__ __forceinline__ void sp_maximum(const SampleParams& p, int row, SampleLocals& s) {
  uint64_t key = 0;
  for (int i = threadIdx.x & 63; i < p.P; i += 64) key = max(key, ldg(p.part_key + (size_t)row * p.P + i));
  key = wave_max_u64(key);
  s.m = sp_logit((uint32_t)(key >> 32));
  s.first = sp_index(key);
  s.empty = !(s.m > -INFINITY);
  s.inf = s.m == INFINITY;
}
// A record that an earlier launch wrote, the same in every lane.
template <typename T>
__device__ __forceinline__ T sp_read(const T* from) {
  T x;
  uint32_t w[sizeof(T) / 4];
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); ++i) w[i] = ldc(reinterpret_cast<const uint32_t*>(from) + i);
  __builtin_memcpy(&x, w, sizeof(T));
  return x;
}

// What a row's workgroups leave for the last of them goes past the XCDs' own L2s, by atomic adds and these; a fence would write a whole L2
// back in every workgroup (measured: 9 rows of 128000 tokens 102 -> 40 us without).
template <typename T>
__device__ __forceinline__ void sp_put(T* to, T v) {
  __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T sp_get(const T* from) {
  return __hip_atomic_load(const_cast<T*>(from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// One of a row's parts is done: everything this workgroup put and added has arrived before its own arrival counts. True in the last one.
__device__ __forceinline__ bool sp_last(uint32_t* mark, int parts) {
  __shared__ uint32_t arrived;
  __builtin_amdgcn_s_waitcnt(0);
  asm volatile("" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) arrived = atomicAdd(mark, 1u);
  __syncthreads();
  return arrived == (uint32_t)parts - 1;
}

template <typename T>
__global__ __launch_bounds__(SP_MAX_THREADS) void sample_max_kernel(SampleParams p) {
  const int part = blockIdx.x % p.P, row = blockIdx.x / p.P;
  const T* z0 = sp_row<T>(p, row);
  const int end = min((part + 1) * p.ps, p.V);
  const SampleLocals s = sp_settings(p, row);
  const bool sums = !s.greedy && s.k == 0 && s.p < 1.f;  // (what sample_hist makes use of)
  const float c = (float)s.inv_t2;
  for (int i = part * SP_MAX_THREADS + threadIdx.x; i < SP_BINS; i += p.P * SP_MAX_THREADS) {
    p.hist_count[(size_t)row * SP_BINS + i] = 0;
    p.hist_mass[(size_t)row * SP_BINS + i] = 0;
  }
  if (part == 0 && threadIdx.x < 2) p.marks[row * 2 + threadIdx.x] = 0;
  if (part == 0 && threadIdx.x == 2) p.whole[row] = p.taken[row] = 0;
  if (part == 0 && threadIdx.x == 3) p.rows[row].s = s;
  float top = -3e38f, sum = 0.f;  // this thread's maximum and its weight in units of that one's
  uint32_t at_top = 0xffffffffu;
  bool none = true;
  sp_units<T, SP_MAX_THREADS>(z0, part * p.ps, end, p.wide, [&](int at, const SampleUnit<T>& x) {
    float z[SP_UNIT], u = -INFINITY;
    int i0 = 0;
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i) {
      z[i] = sp_value((float)x.x[i]);
      if (z[i] > u) {
        u = z[i];
        i0 = i;
      }
    }
    if (u > top || (none && u > -INFINITY)) {
      sum *= fast_exp2((top - u) * c);
      top = u;
      at_top = at + i0;
      none = false;
    }
    if (sums)
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i) sum += fast_exp2((z[i] - top) * c);
  });
  __shared__ uint64_t best[4];
  __shared__ float weight[4];
  const uint64_t mine = none ? 0 : argmax_key(top, at_top);
  uint64_t key = wave_max_u64(mine);
  if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = key;
  __syncthreads();
  key = max(max(best[0], best[1]), max(best[2], best[3]));
  if (sums) {
    const float w = wave_sum(none ? 0.f : sum * fast_exp2((top - sp_logit((uint32_t)(key >> 32))) * c));
    if ((threadIdx.x & 63) == 0) weight[threadIdx.x >> 6] = w;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    p.part_key[(size_t)row * p.P + part] = key;
    if (sums) p.part_sum[(size_t)row * p.P + part] = (weight[0] + weight[1]) + (weight[2] + weight[3]);
  }
}

template <typename T>
__global__ __launch_bounds__(SP_THREADS, SP_WAVES) void sample_hist_kernel(SampleParams p) {
  __shared__ uint64_t mass[SP_BINS];  // top-p
  uint32_t* const count = reinterpret_cast<uint32_t*>(mass);  // top-k
  __shared__ uint64_t scratch[SP_THREADS / 64];
  __shared__ uint32_t cut_at;
  const int part = blockIdx.x % p.P2, row = blockIdx.x / p.P2, lane = threadIdx.x & 63;
  SampleLocals s = sp_read(&p.rows[row].s);
  sp_maximum(p, row, s);
  const T* z0 = sp_row<T>(p, row);
  const int begin = part * p.ps2, end = min(begin + p.ps2, p.V);
  const bool all_kept = s.k == 0 && s.p >= 1.f;  // (but what min-p cuts)
  if (s.empty || s.greedy || s.inf || all_kept) {
    // (an infinite maximum is rare: by the general way, so that the loops need not ask)
    SampleRow r = {};
    r.mode = s.empty ? SP_EMPTY : s.greedy ? SP_GREEDY : s.inf ? SP_ROW : SP_ALL;
    r.s = s;
    if (part == 0 && threadIdx.x == 0) p.result[row] = r;
    if (r.mode != SP_ALL) return;
    // the kept weight by chunks
    uint32_t number = 0;
    sp_units<T>(z0, begin, end, p.wide, [&](int at, const SampleUnit<T>& x) {
      float z[SP_UNIT];
      x.values(z);
      uint64_t sum = 0;
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i) {
        const bool in = z[i] > -INFINITY && sp_high(z[i], s);
        sum += in ? sp_weight_finite(z[i], s) : 0;
        number += in;
      }
      sum = wave_sum_u64(sum);
      if (lane == 0) p.chunk_sum[(size_t)row * p.chunks + at / SP_CHUNK] = sum;
    });
    number = (uint32_t)block_sum_u64(number, scratch);
    if (threadIdx.x == 0 && number) sp_add(p.taken + row, (uint64_t)number << 32);
    return;
  }
  for (int i = threadIdx.x; i < SP_BINS; i += SP_THREADS) mass[i] = 0;
  __syncthreads();
  // Tokens past `far` are in no cut and need no bin. Top-p: those lighter than (1 - p) / V of the whole weigh less than 1 - p of
  // it together, so the cut is above them (a thousandth less, for what fp32 sums and the logarithm lose). Top-k: what is
  // past a bin that k tokens of this part reach, looked up once the first step is through.
  const bool by_k = s.k > 0;
  float far = INFINITY;
  if (!by_k) {
    float whole = 0.f;
    const float c = (float)s.inv_t2;
    for (int i = lane; i < p.P; i += 64) {
      const uint64_t key = ldg(p.part_key + (size_t)row * p.P + i);
      if (key) whole += ldg(p.part_sum + (size_t)row * p.P + i) * fast_exp2((sp_logit((uint32_t)(key >> 32)) - s.m) * c);
    }
    whole = wave_sum(whole);
    const float x = log2f((1.f - s.p) * whole * 0.999f / (float)p.V);
    if (x < 0.f) far = -x / c;  // (not where it is no number)
  }
  uint64_t all = 0;
  if (by_k) {
    auto add = [&](int, const SampleUnit<T>& x) {
      float z[SP_UNIT];
      x.values(z);
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i) {
        const float d = s.m - z[i];
        if (z[i] > -INFINITY && d <= far) atomicAdd(&count[sp_bin(d)], 1u);
      }
    };
    const int first = min(begin + SP_STEP, end);
    sp_units<T>(z0, begin, first, p.wide, add);
    if (first < end) {
      if (threadIdx.x == 0) cut_at = SP_BINS;
      __syncthreads();
      constexpr int EACH = SP_BINS / SP_THREADS;
      uint64_t n = 0, total;
#pragma unroll
      for (int i = 0; i < EACH; ++i) n += count[threadIdx.x * EACH + i];
      const uint64_t before = block_scan_u64(n, scratch, &total) - n;
      if (before < (uint64_t)s.k && before + n >= (uint64_t)s.k) cut_at = threadIdx.x * EACH + EACH - 1;  // (its bins whole)
      __syncthreads();
      if (cut_at < SP_BINS - 1) far = sp_edge(cut_at);
      sp_units<T>(z0, first, end, p.wide, add);
    }
  } else {
    sp_units<T>(z0, begin, end, p.wide, [&](int, const SampleUnit<T>& x) {
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i) {
        const float z = (float)x.x[i];
        const uint64_t w = sp_weight_finite(z, s);  // (0 for a NaN)
        const float d = s.m - z;
        all += w;
        if (d <= far) sp_add(&mass[sp_bin(d)], w);
      }
    });
  }
  if (!by_k) {
    all = block_sum_u64(all, scratch);
    if (threadIdx.x == 0) sp_add(&p.whole[row], all);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < SP_BINS; i += SP_THREADS) {
    if (by_k && count[i]) atomicAdd(&p.hist_count[(size_t)row * SP_BINS + i], count[i]);
    if (!by_k && mass[i]) sp_add(&p.hist_mass[(size_t)row * SP_BINS + i], mass[i]);
  }
  if (!sp_last(&p.marks[row * 2], p.P2)) return;

  // The bin of the cut, by the sums before each thread's bins.
  constexpr int EACH = SP_BINS / SP_THREADS;
  uint64_t n[EACH], ns = 0, seen;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const size_t b = (size_t)row * SP_BINS + threadIdx.x * EACH + i;
    n[i] = by_k ? sp_get(p.hist_count + b) : sp_get(p.hist_mass + b);
    ns += n[i];
  }
  const uint64_t whole = by_k ? 0 : sp_get(p.whole + row);
  uint64_t before = block_scan_u64(ns, scratch, &seen) - ns;
  SampleRow r = {};
  r.s = s;
  r.by_mass = !by_k;
  r.limit = by_k ? (uint64_t)s.k : sp_limit(s.p, whole);
  if (seen < r.limit) {  // fewer live tokens than top-k keeps: all of them stay
    if (threadIdx.x == 0) {
      r.bin = SP_BINS - 1;
      r.mode = by_k && seen <= SP_LIST ? SP_LISTED : SP_ROW;
      p.result[row] = r;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (before < r.limit && before + n[i] >= r.limit) {  // (one thread, one bin)
      r.bin = threadIdx.x * EACH + i;
      r.above = before;
      const uint64_t to = before + n[i];
      // (top-p behind a top-k of more than a list's tokens: its part of the whole is of what top-k leaves)
      r.mode = !by_k || (s.p >= 1.f && to > SP_SMALL) ? SP_BELOW : to <= (s.p < 1.f ? SP_LIST : SP_SMALL) ? SP_LISTED : SP_ROW;
      p.result[row] = r;
    }
    before += n[i];
  }
}

// The row's outputs (one thread).
__device__ __forceinline__ void sp_store(const SampleParams& p, int row, int token, float z, uint64_t kept, uint64_t w, uint64_t whole) {
  if (p.tokens) p.tokens[row] = token;
  if (p.keys) p.keys[row] = token < 0 ? 0 : argmax_key(z, (uint32_t)token);
  if (p.kept) p.kept[row] = (int)kept;
  if (p.logprob) p.logprob[row] = (float)log((double)w / (double)whole);
}
// How much weight lies in front of the draw.
__device__ __forceinline__ uint64_t sp_target(const SampleRow& r, uint64_t whole) {
  const float u = r.u;
  const double x = u > 0.f ? (double)fminf(u, 1.f - 0x1p-24f) * (double)whole : 0.0;
  return x < (double)(whole - 1) ? (uint64_t)x : whole - 1;
}

// What is kept so far: keys above `key`, or equal to it with index <= idx.
struct SampleCut {
  uint32_t key, idx;
  __device__ __forceinline__ bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= idx); }
};

// What the helpers below share. Each may write any of it at once, so whoever reads a word has a barrier between that and the next helper:
// its own before it returns false, the sums' of the code behind it after sp_rank and a narrowed list.
struct SampleShared {
  alignas(16) uint64_t mass[256];
  alignas(16) uint64_t key[SP_SMALL];
  uint32_t count[256];
  uint64_t scratch[SP_THREADS / 64];
  uint64_t c, w;
  uint32_t digit, found, at, number;
};

// The tokens of a list (argmax keys in LDS) or of the whole row, in any order.
struct SampleList {
  const uint64_t* key;
  int n;
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int i = threadIdx.x; i < n; i += SP_THREADS) f(sp_index(key[i]), sp_logit((uint32_t)(key[i] >> 32)));
  }
};
template <typename T>
struct SampleWhole {
  const T* z0;
  int V;
  bool wide;
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    sp_units<T>(z0, 0, V, wide, [&](int at, const SampleUnit<T>& x) {
      float z[SP_UNIT];
      x.values(z);
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i)
        if (z[i] > -INFINITY) f((uint32_t)(at + i), z[i]);
    });
  }
};

// Among the tokens that of(idx, z, &order) takes, ranked by `order` descending, behind `c` tokens of weight `w`: the order at which the
// tokens (by_mass: their weight) reach `limit`, by digits of eight bits. c and w become what stands in front of that order, `key` the
// order; false: they never reach it.
template <typename Items, typename Of>
__device__ __forceinline__ bool sp_descend(const Items& it, const SampleLocals& s, SampleShared& sh, bool by_mass, uint64_t limit, uint64_t& c,
                                           uint64_t& w, uint32_t& key, Of of) {
  // the bits in which the orders differ
  if (threadIdx.x == 0) sh.digit = 0, sh.found = 0xffffffffu;
  __syncthreads();
  uint32_t any = 0, every = 0xffffffffu;
  it.each([&](uint32_t idx, float z) {
    uint32_t o;
    if (of(idx, z, o)) any |= o, every &= o;
  });
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    any |= __shfl_xor(any, d);
    every &= __shfl_xor(every, d);
  }
  if ((threadIdx.x & 63) == 0) {
    atomicOr(&sh.digit, any);
    atomicAnd(&sh.found, every);
  }
  __syncthreads();
  any = sh.digit;
  every = sh.found;
  const uint32_t differ = any & ~every;
  int hi = differ ? 32 - __clz(differ) : 0;       // bits from hi up are the same everywhere
  const int lo = differ ? __ffs(differ) - 1 : 0;  // and those below lo
  uint32_t prefix = every;                        // right outside [lo, hi)
  __syncthreads();
  do {
    const int shift = max(hi - 8, lo), bits = hi - shift;
    const uint32_t mask = bits ? (0xffffffffu >> (32 - bits)) << shift : 0;
    const uint32_t above = hi < 32 ? 0xffffffffu << hi : 0;  // bits already settled
    if (threadIdx.x < 256) sh.mass[threadIdx.x] = sh.count[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.found = 0;
    __syncthreads();
    it.each([&](uint32_t idx, float z) {
      uint32_t o;
      if (!of(idx, z, o) || ((o ^ prefix) & above)) return;
      const uint32_t d = 255 - ((o & mask) >> shift);  // the largest digit first
      atomicAdd(&sh.count[d], 1u);
      if (by_mass) sp_add(&sh.mass[d], sp_weight(z, s));
    });
    __syncthreads();
    const bool digit = threadIdx.x < 256;
    const uint64_t hc = digit ? sh.count[threadIdx.x] : 0, hw = digit ? sh.mass[threadIdx.x] : 0;
    uint64_t total;
    const uint64_t c1 = c + block_scan_u64(hc, sh.scratch, &total), w1 = by_mass ? w + block_scan_u64(hw, sh.scratch, &total) : 0;
    if (by_mass ? w1 - hw < limit && w1 >= limit : c1 - hc < limit && c1 >= limit) {
      sh.digit = 255 - threadIdx.x;
      sh.c = c1 - hc;
      sh.w = w1 - hw;
      sh.found = 1;
    }
    __syncthreads();
    const bool found = sh.found != 0;
    const uint32_t at = sh.digit;
    const uint64_t c0 = sh.c, w0 = sh.w;
    __syncthreads();  // (read by every wave before any of them goes on, or back to the caller)
    if (!found) return false;
    prefix = (prefix & ~mask) | (at << shift & mask);
    c = c0;
    w = w0;
    hi = shift;
  } while (hi > lo);
  key = prefix;
  return true;
}

// Shrinks `cut` to the first `limit` tokens, or (by_mass) to those with less than `limit` weight in front of them, of the items it keeps,
// `c` tokens of weight `w` standing in front of all of them.
template <typename Items>
__device__ __forceinline__ void sp_shrink(const Items& it, const SampleLocals& s, SampleShared& sh, SampleCut& cut, bool by_mass, uint64_t limit,
                                          uint64_t c, uint64_t w) {
  uint32_t key;
  const SampleCut old = cut;
  if (!sp_descend(it, s, sh, by_mass, limit, c, w, key, [&](uint32_t idx, float z, uint32_t& o) {
        o = argmax_ord(z);
        return old.keeps(o, idx);
      }))
    return;
  // of the tokens of this key the first `more`, by index
  const uint64_t wt = by_mass ? sp_weight(sp_logit(key), s) : 0;
  const uint64_t more = by_mass ? (limit - w + wt - 1) / max(wt, (uint64_t)1) : limit - c;
  uint64_t c2 = 0, w2 = 0;
  uint32_t inv;
  cut.key = key;
  cut.idx = key == old.key ? old.idx : 0xffffffffu;
  if (sp_descend(it, s, sh, false, more, c2, w2, inv, [&](uint32_t idx, float z, uint32_t& o) {
        o = ~idx;
        return argmax_ord(z) == key && old.keeps(key, idx);
      }))
    cut.idx = ~inv;
}

// The draw among items that the cut and min-p keep.
template <typename Items>
__device__ __forceinline__ void sp_draw(const SampleParams& p, int row, const Items& it, const SampleRow& r, SampleShared& sh, const SampleCut& cut) {
  const SampleLocals& s = r.s;
  uint64_t whole = 0, kept = 0;
  it.each([&](uint32_t idx, float z) {
    if (!cut.keeps(argmax_ord(z), idx) || !sp_high(z, s)) return;
    whole += sp_weight(z, s);
    ++kept;
  });
  whole = block_sum_u64(whole, sh.scratch);
  kept = block_sum_u64(kept, sh.scratch);
  const uint64_t target = sp_target(r, whole);
  uint64_t c = 0, w = 0;
  uint32_t inv;
  sp_descend(it, s, sh, true, target + 1, c, w, inv, [&](uint32_t idx, float z, uint32_t& o) {
    o = ~idx;
    return cut.keeps(argmax_ord(z), idx) && sp_high(z, s);
  });
  it.each([&](uint32_t idx, float z) {
    if (idx == ~inv) sp_store(p, row, (int)idx, z, kept, sp_weight(z, s), whole);
  });
}

// All of the cuts and the draw among items that hold every token that may be kept.
template <typename Items>
__device__ __forceinline__ void sp_finish(const SampleParams& p, int row, const Items& it, const SampleRow& r, SampleShared& sh) {
  const SampleLocals& s = r.s;
  SampleCut cut = {0, 0xffffffffu};
  if (s.k) sp_shrink(it, s, sh, cut, false, (uint64_t)s.k, 0, 0);
  if (s.p < 1.f) {
    uint64_t whole = 0;
    it.each([&](uint32_t idx, float z) { whole += cut.keeps(argmax_ord(z), idx) ? sp_weight(z, s) : 0; });
    whole = block_sum_u64(whole, sh.scratch);
    sp_shrink(it, s, sh, cut, true, sp_limit(s.p, whole), 0, 0);
  }
  sp_draw(p, row, it, r, sh, cut);
}

// Of at most SP_SMALL tokens each thread has one (the argmax key, 0: none; its weight). All of them into sh.key and sh.mass, the rest
// of either zeros; then f(key, weight) of each, four at a time (read one by one they are a chain of LDS latencies).
static_assert(SP_SMALL == 256, "sh.mass");
__device__ __forceinline__ void sp_lay(SampleShared& sh, uint64_t key, uint64_t w) {
  if (threadIdx.x < SP_SMALL) {
    sh.key[threadIdx.x] = key;
    sh.mass[threadIdx.x] = w;
  }
  __syncthreads();
}
template <typename F>
__device__ __forceinline__ void sp_all(const SampleShared& sh, int n, F f) {
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
#pragma unroll 2
  for (int j = 0; j < n; j += 4) {
    u64x2 k[2], w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      k[i] = *reinterpret_cast<const u64x2*>(sh.key + j + 2 * i);
      w[i] = *reinterpret_cast<const u64x2*>(sh.mass + j + 2 * i);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f((uint64_t)k[i / 2][i % 2], (uint64_t)w[i / 2][i % 2]);
  }
}

// Of at most SP_SMALL tokens, `above` (tokens or weight) standing in front of all of them: the cut after `limit`. All with all.
__device__ __forceinline__ SampleCut sp_rank(const SampleList& it, const SampleLocals& s, SampleShared& sh, bool by_mass, uint64_t limit,
                                             uint64_t above) {
  const int i = threadIdx.x;
  const bool there = i < it.n, has = (i & ~63) < it.n;  // (waves without a token stay out of the loop)
  const uint64_t key = there ? it.key[i] : 0;
  sp_lay(sh, key, !there ? 0 : by_mass ? sp_weight(sp_logit((uint32_t)(key >> 32)), s) : 1);
  uint32_t rank = 0;
  uint64_t before = above;
  if (has) sp_all(sh, it.n, [&](uint64_t k, uint64_t w) {
    rank += k > key;
    before += k > key ? w : 0;
  });
  const bool keep = there && before < limit;
  const uint64_t kept = block_sum_u64(keep, sh.scratch);
  if (keep && rank == (uint32_t)kept - 1) {  // the last of them
    sh.digit = (uint32_t)(key >> 32);
    sh.at = sp_index(key);
  }
  __syncthreads();
  return SampleCut{sh.digit, sh.at};
}

// Of a longer list the tokens between max - d0 and max - d1 that hold the cut after `limit`: a 256th of the way, to `small`. above becomes what stands in front of them; false if they are more than SP_SMALL.
__device__ __forceinline__ bool sp_narrow(const SampleList& it, const SampleLocals& s, SampleShared& sh, bool by_mass, uint64_t limit, uint64_t& above,
                                          float d0, float d1, uint64_t* small, int* n) {
  if (!(d1 < INFINITY)) return false;
  const float scale = 256.f / (d1 - d0);
  auto of = [&](float z) { return (int)fminf(fmaxf((sp_dist(z, s) - d0) * scale, 0.f), 255.f); };
  if (threadIdx.x < 256) sh.mass[threadIdx.x] = sh.count[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.number = 0;
  __syncthreads();
  it.each([&](uint32_t, float z) {
    const int b = of(z);
    atomicAdd(&sh.count[b], 1u);
    if (by_mass) sp_add(&sh.mass[b], sp_weight(z, s));
  });
  __syncthreads();
  const uint64_t mine = threadIdx.x >= 256 ? 0 : by_mass ? sh.mass[threadIdx.x] : sh.count[threadIdx.x];
  uint64_t total;
  const uint64_t after = above + block_scan_u64(mine, sh.scratch, &total);
  if (after >= limit && after - mine < limit) {  // (one thread)
    sh.digit = threadIdx.x;
    sh.c = after - mine;
  }
  __syncthreads();
  const int bin = (int)sh.digit;
  const uint32_t size = sh.count[bin];
  __syncthreads();  // (read by every wave before one goes back to the caller, whose next helper clears sh.digit)
  if (size > SP_SMALL) return false;
  it.each([&](uint32_t i, float z) {
    if (of(z) != bin) return;
    const uint32_t to = atomicAdd(&sh.number, 1u);
    small[to] = argmax_key(z, i);
  });
  __syncthreads();
  above = sh.c;
  *n = (int)sh.number;
  return true;
}

// The cuts and the draw of a list of at most SP_SMALL tokens, of which top-k keeps some or all.
__device__ __forceinline__ void sp_small(const SampleParams& p, int row, const SampleList& it, const SampleRow& r, SampleShared& sh) {
  const SampleLocals& s = r.s;
  const int i = threadIdx.x;
  const bool there = i < it.n, has = (i & ~63) < it.n;
  const uint64_t key = there ? it.key[i] : 0;
  const float z = sp_logit((uint32_t)(key >> 32));
  const uint64_t w = there ? sp_weight(z, s) : 0;
  sp_lay(sh, key, w);
  uint32_t rank = 0;
  uint64_t before = 0;
  if (has) sp_all(sh, it.n, [&](uint64_t k, uint64_t x) {
    rank += k > key;
    before += k > key ? x : 0;
  });
  bool keep = there && rank < (uint32_t)s.k;
  if (s.p < 1.f) {
    const uint64_t limit = sp_limit(s.p, block_sum_u64(keep ? w : 0, sh.scratch));  // (every thread)
    keep = keep && before < limit;
  }
  keep = keep && sp_high(z, s);
  __syncthreads();
  if (i < SP_SMALL) sh.mass[i] = keep ? w : 0;
  const uint64_t whole = block_sum_u64(keep ? w : 0, sh.scratch), kept = block_sum_u64(keep, sh.scratch);
  const uint64_t target = sp_target(r, whole);
  uint64_t sum = 0;
  if (has) sp_all(sh, it.n, [&](uint64_t k, uint64_t x) { sum += (uint32_t)k > (uint32_t)key ? x : 0; });  // (lower indexes: larger low words)
  if (keep && sum <= target && sum + w > target) sp_store(p, row, (int)sp_index(key), z, kept, w, whole);
}

// The draw where the kept weight lies by chunks (in LDS): the chunk, then its tokens, by one wave.
template <typename T, typename Keep>
__device__ __forceinline__ void sp_draw_chunk(const SampleParams& p, int row, const T* z0, uint64_t* sums, uint64_t kept, const SampleRow& r,
                                              SampleShared& sh, Keep keep) {
  const SampleLocals& s = r.s;
  constexpr int EACH = SP_CHUNKS / SP_THREADS;
  uint64_t mine = 0, whole;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int c = threadIdx.x * EACH + i;
    mine += c < p.chunks ? sums[c] : 0;
  }
  uint64_t before = block_scan_u64(mine, sh.scratch, &whole) - mine;
  const uint64_t target = sp_target(r, whole);
  if (before <= target && before + mine > target) {  // (one thread)
    int c = threadIdx.x * EACH;
    while (before + sums[c] <= target) before += sums[c++];
    sh.at = c;
    sh.c = before;
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const int at = sh.at * SP_CHUNK + threadIdx.x * SP_UNIT;
  SampleUnit<T> x;
  float z[SP_UNIT];
  uint64_t w[SP_UNIT], run = 0;
  x.load(z0, at, p.V, p.wide);
  x.values(z);
#pragma unroll
  for (int i = 0; i < SP_UNIT; ++i) {
    w[i] = z[i] > -INFINITY && keep((uint32_t)(at + i), z[i]) && sp_high(z[i], s) ? sp_weight(z[i], s) : 0;
    run += w[i];
  }
  uint64_t sum = wave_scan_u64(run);
  sum += sh.c - run;
#pragma unroll
  for (int i = 0; i < SP_UNIT; ++i) {
    if (sum <= target && sum + w[i] > target) sp_store(p, row, at + i, z[i], kept, w[i], whole);
    sum += w[i];
  }
}

// A row whose bin, max - z from d0 to d1, holds more tokens than a list (`sums`: the kept weight above the bin by chunks, of `kept`
// tokens): the bin in 1024 parts, one pass to find the cut's part and one to list it. A part of more tokens than a list are equal
// logits in all likelihood (bfloat16 has 33 values between 32 and 40): then their numbers by chunks say which is the last one kept.
// False if they are not, or the bin is the last.
constexpr int SP_SUB = 1024;
static_assert(SP_SUB * 12 <= SP_LIST * 8 && SP_CHUNKS * 4 <= SP_LIST * 8, "in the list's place");
template <typename T>
__device__ __forceinline__ bool sp_crowded(const SampleParams& p, int row, const T* z0, const SampleRow& r, float d0, float d1, uint64_t* list,
                                           uint64_t* sums, uint64_t kept, SampleShared& sh) {
  if (!(d1 < INFINITY)) return false;
  const SampleLocals& s = r.s;
  const bool by_mass = r.by_mass != 0;
  const int lane = threadIdx.x & 63;
  const float scale = SP_SUB / (d1 - d0);
  auto of = [&](float d) { return (int)fminf(fmaxf((d - d0) * scale, 0.f), SP_SUB - 1.f); };
  uint32_t* const count = reinterpret_cast<uint32_t*>(list + SP_SUB);
  for (int i = threadIdx.x; i < SP_SUB; i += SP_THREADS) list[i] = count[i] = 0;
  __syncthreads();
  sp_units<T>(z0, 0, p.V, p.wide, [&](int, const SampleUnit<T>& x) {
    float z[SP_UNIT];
    x.values(z);
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i) {
      const float d = s.m - z[i];
      if (!(d >= d0 && d < d1)) continue;
      const int b = of(d);
      atomicAdd(&count[b], 1u);
      if (by_mass) sp_add(&list[b], sp_weight_finite(z[i], s));
    }
  });
  __syncthreads();
  constexpr int EACH = SP_SUB / SP_THREADS;
  uint64_t n[EACH], ns = 0, total;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int b = threadIdx.x * EACH + i;
    n[i] = by_mass ? list[b] : count[b];
    ns += n[i];
  }
  if (threadIdx.x == 0) sh.found = sh.number = 0;
  uint64_t front = r.above + block_scan_u64(ns, sh.scratch, &total) - ns;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (front < r.limit && front + n[i] >= r.limit) {  // (one thread, one part)
      sh.digit = threadIdx.x * EACH + i;
      sh.count[0] = count[threadIdx.x * EACH + i];
      sh.c = front;
      sh.found = 1;
    }
    front += n[i];
  }
  __syncthreads();
  const bool found = sh.found != 0;
  const int part = (int)sh.digit, size = (int)sh.count[0];
  const bool alike = size > SP_LIST;
  uint32_t* const number = reinterpret_cast<uint32_t*>(list);  // (alike) by chunks
  front = sh.c;
  __syncthreads();
  if (!found) return false;  // (the same in every thread)
  if (threadIdx.x == 0) sh.digit = 0, sh.found = 0xffffffffu;
  __syncthreads();
  uint32_t over = 0, any = 0, every = 0xffffffffu;
  sp_units<T>(z0, 0, p.V, p.wide, [&](int at, const SampleUnit<T>& x) {
    float z[SP_UNIT];
    x.values(z);
    uint64_t sum = 0;
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i) {
      const float d = s.m - z[i];
      if (!(d >= d0 && d < d1)) continue;
      const int b = of(d);
      if (b < part && sp_high(z[i], s)) {
        sum += sp_weight_finite(z[i], s);
        ++over;
      }
      if (b != part) continue;
      ++mine;
      if (alike) {
        any |= argmax_ord(z[i]);
        every &= argmax_ord(z[i]);
      } else {
        const uint32_t to = atomicAdd(&sh.number, 1u);
        if (to < SP_LIST) list[to] = argmax_key(z[i], (uint32_t)(at + i));
      }
    }
    sum = wave_sum_u64(sum);
    const uint64_t here = alike ? wave_sum_u64(mine) : 0;
    if (lane == 0) {
      sums[at / SP_CHUNK] += sum;
      if (alike) number[at / SP_CHUNK] = (uint32_t)here;
    }
  });
  kept += block_sum_u64(over, sh.scratch);  // (a barrier too)
  SampleCut cut = {0, 0xffffffffu};
  if (!alike) {
    const SampleList it = {list, size};
    if (size <= SP_SMALL)
      cut = sp_rank(it, s, sh, by_mass, r.limit, front);
    else
      sp_shrink(it, s, sh, cut, by_mass, r.limit, front, front);
    __syncthreads();
    uint64_t more = 0;
    it.each([&](uint32_t i, float z) {
      if (!cut.keeps(argmax_ord(z), i) || !sp_high(z, s)) return;
      sp_add(&sums[i / SP_CHUNK], sp_weight(z, s));
      ++more;
    });
    kept += block_sum_u64(more, sh.scratch);
  } else {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      any |= __shfl_xor(any, d);
      every &= __shfl_xor(every, d);
    }
    if (lane == 0) {
      atomicOr(&sh.digit, any);
      atomicAnd(&sh.found, every);
    }
    __syncthreads();
    cut.key = sh.digit;
    const bool differ = sh.found != cut.key;
    __syncthreads();
    if (differ) return false;
    const float z = sp_logit(cut.key);
    const uint64_t w = sp_weight(z, s), one = by_mass ? max(w, (uint64_t)1) : 1;
    const uint64_t m = min((r.limit - front + one - 1) / one, (uint64_t)size);  // so many of them, by index
    const bool high = sp_high(z, s);
    constexpr int OF = SP_CHUNKS / SP_THREADS;
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < OF; ++i) {
      const int c = threadIdx.x * OF + i;
      mine += c < p.chunks ? number[c] : 0;
    }
    uint64_t before = block_scan_u64(mine, sh.scratch, &total) - mine;
#pragma unroll
    for (int i = 0; i < OF; ++i) {
      const int c = threadIdx.x * OF + i;
      const uint64_t k = c < p.chunks ? number[c] : 0, take = min(k, m - min(m, before));
      if (high && take) sums[c] += take * w;
      if (before < m && before + k >= m) {  // (one thread, one chunk)
        sh.at = c;
        sh.number = (uint32_t)(m - before);
      }
      before += k;
    }
    __syncthreads();
    if (threadIdx.x < 64) {  // the last one kept within its chunk
      const int at = (int)sh.at * SP_CHUNK + lane * SP_UNIT;
      SampleUnit<T> x;
      float v[SP_UNIT];
      uint32_t equal = 0;
      x.load(z0, at, p.V, p.wide);
      x.values(v);
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i) equal |= v[i] == z ? 1u << i : 0u;
      uint32_t rank = (uint32_t)wave_scan_u64(__popc(equal)) - __popc(equal);
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i)
        if (equal >> i & 1 && ++rank == sh.number) sh.digit = at + i;
    }
    __syncthreads();
    cut.idx = sh.digit;
    kept += high ? m : 0;
    __syncthreads();
  }
  sp_draw_chunk<T>(p, row, z0, sums, kept, r, sh, [&](uint32_t i, float z) { return cut.keeps(argmax_ord(z), i); });
  return true;
}

template <typename T>
__global__ __launch_bounds__(SP_THREADS) void sample_pick_kernel(SampleParams p) {
  __shared__ uint64_t list[SP_LIST];
  extern __shared__ uint64_t sums[];  // [chunks]
  __shared__ uint64_t small[SP_SMALL];
  __shared__ SampleShared sh;
  const int part = blockIdx.x % p.P3, row = blockIdx.x / p.P3, lane = threadIdx.x & 63;
  SampleRow r = sp_read(p.result + row);
  r.u = ldc(p.u + row);
  if (part && (r.mode == SP_EMPTY || r.mode == SP_GREEDY || r.mode == SP_ALL || r.mode == SP_ROW)) return;
  const SampleLocals s = r.s;
  const T* z0 = sp_row<T>(p, row);
  if (r.mode == SP_EMPTY || r.mode == SP_GREEDY) {
    if (threadIdx.x == 0) {
      if (r.mode == SP_EMPTY)
        sp_store(p, row, -1, 0.f, 0, 0, 1);
      else
        sp_store(p, row, (int)s.first, s.m, 1, 1, 1);
    }
    return;
  }
  if (r.mode == SP_ALL) {
    for (int c = threadIdx.x; c < p.chunks; c += SP_THREADS) sums[c] = p.chunk_sum[(size_t)row * p.chunks + c];
    __syncthreads();
    sp_draw_chunk<T>(p, row, z0, sums, p.taken[row] >> 32, r, sh, [](uint32_t, float) { return true; });
    return;
  }
  if (r.mode == SP_ROW) {
    sp_finish(p, row, SampleWhole<T>{z0, p.V, p.wide != 0}, r, sh);
    return;
  }
  // This part's tokens for the list, and (SP_BELOW) the kept weight above the bin by chunks
  const int begin = part * p.ps3, end = min(begin + p.ps3, p.V);
  const bool listed = r.mode == SP_LISTED;
  const float edge = sp_edge(r.bin), inner = r.bin ? sp_edge(r.bin - 1) : 0.f;  // (bin 0 has nothing above it)
  if (threadIdx.x == 0) sh.number = 0;
  __syncthreads();
  uint32_t number = 0;
  sp_units<T>(z0, begin, end, p.wide, [&](int at, const SampleUnit<T>& x) {
    float z[SP_UNIT];
    x.values(z);
    uint32_t take = 0, over = 0;
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i) {
      const float d = s.m - z[i];
      const bool up = z[i] > -INFINITY && !(d >= edge), above = !listed && r.bin && !(d >= inner);
      take |= up && !above ? 1u << i : 0u;
      over |= up && above ? 1u << i : 0u;
    }
    if (__builtin_amdgcn_ballot_w64(take != 0)) {  // the wave's ones side by side
      const uint32_t mine = (uint32_t)__popc(take);
      const uint64_t upto = wave_scan_u64(mine);
      uint32_t to = 0;
      if (lane == 63) to = atomicAdd(&sh.number, (uint32_t)upto);
      to = (uint32_t)__builtin_amdgcn_readlane((int)to, 63) + (uint32_t)upto - mine;
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i)
        if (take >> i & 1) {
          if (to < SP_LIST) list[to] = argmax_key(z[i], (uint32_t)(at + i));
          ++to;
        }
    }
    if (!listed) {
      uint64_t sum = 0;
      if (__builtin_amdgcn_ballot_w64(over != 0)) {
#pragma unroll
        for (int i = 0; i < SP_UNIT; ++i) {
          const bool in = (over >> i & 1) && sp_high(z[i], s);
          sum += in ? sp_weight_finite(z[i], s) : 0;
          number += in;
        }
        sum = wave_sum_u64(sum);
      }
      if (lane == 0) sp_put(p.chunk_sum + (size_t)row * p.chunks + at / SP_CHUNK, sum);
    }
  });
  number = (uint32_t)block_sum_u64(number, sh.scratch);  // (a barrier too)
  const uint32_t here = sh.number;
  if (threadIdx.x == 0)
    sh.at = here || number ? (uint32_t)atomicAdd(reinterpret_cast<unsigned long long*>(p.taken + row), (unsigned long long)number << 32 | here) : 0;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < here && sh.at + i < SP_LIST; i += SP_THREADS) sp_put(p.list + (size_t)row * SP_LIST + sh.at + i, list[i]);
  if (!sp_last(&p.marks[row * 2 + 1], p.P3)) return;

  // The last part finishes the row
  const uint64_t taken = sp_get(p.taken + row);
  if (!listed)
    for (int c = threadIdx.x; c < p.chunks; c += SP_THREADS) sums[c] = sp_get(p.chunk_sum + (size_t)row * p.chunks + c);
  const int n = (int)(uint32_t)taken;
  if (n > SP_LIST) {
    if (!sp_crowded<T>(p, row, z0, r, r.bin ? inner : 0.f, edge, list, sums, taken >> 32, sh)) sp_finish(p, row, SampleWhole<T>{z0, p.V, p.wide != 0}, r, sh);
    return;
  }
  const uint64_t first = sp_get(p.list + (size_t)row * SP_LIST + threadIdx.x);  // (there or not: asked for along with their number)
  if ((int)threadIdx.x < n) list[threadIdx.x] = first;
  for (int i = threadIdx.x + SP_THREADS; i < n; i += SP_THREADS) list[i] = sp_get(p.list + (size_t)row * SP_LIST + i);
  __syncthreads();
  const SampleList it = {list, n};
  if (listed && n <= SP_SMALL) {
    sp_small(p, row, it, r, sh);
    return;
  }
  if (listed) {  // more than SP_SMALL tokens, by top-k
    sp_finish(p, row, it, r, sh);
    return;
  }
  SampleCut cut = {0, 0xffffffffu};
  SampleList few = {small, 0};
  uint64_t front = r.above;
  if (n <= SP_SMALL)
    cut = sp_rank(it, s, sh, r.by_mass != 0, r.limit, front);
  else if (sp_narrow(it, s, sh, r.by_mass != 0, r.limit, front, r.bin ? inner : 0.f, edge, small, &few.n))
    cut = sp_rank(few, s, sh, r.by_mass != 0, r.limit, front);
  else
    sp_shrink(it, s, sh, cut, r.by_mass != 0, r.limit, r.above, r.above);
  uint64_t more = 0;
  it.each([&](uint32_t i, float z) {
    if (!cut.keeps(argmax_ord(z), i) || !sp_high(z, s)) return;
    sp_add(&sums[i / SP_CHUNK], sp_weight(z, s));
    ++more;
  });
  more = block_sum_u64(more, sh.scratch);
  sp_draw_chunk<T>(p, row, z0, sums, (taken >> 32) + more, r, sh, [&](uint32_t i, float z) {
    return (r.bin && !(sp_dist(z, s) >= inner)) || cut.keeps(argmax_ord(z), i);
  });
}

// Parts of a row: up to about 1024 workgroups in each launch, which all run at once, none of less than a step.
void sample_plan(SampleParams& p) {
  auto parts = [&](int step, int most, int& n, int& size) {
    const int steps = (p.V + step - 1) / step;
    const int want = std::min(steps, std::max(1, most / p.n));
    size = (steps + want - 1) / want * step;
    n = (p.V + size - 1) / size;
  };
  parts(SP_MAX_THREADS * SP_UNIT, std::min(1024, SP_PARTS * p.n), p.P, p.ps);
  parts(SP_STEP, 1024, p.P2, p.ps2);
  parts(SP_STEP, 1024, p.P3, p.ps3);
  p.chunks = (p.V + SP_CHUNK - 1) / SP_CHUNK;
}

// Carves the workspace (nullptr: its size alone), the 8-byte pieces first.
size_t sample_workspace(SampleParams& p, void* ws) {
  const size_t n = p.n, parts = n * p.P;
  char* at = static_cast<char*>(ws);
  auto piece = [&](auto*& to, size_t count) {
    to = reinterpret_cast<std::remove_reference_t<decltype(to)>>(at);
    at += count * sizeof(*to);
  };
  piece(p.part_key, parts);
  piece(p.chunk_sum, n * p.chunks);
  piece(p.hist_mass, n * SP_BINS);
  piece(p.whole, n);
  piece(p.taken, n);
  piece(p.list, n * SP_LIST);
  piece(p.rows, n);
  piece(p.result, n);
  piece(p.part_sum, parts);
  piece(p.hist_count, n * SP_BINS);
  piece(p.marks, n * 2);
  return (size_t)(at - static_cast<char*>(ws));
}

int sample_launch(const SampleParams& p, int type, hipStream_t s) {
  const dim3 block(SP_THREADS);
#define SP_GO(T)                                                       \
  do {                                                                 \
    hipLaunchKernelGGL((sample_max_kernel<T>), dim3((unsigned)p.n * p.P), dim3(SP_MAX_THREADS), 0, s, p);  \
    hipLaunchKernelGGL((sample_hist_kernel<T>), dim3((unsigned)p.n * p.P2), block, 0, s, p); \
    hipLaunchKernelGGL((sample_pick_kernel<T>), dim3((unsigned)p.n * p.P3), block, p.chunks * sizeof(uint64_t), s, p); \
  } while (0)
  if (type == DSPARK_F32)
    SP_GO(float);
  else if (type == DSPARK_BF16)
    SP_GO(__bf16);
  else
    SP_GO(_Float16);
#undef SP_GO
  return (int)hipGetLastError();
}

}  // namespace dspark
