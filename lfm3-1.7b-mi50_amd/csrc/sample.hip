// Sampling a token from each row of logits: temperature, top-k, top-p, min-p and a given random number (include/dspark.h).
//
// A token's weight exp((z - max) / T) is a fixed-point number w = rint(2^44 exp(..)), computed in 64 bits, so that every sum of
// weights is a whole number whatever the order it is taken in: histograms by atomic adds, partial sums of workgroups and the
// draw itself give the same bits always, and sums of 2^20 weights stay under 2^64. (Sums of fp32 weights move the borders
// between tokens by 2^-24 of the whole, more than most of a vocabulary's tokens have; one draw in a thousand then falls to
// another token than the definition's.)
//
// Top-k and top-p both keep a prefix of the tokens ranked by (z descending, index), min-p one by z alone: what is kept is
// "key above key*, or equal to it and index up to idx*" and z at least the min-p bound. The cut is found without sorting:
//   1 sample_max    a part of a row each: the largest key; clears the row's histogram
//   2 sample_hist   a part each: tokens by bins of max - z, logarithmic (128 an octave), counts and weights by LDS atomics, added
//                   to the row's; the last part to finish finds the bin in which the cut lies
//   3 sample_pick   a part each: the tokens down to that bin into the row's list if they are at most LIST of them (as for most
//                   settings), else the bin's own and the weight above it by parts; the last part finds the cut in the list by
//                   digits of the key, then the token.
// Rows that need no cut take no histogram; a row whose bin alone passes LIST (a flat one) is finished by one workgroup from
// the row itself.
#include <algorithm>
#include <type_traits>

#include "batch.h"
#include "dspark.h"

namespace dspark {

constexpr int SP_THREADS = 256, SP_UNIT = 8, SP_STEP = SP_THREADS * SP_UNIT;  // tokens of a thread and of a workgroup at a time
constexpr uint32_t SP_BIN0 = (127 - 9) << 7;  // bin 1 begins at max - z = 2^-9, the last one at 2^7
constexpr double SP_ONE = 17592186044416.0;   // 2^44

enum : uint32_t { SP_EMPTY, SP_GREEDY, SP_ALL, SP_LISTED, SP_BELOW, SP_ROW };

struct SampleLocals {
  float m;               // the row's maximum
  uint32_t first;        // where it is first
  double inv_t, low;     // 1 / T; min-p's bound of (z - m) / T
  bool greedy, empty, cut_low;
  int k;                 // top-k (0: none)
  float p;               // top-p (1: none)
};

__device__ __forceinline__ float sp_value(float z) { return z != z ? -INFINITY : z == 0.f ? 0.f : z; }  // (-0 is 0)

template <typename T>
__device__ __forceinline__ float sp_to_f32(T x) { return (float)x; }

// Eight logits from `at`; those from `end` on are -inf.
template <typename T>
__device__ __forceinline__ void sp_load(const T* row, int at, int end, bool wide, float (&z)[SP_UNIT]) {
  if (wide && at + SP_UNIT <= end) {
    T x[SP_UNIT];
#pragma unroll
    for (int i = 0; i < (int)sizeof(x) / 16; ++i) {
      const u32x4 u = ldg(reinterpret_cast<const u32x4*>(row + at) + i);
      __builtin_memcpy(reinterpret_cast<char*>(x) + 16 * i, &u, 16);
    }
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i) z[i] = sp_value(sp_to_f32(x[i]));
  } else {
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i) z[i] = at + i < end ? sp_value(sp_to_f32(row[at + i])) : -INFINITY;
  }
}

__device__ __forceinline__ uint32_t sp_bin(float z, float m) {
  const float d = m - z;  // rounded, but the bins stay in the order of z
  if (!(d > 0.f)) return 0;  // (also +inf - +inf)
  const uint32_t b = __float_as_uint(d) >> 16;
  return b < SP_BIN0 ? 0 : min(b - SP_BIN0 + 1, (uint32_t)SP_BINS - 1);
}

// 2^44 exp((z - m) / T) as a whole number: 2^x by its whole part and the series of 2^f = e^(f ln 2), |f| <= 1/2, to the 11th
// power (the next term is under 7e-15 = 2^-47).
__device__ __forceinline__ uint64_t sp_weight(float z, const SampleLocals& s) {
  if (z == s.m) return (uint64_t)1 << 44;
  const double x = ((double)z - (double)s.m) * s.inv_t * 1.4426950408889634074;
  if (!(x > -46.0)) return 0;
  const double k = rint(x), f = (x - k) * 0.69314718055994530942;
  double e = 1.0 / 39916800.0;
  e = fma(e, f, 1.0 / 3628800.0);
  e = fma(e, f, 1.0 / 362880.0);
  e = fma(e, f, 1.0 / 40320.0);
  e = fma(e, f, 1.0 / 5040.0);
  e = fma(e, f, 1.0 / 720.0);
  e = fma(e, f, 1.0 / 120.0);
  e = fma(e, f, 1.0 / 24.0);
  e = fma(e, f, 1.0 / 6.0);
  e = fma(e, f, 0.5);
  e = fma(e, f, 1.0);
  e = fma(e, f, 1.0);
  // the weight in units of one, rounded to a whole number by the unit of 2^52
  const double y = __builtin_ldexp(e, (int)k + 44) + 4503599627370496.0;
  return (uint64_t)__double_as_longlong(y) & 0xfffffffffffffull;
}
__device__ __forceinline__ bool sp_high(float z, const SampleLocals& s) {  // min-p
  return !s.cut_low || z == s.m || ((double)z - (double)s.m) * s.inv_t >= s.low;
}

// A wave's and a workgroup's sums of whole numbers. scratch: 4 words.
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t lo = __shfl_up((uint32_t)v, d), hi = __shfl_up((uint32_t)(v >> 32), d);
    if (lane >= d) v += ((uint64_t)hi << 32) | lo;
  }
  return v;
}
// Inclusive sums over the workgroup in thread order; *total the whole. Ends with every thread past the scratch.
__device__ __forceinline__ uint64_t block_scan_u64(uint64_t v, uint64_t* scratch, uint64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan_u64(v, lane);
  if (lane == 63) scratch[wave] = v;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) before += scratch[w];
    all += scratch[w];
  }
  *total = all;
  __syncthreads();
  return before + v;
}

template <typename T>
__device__ __forceinline__ const T* sp_row(const SampleParams& p, int row) {
  return static_cast<const T*>(p.logits) + (size_t)row * p.stride;
}

// The row's settings and maximum (the same in every thread; called by whole workgroups, after sample_max).
__device__ __forceinline__ SampleLocals sp_locals(const SampleParams& p, int row) {
  SampleLocals s;
  uint64_t key = 0;
  for (int i = threadIdx.x & 63; i < p.P; i += 64) key = max(key, ldg(p.part_key + (size_t)row * p.P + i));
  key = wave_max_u64(key);
  const uint32_t ord = (uint32_t)(key >> 32), bits = ord & 0x80000000u ? ord ^ 0x80000000u : ~ord;
  s.m = __uint_as_float(bits);
  s.first = 0xffffffffu - (uint32_t)key;
  s.empty = !(s.m > -INFINITY);
  const float t = p.temperature ? p.temperature[row] : p.temperature_all;
  s.greedy = !(t > 0.f);
  s.inv_t = s.greedy ? 1.0 : 1.0 / (double)t;
  s.k = p.top_k ? p.top_k[row] : p.top_k_all;
  if (s.k <= 0 || s.k >= p.V) s.k = 0;
  s.p = p.top_p ? p.top_p[row] : p.top_p_all;
  if (!(s.p < 1.f)) s.p = 1.f;
  s.p = fmaxf(s.p, 0.f);
  const float low = p.min_p ? p.min_p[row] : p.min_p_all;
  s.cut_low = low > 0.f;
  s.low = s.cut_low ? log((double)fminf(low, 1.f)) : 0.0;
  return s;
}

// One of a row's parts is done; true in the last one, which then sees what the others wrote.
__device__ __forceinline__ bool sp_last(uint32_t* mark, int parts) {
  __shared__ uint32_t arrived;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) arrived = atomicAdd(mark, 1u);
  __syncthreads();
  const bool last = arrived == (uint32_t)parts - 1;
  if (last) __threadfence();
  return last;
}

template <typename T>
__global__ __launch_bounds__(SP_THREADS) void sample_max_kernel(SampleParams p) {
  const int part = blockIdx.x % p.P, row = blockIdx.x / p.P;
  const T* z0 = sp_row<T>(p, row);
  const int end = min((part + 1) * p.ps, p.V);
  for (int i = part * SP_THREADS + threadIdx.x; i < SP_BINS; i += p.P * SP_THREADS) {
    p.hist_count[(size_t)row * SP_BINS + i] = 0;
    p.hist_mass[(size_t)row * SP_BINS + i] = 0;
  }
  if (part == 0 && threadIdx.x < 4) p.marks[row * 4 + threadIdx.x] = 0;
  uint64_t key = 0;
  for (int at = part * p.ps + threadIdx.x * SP_UNIT; at < end; at += SP_STEP) {
    float z[SP_UNIT];
    sp_load<T>(z0, at, end, p.wide, z);
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i) key = max(key, argmax_key(z[i], (uint32_t)(at + i)));
  }
  __shared__ uint64_t best[4];
  key = wave_max_u64(key);
  if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = key;
  __syncthreads();
  if (threadIdx.x == 0) p.part_key[(size_t)row * p.P + part] = max(max(best[0], best[1]), max(best[2], best[3]));
}

template <typename T>
__global__ __launch_bounds__(SP_THREADS) void sample_hist_kernel(SampleParams p) {
  __shared__ uint64_t mass[SP_BINS];
  __shared__ uint32_t count[SP_BINS];
  __shared__ uint64_t scratch[4];
  const int part = blockIdx.x % p.P, row = blockIdx.x / p.P;
  const SampleLocals s = sp_locals(p, row);
  if (s.empty || s.greedy || (s.k == 0 && s.p >= 1.f)) {
    if (part == 0 && threadIdx.x == 0) p.rows[row].mode = s.empty ? SP_EMPTY : s.greedy ? SP_GREEDY : SP_ALL;
    return;
  }
  for (int i = threadIdx.x; i < SP_BINS; i += SP_THREADS) {
    mass[i] = 0;
    count[i] = 0;
  }
  __syncthreads();
  const T* z0 = sp_row<T>(p, row);
  const int end = min((part + 1) * p.ps, p.V);
  for (int at = part * p.ps + threadIdx.x * SP_UNIT; at < end; at += SP_STEP) {
    float z[SP_UNIT];
    sp_load<T>(z0, at, end, p.wide, z);
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i) {
      if (!(z[i] > -INFINITY)) continue;
      const uint32_t b = sp_bin(z[i], s.m);
      atomicAdd(&count[b], 1u);
      if (s.p < 1.f) {
        const uint64_t w = sp_weight(z[i], s);
        if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&mass[b]), (unsigned long long)w);
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < SP_BINS; i += SP_THREADS) {
    if (count[i]) atomicAdd(&p.hist_count[(size_t)row * SP_BINS + i], count[i]);
    if (mass[i]) atomicAdd(reinterpret_cast<unsigned long long*>(&p.hist_mass[(size_t)row * SP_BINS + i]), (unsigned long long)mass[i]);
  }
  if (!sp_last(&p.marks[row * 4], p.P)) return;

  // The bin of the cut: eight bins a thread, their sums before them.
  constexpr int EACH = SP_BINS / SP_THREADS;
  uint64_t c[EACH], w[EACH], cs = 0, ws = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const size_t b = (size_t)row * SP_BINS + threadIdx.x * EACH + i;
    c[i] = p.hist_count[b];
    w[i] = p.hist_mass[b];
    cs += c[i];
    ws += w[i];
  }
  uint64_t live, whole;
  uint64_t c0 = block_scan_u64(cs, scratch, &live) - cs, w0 = block_scan_u64(ws, scratch, &whole) - ws;
  const bool by_k = s.k > 0 && (uint64_t)s.k < live;
  const uint64_t limit_w = max((uint64_t)ceil((double)s.p * (double)whole), (uint64_t)1);
  if (!by_k && s.p >= 1.f) {
    if (threadIdx.x == 0) p.rows[row].mode = SP_ALL;
    return;
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const bool here = by_k ? c0 < (uint64_t)s.k && c0 + c[i] >= (uint64_t)s.k : w0 < limit_w && w0 + w[i] >= limit_w;
    if (here) {  // (one thread, one bin)
      SampleRow r;
      r.bin = threadIdx.x * EACH + i;
      r.above = (uint32_t)c0;
      r.mass_above = w0;
      r.by_mass = !by_k;
      r.limit = by_k ? (uint64_t)s.k : limit_w;
      // (top-k and top-p with more than a list's tokens: top-p's part of the whole is of what top-k leaves)
      r.mode = c0 + c[i] <= SP_LIST ? SP_LISTED : c[i] <= SP_LIST && !(by_k && s.p < 1.f) ? SP_BELOW : SP_ROW;
      p.rows[row] = r;
    }
    c0 += c[i];
    w0 += w[i];
  }
}

// Tokens in index order, from the list in LDS or (ROW) the row itself.
template <typename T, bool ROW>
struct SampleItems {
  const T* z0;
  const uint32_t* idx;
  int n;
  __device__ __forceinline__ uint32_t index(int i) const { return ROW ? (uint32_t)i : idx[i]; }
  __device__ __forceinline__ float value(int i) const { return sp_value(sp_to_f32(z0[index(i)])); }
};

// What is kept so far: keys above `key`, or equal to it with index <= idx.
struct SampleCut {
  uint32_t key, idx;
  __device__ __forceinline__ bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= idx); }
};

struct SampleShared {
  uint64_t mass[256];
  uint32_t count[256];
  uint64_t scratch[4];
  uint64_t c, w;         // tokens and weight above the digits found so far
  uint32_t digit, found;
  uint64_t w_at;
  uint32_t at, kept;
};

// Shrinks `cut` to the first `limit` tokens (by_mass false) or to those with less than `limit` weight in front of them, of the items it
// keeps, `above` tokens of weight `mass_above` standing in front of all of them. Digits of eight bits from the top, then ties.
template <typename Items>
__device__ __forceinline__ void sp_shrink(const Items& it, const SampleLocals& s, SampleShared& sh, SampleCut& cut, bool by_mass, uint64_t limit,
                                          uint64_t above, uint64_t mass_above) {
  uint32_t prefix = 0;
  uint64_t c = above, w = mass_above;
  for (int shift = 24; shift >= 0; shift -= 8) {
    sh.mass[threadIdx.x] = 0;
    sh.count[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.found = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < it.n; i += SP_THREADS) {
      const float z = it.value(i);
      if (!(z > -INFINITY)) continue;
      const uint32_t key = argmax_ord(z);
      if (!cut.keeps(key, it.index(i)) || (shift < 24 && (key >> (shift + 8)) != prefix)) continue;
      const uint32_t d = 255 - ((key >> shift) & 255);  // the largest digit first
      atomicAdd(&sh.count[d], 1u);
      if (by_mass) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[d]), (unsigned long long)sp_weight(z, s));
    }
    __syncthreads();
    const uint64_t hc = sh.count[threadIdx.x], hw = sh.mass[threadIdx.x];
    uint64_t all;
    const uint64_t c1 = c + block_scan_u64(hc, sh.scratch, &all), w1 = w + block_scan_u64(hw, sh.scratch, &all);
    if (by_mass ? w1 - hw < limit && w1 >= limit : c1 - hc < limit && c1 >= limit) {
      sh.digit = 255 - threadIdx.x;
      sh.c = c1 - hc;
      sh.w = w1 - hw;
      sh.found = 1;
    }
    __syncthreads();
    if (!sh.found) return;  // all of them stay
    prefix = prefix << 8 | sh.digit;
    c = sh.c;
    w = sh.w;
    __syncthreads();
  }
  // of the tokens of this key the first `more`, in index order
  float z;
  {
    const uint32_t bits = prefix & 0x80000000u ? prefix ^ 0x80000000u : ~prefix;
    z = __uint_as_float(bits);
  }
  const uint64_t wt = sp_weight(z, s);
  const uint64_t more = by_mass ? (wt ? (limit - w + wt - 1) / wt : 1) : limit - c;
  const int each = (it.n + SP_THREADS - 1) / SP_THREADS, lo = min((int)threadIdx.x * each, it.n), hi = min(lo + each, it.n);
  auto tie = [&](int i) { return argmax_ord(it.value(i)) == prefix && cut.keeps(prefix, it.index(i)); };
  uint64_t mine = 0, ties;
  for (int i = lo; i < hi; ++i) mine += tie(i);
  uint64_t before = block_scan_u64(mine, sh.scratch, &ties) - mine;
  if (threadIdx.x == 0) sh.at = 0xffffffffu;
  __syncthreads();
  if (more < ties && before < more && before + mine >= more)
    for (int i = lo; i < hi; ++i)
      if (tie(i) && ++before == more) sh.at = it.index(i);
  __syncthreads();
  const uint32_t all_ties = prefix == cut.key ? cut.idx : 0xffffffffu;  // (an earlier cut among the same ties)
  cut.idx = sh.at == 0xffffffffu ? all_ties : sh.at;
  cut.key = prefix;
  __syncthreads();
}

// The row's outputs (one thread).
__device__ __forceinline__ void sp_store(const SampleParams& p, int row, int token, float z, int kept, float logprob) {
  if (p.tokens) p.tokens[row] = token;
  if (p.keys) p.keys[row] = token < 0 ? 0 : argmax_key(z, (uint32_t)token);
  if (p.kept) p.kept[row] = kept;
  if (p.logprob) p.logprob[row] = logprob;
}
__device__ __forceinline__ uint64_t sp_target(const SampleParams& p, int row, uint64_t whole) {
  const float u = p.u[row];
  const double x = u > 0.f ? (double)fminf(u, 1.f - 0x1p-24f) * (double)whole : 0.0;
  return x < (double)(whole - 1) ? (uint64_t)x : whole - 1;
}
__device__ __forceinline__ float sp_logprob(uint64_t w, uint64_t whole) { return (float)log((double)w / (double)whole); }

// The draw among items: each thread's run of them, the run that the target falls into, the item.
template <typename Items>
__device__ __forceinline__ void sp_draw(const SampleParams& p, int row, const Items& it, const SampleLocals& s, SampleShared& sh, const SampleCut& cut) {
  const int each = (it.n + SP_THREADS - 1) / SP_THREADS, lo = min((int)threadIdx.x * each, it.n), hi = min(lo + each, it.n);
  uint64_t mine = 0, kept = 0, whole, all;
  for (int i = lo; i < hi; ++i) {
    const float z = it.value(i);
    if (!(z > -INFINITY) || !cut.keeps(argmax_ord(z), it.index(i)) || !sp_high(z, s)) continue;
    mine += sp_weight(z, s);
    ++kept;
  }
  uint64_t sum = block_scan_u64(mine, sh.scratch, &whole) - mine;
  block_scan_u64(kept, sh.scratch, &all);
  const uint64_t target = sp_target(p, row, whole);
  if (sum > target || sum + mine <= target) return;
  for (int i = lo; i < hi; ++i) {  // (one thread)
    const float z = it.value(i);
    if (!(z > -INFINITY) || !cut.keeps(argmax_ord(z), it.index(i)) || !sp_high(z, s)) continue;
    const uint64_t w = sp_weight(z, s);
    sum += w;
    if (sum > target) {
      sp_store(p, row, (int)it.index(i), z, (int)all, sp_logprob(w, whole));
      return;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(SP_THREADS) void sample_pick_kernel(SampleParams p) {
  __shared__ uint32_t list[SP_LIST];
  __shared__ SampleShared sh;
  const int part = blockIdx.x % p.P, row = blockIdx.x / p.P;
  const SampleRow r = p.rows[row];
  const SampleLocals s = sp_locals(p, row);
  if (r.mode == SP_EMPTY || r.mode == SP_GREEDY) {
    if (part == 0 && threadIdx.x == 0) {
      if (r.mode == SP_EMPTY)
        sp_store(p, row, -1, 0.f, 0, -INFINITY);
      else
        sp_store(p, row, (int)s.first, s.m, 1, 0.f);
    }
    return;
  }
  const T* z0 = sp_row<T>(p, row);
  const size_t mine = (size_t)row * p.P + part;
  if (r.mode == SP_ROW) {
    if (part) return;
    const SampleItems<T, true> it = {z0, nullptr, p.V};
    SampleCut cut = {0, 0xffffffffu};
    if (s.k) sp_shrink(it, s, sh, cut, false, (uint64_t)s.k, 0, 0);
    if (s.p < 1.f) {
      uint64_t w = 0, whole;
      for (int i = threadIdx.x; i < p.V; i += SP_THREADS) {
        const float z = it.value(i);
        if (z > -INFINITY && cut.keeps(argmax_ord(z), (uint32_t)i)) w += sp_weight(z, s);
      }
      block_scan_u64(w, sh.scratch, &whole);
      sp_shrink(it, s, sh, cut, true, max((uint64_t)ceil((double)s.p * (double)whole), (uint64_t)1), 0, 0);
    }
    sp_draw(p, row, it, s, sh, cut);
    return;
  }
  // This part's listed tokens in index order, and the weight and number of its tokens above the bin
  const int end = min((part + 1) * p.ps, p.V);
  const bool listed = r.mode == SP_LISTED, all = r.mode == SP_ALL;
  uint64_t sum = 0, number = 0;
  uint32_t here = 0;
  for (int at0 = part * p.ps; at0 < end; at0 += SP_STEP) {
    const int at = at0 + threadIdx.x * SP_UNIT;
    float z[SP_UNIT];
    if (at < end) {
      sp_load<T>(z0, at, end, p.wide, z);
    } else {
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i) z[i] = -INFINITY;
    }
    uint32_t take = 0;
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i) {
      if (!(z[i] > -INFINITY)) continue;
      const uint32_t b = all ? 0 : sp_bin(z[i], s.m);
      if (!all && (listed ? b <= r.bin : b == r.bin)) take |= 1u << i;
      if (!listed && (all || b < r.bin) && sp_high(z[i], s)) {
        sum += sp_weight(z[i], s);
        ++number;
      }
    }
    if (all) continue;
    uint64_t total;
    uint32_t to = here + (uint32_t)(block_scan_u64((uint64_t)__popc(take), sh.scratch, &total) - __popc(take));
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i)
      if (take >> i & 1) list[to++] = (uint32_t)(at + i);  // (at most SP_LIST in the whole row)
    here += (uint32_t)total;
  }
  __syncthreads();
  if (!all) {
    if (threadIdx.x == 0) {
      sh.at = here ? atomicAdd(&p.marks[row * 4 + 2], here) : 0;
      p.part_at[mine] = sh.at;
      p.part_listed[mine] = here;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < here; i += SP_THREADS) p.list[(size_t)row * SP_LIST + sh.at + i] = list[i];
  }
  if (!listed) {
    uint64_t s_all, n_all;
    block_scan_u64(sum, sh.scratch, &s_all);
    block_scan_u64(number, sh.scratch, &n_all);
    if (threadIdx.x == 0) {
      p.part_sum[mine] = s_all;
      p.part_count[mine] = (uint32_t)n_all;
    }
  }
  if (!sp_last(&p.marks[row * 4 + 1], p.P)) return;

  // The last part finishes the row. The list, part by part, so that it is in index order:
  const bool mine_is = (int)threadIdx.x < p.P;
  const size_t of = (size_t)row * p.P + threadIdx.x;
  SampleItems<T, false> it = {z0, list, 0};
  if (!all) {
    const uint64_t n = mine_is ? p.part_listed[of] : 0;
    uint64_t total;
    const uint32_t to = (uint32_t)(block_scan_u64(n, sh.scratch, &total) - n);
    sh.count[threadIdx.x] = to - (n ? p.part_at[of] : 0);  // from an entry's place in the row's list to its place here
    __syncthreads();
    it.n = (int)total;
    for (int i = threadIdx.x; i < it.n; i += SP_THREADS) {
      const uint32_t idx = p.list[(size_t)row * SP_LIST + i];
      list[(uint32_t)i + sh.count[idx / (uint32_t)p.ps]] = idx;
    }
    __syncthreads();
  }
  SampleCut cut = {0, 0xffffffffu};
  if (listed) {
    if (s.k && (!r.by_mass)) sp_shrink(it, s, sh, cut, false, r.limit, 0, 0);
    if (s.p < 1.f) {
      uint64_t limit = r.limit;
      if (!r.by_mass) {
        uint64_t w = 0, whole;
        for (int i = threadIdx.x; i < it.n; i += SP_THREADS) {
          const float z = it.value(i);
          if (cut.keeps(argmax_ord(z), it.index(i))) w += sp_weight(z, s);
        }
        block_scan_u64(w, sh.scratch, &whole);
        limit = max((uint64_t)ceil((double)s.p * (double)whole), (uint64_t)1);
      }
      sp_shrink(it, s, sh, cut, true, limit, 0, 0);
    }
    sp_draw(p, row, it, s, sh, cut);
    return;
  }
  // Weights by parts: above the bin, and the bin's kept ones
  if (!all) sp_shrink(it, s, sh, cut, r.by_mass != 0, r.limit, r.above, r.mass_above);
  sh.mass[threadIdx.x] = mine_is ? p.part_sum[of] : 0;
  sh.count[threadIdx.x] = mine_is ? p.part_count[of] : 0;
  __syncthreads();
  for (int i = threadIdx.x; i < it.n; i += SP_THREADS) {
    const float z = it.value(i);
    const uint32_t idx = it.index(i);
    if (!cut.keeps(argmax_ord(z), idx) || !sp_high(z, s)) continue;
    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[idx / (uint32_t)p.ps]), (unsigned long long)sp_weight(z, s));
    atomicAdd(&sh.count[idx / (uint32_t)p.ps], 1u);
  }
  __syncthreads();
  const uint64_t w = sh.mass[threadIdx.x], cnt = sh.count[threadIdx.x];
  uint64_t whole, kept;
  const uint64_t after = block_scan_u64(w, sh.scratch, &whole);
  block_scan_u64(cnt, sh.scratch, &kept);
  const uint64_t target = sp_target(p, row, whole);
  if (after > target && after - w <= target) {  // (one thread)
    sh.found = threadIdx.x;
    sh.c = after - w;
  }
  __syncthreads();
  // the part, in index order, a workgroup's step at a time
  uint64_t base = sh.c;
  const int first = (int)sh.found * p.ps, last = min(first + p.ps, p.V);
  for (int at0 = first; at0 < last; at0 += SP_STEP) {
    const int at = at0 + threadIdx.x * SP_UNIT;
    float z[SP_UNIT];
    uint64_t ws[SP_UNIT], run = 0, step;
    if (at < last) {
      sp_load<T>(z0, at, last, p.wide, z);
    } else {
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i) z[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < SP_UNIT; ++i) {
      const bool in = z[i] > -INFINITY && (all || sp_bin(z[i], s.m) < r.bin || cut.keeps(argmax_ord(z[i]), (uint32_t)(at + i))) && sp_high(z[i], s);
      ws[i] = in ? sp_weight(z[i], s) : 0;
      run += ws[i];
    }
    uint64_t sum0 = base + block_scan_u64(run, sh.scratch, &step) - run;
    if (sum0 <= target && sum0 + run > target) {
#pragma unroll
      for (int i = 0; i < SP_UNIT; ++i) {
        if (sum0 <= target && sum0 + ws[i] > target) sp_store(p, row, at + i, z[i], (int)kept, sp_logprob(ws[i], whole));
        sum0 += ws[i];
      }
    }
    base += step;
    if (base > target) return;
  }
}

// Parts of a row: about 1024 workgroups in all, none of less than a step.
void sample_plan(SampleParams& p) {
  const int steps = (p.V + SP_STEP - 1) / SP_STEP;
  const int parts = std::min({SP_PARTS, steps, std::max(1, 1024 / p.n)});
  p.ps = (steps + parts - 1) / parts * SP_STEP;
  p.P = (p.V + p.ps - 1) / p.ps;
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
  piece(p.part_sum, parts);
  piece(p.hist_mass, n * SP_BINS);
  piece(p.rows, n);
  piece(p.hist_count, n * SP_BINS);
  piece(p.part_count, parts);
  piece(p.part_at, parts);
  piece(p.part_listed, parts);
  piece(p.list, n * SP_LIST);
  piece(p.marks, n * 4);
  return (size_t)(at - static_cast<char*>(ws));
}

int sample_launch(const SampleParams& p, int type, hipStream_t s) {
  const dim3 grid((unsigned)p.n * p.P), block(SP_THREADS);
#define SP_GO(T)                                                  \
  do {                                                            \
    hipLaunchKernelGGL((sample_max_kernel<T>), grid, block, 0, s, p);  \
    hipLaunchKernelGGL((sample_hist_kernel<T>), grid, block, 0, s, p); \
    hipLaunchKernelGGL((sample_pick_kernel<T>), grid, block, 0, s, p); \
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
