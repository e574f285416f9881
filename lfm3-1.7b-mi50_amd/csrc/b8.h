// The 8-bit block-scaled K/V cache ("b8" pages, include/dspark.h): launch descriptors and the code arithmetic that its
// writer, reader, attention and eviction share.
#pragma once
#include "common.h"

namespace dspark {

// Codes [pages][KVH][PAGE][D] of one byte, scales [pages][KVH]. Block (page, head) starts at byte
// (page * KVH + head) * PAGE * D: 64 bits, a pool may pass 4 GiB.
struct B8Pool {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  const int32_t* bt;  // logical -> physical page, nullptr = identity
  int64_t pages;
  int KVH;
};

// Physical page of a logical one, or -1 (an absent page).
__device__ __forceinline__ int b8_page(const B8Pool& c, int lp) {
  const int pg = c.bt ? ldg(c.bt + lp) : lp;
  return pg >= 0 && pg < c.pages ? pg : -1;
}

// The scale of a block of fp16 values whose largest finite magnitude is amax >= 0.
// int8: amax / 127 rounded up to 16 significant bits, so that code * scale (7 + 16 bits) is exact in fp32.
// e4m3: the least power of two s with amax <= 448 s (448 = 1.75 * 2^8 is the largest code), so that both directions are
// exact but for the code's own rounding.
template <bool FP8>
__device__ __forceinline__ float b8_scale(float amax) {
  if (!(amax > 0.f)) return 0.f;
  if constexpr (FP8) {
    const uint32_t u = __float_as_uint(amax);  // normal: the least fp16 magnitude is 2^-24
    const uint32_t e = (u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float(e << 23);
  } else {
    return __uint_as_float((__float_as_uint(__fdiv_rn(amax, 127.f)) + 255u) & ~255u);
  }
}

// What x is divided by its block's scale with (exact for e4m3; int8 codes are corrected against the scale itself).
__device__ __forceinline__ float b8_inv(float scale) { return scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f; }

// The int8 code of x at scale s: x / s rounded to nearest, ties to even, decided exactly. t = rint(x inv) is off by at
// most one next to a border; the sign of x - (t +- 1/2) s, from one fma (t +- 1/2 is exact, and rounding keeps a sign
// and a zero), says on which side x lies. NaN is coded 0, what lies past the codes +-127.
__device__ __forceinline__ uint32_t b8_code_i8(float x, float s, float inv) {
  x = x != x ? 0.f : fminf(fmaxf(x, -127.f * s), 127.f * s);
  float t = rintf(x * inv);
  const float up = fmaf(-(t + 0.5f), s, x), dn = fmaf(-(t - 0.5f), s, x);
  const bool odd = ((int)t & 1) != 0;
  if (up > 0.f || (up == 0.f && odd && s > 0.f)) t += 1.f;
  else if (dn < 0.f || (dn == 0.f && odd && s > 0.f)) t -= 1.f;
  return (uint32_t)(int)t;
}

// Four values as four codes (one word, the first in the low byte). ANY: values may be infinite or no numbers; without it they
// are finite and the block's scale covers them.
template <bool FP8, bool ANY>
__device__ __forceinline__ uint32_t b8_code4(float x0, float x1, float x2, float x3, float s, float inv) {
  if constexpr (FP8) {  // x inv is exact: inv is a power of two
    auto y = [&](float x) {
      const float z = x * inv;
      if constexpr (ANY) return z != z ? 0.f : fminf(fmaxf(z, -448.f), 448.f);
      else return z;
    };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y(x0), y(x1), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y(x2), y(x3), w, true);
  } else {
    // y = x inv + 1.5 2^23 holds the rounded code in its low byte. x inv is off by 2^-16 at most (codes up to 127, two
    // roundings), so only values within 2^-14 of a border, and those that are no numbers, are decided anew.
    constexpr float MAGIC = 12582912.f;
    const float x[4] = {x0, x1, x2, x3};
    uint32_t y[4];
    bool near = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float r = fmaf(x[i], inv, MAGIC);
      y[i] = __float_as_uint(r);
      near |= !(fabsf(fmaf(x[i], inv, MAGIC - r)) < 0.5f - 0x1p-14f);
    }
    if (__builtin_expect(__ballot(near) != 0, 0)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = b8_code_i8(x[i], s, inv);
    }
    const uint32_t lo = __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(y[3], y[2], 0x04000c0cu);
    return lo | hi;
  }
}

// Four codes as the numbers they are (unscaled).
template <bool FP8>
__device__ __forceinline__ f32x4 b8_value4(uint32_t w) {
  if constexpr (FP8) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return f32x4{lo[0], lo[1], hi[0], hi[1]};
  } else {
    return f32x4{(float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24)};
  }
}

// The codes of one word under scale `from`, at scale `to` (code * from is exact in fp32).
template <bool FP8>
__device__ __forceinline__ uint32_t b8_recode4(uint32_t w, float from, float to, float inv_to) {
  const f32x4 x = b8_value4<FP8>(w) * from;
  return b8_code4<FP8, false>(x[0], x[1], x[2], x[3], to, inv_to);
}

struct B8Write {
  B8Pool c;
  const _Float16* k;
  const _Float16* v;
  int64_t row_stride;
  int pos0, n;
};
struct B8Read {
  B8Pool c;
  float* k;
  float* v;
  int64_t row_stride;
  int pos0, n;
};
struct B8Evict {
  B8Pool src, dst;
  int T, keep, sinks, recent;
  const float* mass;
  int64_t mass_stride;
  int32_t* kept;  // [KVH][keep]
  float* mass_out;
  int64_t mass_out_stride;
};
int b8_write_launch(const B8Write& p, int D, bool fp8, hipStream_t s);
int b8_read_launch(const B8Read& p, int D, bool fp8, hipStream_t s);
int b8_evict_launch(const B8Evict& p, int D, bool fp8, void* ws, hipStream_t s);
size_t b8_evict_workspace(int KVH, int length);

struct B8Attn {
  B8Pool c;
  const _Float16* q;
  int64_t q_stride;     // elements between tokens
  _Float16* out16;      // [M][QH][D]
  float* out32;
  float* lse;           // [M][QH] natural log
  const float* gate;    // [M][QH]
  float* part_acc;      // [KVH][rows][S][D]
  f32x2* part_ml;       // [KVH][rows][S] (reference exponent, sum)
  uint32_t* arrivals;   // [KVH][RG] zero between calls, or nullptr
  int M, QH, G, R;      // R = G M rows per KV head, row r = token r / G, query head r % G of the KV head's
  uint32_t g_div;
  int a, start, window, causal;
  int page0, npages;    // logical pages any row sees
  int full_lo, full_hi; // pages in [full_lo, full_hi) are seen whole by every row
  int S, RG;            // key splits, row groups
  int pps, more;        // pages of a wave, and waves that take one more
  int rb;               // 16-row blocks of a row group
  float c2;             // log2(e) / sqrt(D)
  // the key accounts
  int seen_lo;          // first logical page any row sees
  const float* lse_in;
  const int32_t* rows;
  const float* mass_in;
  float* mass_out;
  int64_t mass_stride;
};
void b8_attn_plan(B8Attn& p, int D, int splits, int cus);
size_t b8_attn_workspace(const B8Attn& p, int D);
int b8_attn_launch(const B8Attn& p, int D, bool fp8, hipStream_t s);
int b8_mass_launch(const B8Attn& p, int D, bool fp8, int cus, hipStream_t s);

}  // namespace dspark
