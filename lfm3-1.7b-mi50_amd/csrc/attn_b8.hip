// Verify attention over the 8-bit block-scaled K/V cache, and the accounts of attention weight its keys draw.
//
// o = softmax(q k^T / sqrt(D)) v for the rows of a KV head (row r = token r / G, query head r % G of the head's), keys in
// blocks of 32 (a page) whose codes carry one scale: x = (q . code) ks log2(e) / sqrt(D). V's scale goes into the exponent:
// P = 2^(x + log2 vs - ref) with the row's running reference over x + log2 vs, so that o += P . codes accumulates in the matrix
// cores whatever the blocks' scales, and l += (sum of P) / vs keeps the softmax sum in the same units (with o += vs (P . codes)
// instead, D / 4 multiply-adds a row block and page: 79 -> 69 us at 128k keys and 33 tokens). Codes (int8 or e4m3) are exact
// in fp16, so the products are of exact operands but for P, which is rounded to fp16 once; scales, references, sums and
// outputs are fp32.
//
// A wave owns whole pages and all rows of its row group, and takes its operands from memory in registers: nothing is shared
// until the end. Score product: A = K (16 keys), B = Q, so that a lane holds one row's scores of keys 16 b + 4 g + i
// (lane = 16 g + n, row n); these eight are, in this order, the lane's B operand of the second product (A = V^T), so P never
// leaves its lane. The contraction order is free as long as both operands agree: dims go in 16-byte pieces of a K row, and
// V rows are transposed in registers by byte permutes.
#include "b8.h"
#include "dspark.h"
#include "dspark_internal.h"

namespace dspark {

// Waves of a workgroup, which fills a CU: as many as the registers of RB row blocks leave (o alone takes D RB / 4).
constexpr int b8_waves(int D, int RB) { return D == 64 ? (RB == 1 ? 16 : RB <= 3 ? 12 : 8) : RB == 1 ? 12 : 8; }
constexpr int MASS_WAVES = 4;
constexpr int B8_COHERENT = 16;    // buffer cache policy SC1: device-scope coherent store / load
constexpr int B8_FUSED_BYTES = 64 << 10;  // sums of one row block's splits that the last of them adds (b8_attn_plan)
// Running reference in log2 units, set to the row's largest x + log2 vs less 8 when one passes ref + 15: P stays under 2^15,
// and a P of 2^-22 of the largest is still a normal half (one below is off by 2^-33 of the largest at most).
constexpr float REF_INIT = -1e30f, REF_BELOW = 8.f, REF_SLACK = 15.f;
// log2 of the scale that stands in for a block of zeros': scales are at least 2^-33 (2^-24, the least half, over 127 or 448).
constexpr float ZERO_LOG2 = -40.f;

template <int D>
struct B8Tile {
  u32x4 k[2][D / 64];  // key 16 b + n, dims 64 u + 16 g .. + 16
  uint32_t v[8][D / 64];  // key 16 (j / 4) + 4 g + j % 4, dims (D / 16) n .. + D / 16
};

// A block as a buffer (wave-uniform), so that a load is the lane's 32-bit offset and registers of pending loads are not needed
// for addresses; an absent page (pg < 0) is an empty one, whose loads return zeros.
template <int D>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t b8_block(const uint8_t* pool, int KVH, int h, int pg) {
  const size_t blk = ((size_t)max(pg, 0) * KVH + h) * (PAGE * D);
  return __builtin_amdgcn_make_buffer_rsrc((void*)(pool + blk), (short)0, pg < 0 ? 0 : PAGE * D, 0x00020000);
}
template <int D>
__device__ __forceinline__ void b8_load_k(__amdgpu_buffer_rsrc_t r, int lane, u32x4 (&k)[2][D / 64]) {
  const int off = (lane & 15) * D + (lane >> 4) * 16;
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int u = 0; u < D / 64; ++u) k[b][u] = __builtin_amdgcn_raw_buffer_load_b128(r, off + (16 * b * D + 64 * u), 0, 0);
}
template <int D>
__device__ __forceinline__ void b8_load_v(__amdgpu_buffer_rsrc_t r, int lane, uint32_t (&v)[8][D / 64]) {
  const int off = (lane >> 4) * 4 * D + (lane & 15) * (D / 16);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int at = off + (16 * (j / 4) + j % 4) * D;
    if constexpr (D == 64) {
      v[j][0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0);
    } else {
      const u32x2 t = __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0);
      v[j][0] = t[0];
      v[j][1] = t[1];
    }
  }
}

// Two codes (bytes 2 H, 2 H + 1 of w) as halves, exactly. int8 codes come with their sign bit flipped (code + 128).
template <bool FP8, bool H>
__device__ __forceinline__ half2v b8_half2(uint32_t w) {
  if constexpr (FP8) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, H));
  } else {
    const uint32_t u = __builtin_amdgcn_perm(0x64646464u, w, H ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(half2v, u) - half2v{1152, 1152};
  }
}
template <bool FP8>
__device__ __forceinline__ uint32_t b8_flip(uint32_t w) {
  if constexpr (FP8) return w;
  else return w ^ 0x80808080u;
}
template <bool FP8>
__device__ __forceinline__ half8 b8_half8(uint32_t w0, uint32_t w1) {
  const half2v a = b8_half2<FP8, false>(w0), b = b8_half2<FP8, true>(w0), c = b8_half2<FP8, false>(w1), d = b8_half2<FP8, true>(w1);
  return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// V^T operands of dims db and db + 1 (bytes E, E + 1 of the eight keys' words): pairs of keys by one permute for both dims.
template <bool FP8, int E>
__device__ __forceinline__ void b8_vt(const uint32_t (&w)[8], half8& v0, half8& v1) {
  half2v a[4], b[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    // bytes: key 2q dim E, key 2q+1 dim E, key 2q dim E+1, key 2q+1 dim E+1
    const uint32_t t = __builtin_amdgcn_perm(w[2 * q + 1], w[2 * q], E == 0 ? 0x05010400u : 0x07030602u);
    a[q] = b8_half2<FP8, false>(t);
    b[q] = b8_half2<FP8, true>(t);
  }
  v0 = half8{a[0][0], a[0][1], a[1][0], a[1][1], a[2][0], a[2][1], a[3][0], a[3][1]};
  v1 = half8{b[0][0], b[0][1], b[1][0], b[1][1], b[2][0], b[2][1], b[3][0], b[3][1]};
}

// The larger one by the instruction that passes a NaN on: fmaxf costs a second one to quiet its operands.
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float max3(float a, float b, float c) { return max_of(max_of(a, b), c); }
// Largest over the four lanes of a row (lanes n, 16 + n, 32 + n, 48 + n), in all of them; and the sum.
__device__ __forceinline__ float row_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = max_of(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_of(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Q operands of a row group (row0 = its first row): lane (n, g) holds row n's dims 64 u + 16 g + 8 h .. + 8. Rows past the
// last repeat it; what is computed of them is stored nowhere.
template <int D, int RB>
__device__ __forceinline__ void b8_load_q(const B8Attn& p, int h, int row0, int lane, half8 (&q)[RB][D / 32], int (&tok)[RB]) {
  const int n = lane & 15, g = lane >> 4;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = min(row0 + 16 * rb + n, p.R - 1), t = div_by(row, p.g_div);
    tok[rb] = t;
    const _Float16* at = p.q + (size_t)t * p.q_stride + (size_t)(h * p.G + row - t * p.G) * D + 16 * g;
#pragma unroll
    for (int u = 0; u < D / 64; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e) q[rb][2 * u + e] = as_half8(ldg(reinterpret_cast<const u32x4*>(at + 64 * u + 8 * e)));
  }
}
constexpr int NOWHERE = 0x7fffffff - PAGE;  // the position of an absent page's first key: past every range
// What token t sees: the keys lo, lo + 1, ... of the range's `n` (context keys from start and the window on, then the block's;
// one comparison a key).
struct B8Sight {
  int lo;
  uint32_t n;
  __device__ __forceinline__ bool sees(int kp) const { return (uint32_t)(kp - lo) < n; }
};
__device__ __forceinline__ B8Sight b8_sight(const B8Attn& p, int t) {
  const int lo = min(p.a, max(p.start, p.window > 0 ? p.a + t - p.window + 1 : 0));
  return B8Sight{lo, (uint32_t)((p.causal ? p.a + t + 1 : p.a + p.M) - lo)};
}

template <int D, bool FP8>
__device__ __forceinline__ void b8_k_operand(const u32x4 (&k)[D / 64], half8 (&kf)[D / 32]) {
#pragma unroll
  for (int u = 0; u < D / 64; ++u) {
    kf[2 * u] = b8_half8<FP8>(b8_flip<FP8>(k[u][0]), b8_flip<FP8>(k[u][1]));
    kf[2 * u + 1] = b8_half8<FP8>(b8_flip<FP8>(k[u][2]), b8_flip<FP8>(k[u][3]));
  }
}
// q . code of one page: s[rb][b][i] of key 16 b + 4 g + i, still to be multiplied by the block's scale.
template <int D, int RB, bool FP8>
__device__ __forceinline__ void b8_scores(const u32x4 (&k)[2][D / 64], const half8 (&q)[RB][D / 32], f32x4 (&s)[RB][2]) {
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    half8 kf[D / 32];
    b8_k_operand<D, FP8>(k[b], kf);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      s[rb][b] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < D / 32; ++e) s[rb][b] = mfma16x16x32(kf[e], q[rb][e], s[rb][b]);
    }
  }
}
// The scores of a page that some row does not see whole, scaled (a block of zeros has scale 0: -inf comes after it), with -inf
// where the row does not see the key.
template <int RB>
__device__ __forceinline__ void b8_mask(const B8Attn& p, float ks, int pos, const int (&tok)[RB], int lane, f32x4 (&s)[RB][2]) {
  const int g = lane >> 4;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const B8Sight sight = b8_sight(p, tok[rb]);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = s[rb][b][i] * ks;
        s[rb][b][i] = sight.sees(pos + 16 * b + 4 * g + i) ? x : -INFINITY;
      }
  }
}

// ---------------------------------------------------------------- attention
template <int D>
__device__ __forceinline__ void b8_load_tile(const B8Attn& p, int h, int pg, int lane, B8Tile<D>& t) {
  b8_load_k<D>(b8_block<D>(p.c.k, p.c.KVH, h, pg), lane, t.k);
  b8_load_v<D>(b8_block<D>(p.c.v, p.c.KVH, h, pg), lane, t.v);
}

// Running state of a wave's rows: o[rb][d] of row 16 rb + n, dims (D / 16) (4 g + i) + d; l the lane's part of the sum of P,
// before P's rounding (the log-sum-exp is an fp32 output: a sum of rounded P, from a product with ones, is 2^-12 off).
template <int D, int RB>
struct B8Rows {
  float ref[RB];
  float l[RB];
  f32x4 o[RB][D / 16];
};

// One page; lp < 0: an absent one, which no row sees.
template <int D, int RB, bool FP8>
__device__ __forceinline__ void b8_page(const B8Attn& p, const B8Tile<D>& t, const half8 (&q)[RB][D / 32], const int (&tok)[RB],
                                        float ks, float lv, float iv, int lp, int lane, B8Rows<D, RB>& st) {
  f32x4 s[RB][2];
  b8_scores<D, RB, FP8>(t.k, q, s);
  if (lp < p.full_lo || lp >= p.full_hi) {
    int pos = lp < 0 ? NOWHERE : lp * PAGE;
    asm volatile("" : "+s"(pos));  // (keeps the comparisons in this branch: they were made for every page)
    b8_mask<RB>(p, ks, pos, tok, lane, s);
    ks = 1.f;
  }
  float top[RB], at[RB];
  bool over = false;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    top[rb] = fmaf(ks, max3(max3(s[rb][0][0], s[rb][0][1], s[rb][0][2]), max3(s[rb][0][3], s[rb][1][0], s[rb][1][1]),
                            max_of(s[rb][1][2], s[rb][1][3])), lv);
    over |= top[rb] > st.ref[rb] + REF_SLACK;
  }
  if (__ballot(over)) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const float m = row_max(top[rb]);
      const float to = m > st.ref[rb] + REF_SLACK ? m - REF_BELOW : st.ref[rb];
      const float f = fast_exp2(st.ref[rb] - to);
      st.ref[rb] = to;
      st.l[rb] *= f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) st.o[rb][d] *= f;
    }
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) at[rb] = lv - st.ref[rb];
  half8 pf[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e[j] = fast_exp2(fmaf(s[rb][j / 4][j % 4], ks, at[rb]));
      pf[rb][j] = (_Float16)e[j];
    }
    st.l[rb] = fmaf(((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7])), iv, st.l[rb]);
  }
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = b8_flip<FP8>(t.v[j][c]);
    half8 vt[4];
    b8_vt<FP8, 0>(w, vt[0], vt[1]);
    b8_vt<FP8, 2>(w, vt[2], vt[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) st.o[rb][4 * c + e] = mfma16x16x32(vt[e], pf[rb], st.o[rb][4 * c + e]);
  }
}

// Four dims (4 c ...) of a row's result from its sums: 1 / l, the gate, the stores.
template <int D>
__device__ __forceinline__ void b8_store(const B8Attn& p, int h, int row, int c, f32x4 acc, float ref, float l, float gate) {
  const int t = div_by(row, p.g_div), qh = h * p.G + row - t * p.G;
  const f32x4 o = l == 0.f ? f32x4{0, 0, 0, 0} : acc * (gate / l);
  const size_t e = ((size_t)t * p.QH + qh) * D + 4 * c;
  if (p.out16) *reinterpret_cast<half4*>(p.out16 + e) = half4{(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
  if (p.out32) *reinterpret_cast<f32x4*>(p.out32 + e) = o;
  if (p.lse && c == 0) p.lse[(size_t)t * p.QH + qh] = l == 0.f ? -INFINITY : (ref + log2f(l)) * 0.69314718055994531f;
}
__device__ __forceinline__ float b8_gate(const B8Attn& p, int h, int row) {
  const int t = div_by(row, p.g_div), qh = h * p.G + row - t * p.G;
  return p.gate ? 1.f / (1.f + __expf(-ldg(p.gate + (size_t)t * p.QH + qh))) : 1.f;
}

// The splits of a row are added in an order of its own, whoever adds them: split lane j takes splits j, j + 4, ... in batches
// of 8, each batch rescaled to the largest reference so far; then the lanes in order. (With no more than BATCH splits a lane a
// smaller batch gives the same bits: the missing ones add zeros.)
constexpr int SPLIT_LANES = 4, SPLIT_BATCH = 8;
template <int D, int BATCH>
struct B8Splits {
  f32x2 ml[BATCH];
  f32x4 v[BATCH];
  // Splits s0, s0 + 4, ... of a row whose sums start at `first` (past the last split: the last again; past the rows: zeros).
  __device__ __forceinline__ void load(const B8Attn& p, __amdgpu_buffer_rsrc_t racc, __amdgpu_buffer_rsrc_t rml, int first, int s0, int c) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int at = first + min(s0 + i * SPLIT_LANES, p.S - 1);
      ml[i] = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(rml, at * (int)sizeof(f32x2), 0, B8_COHERENT));
      v[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(racc, (at * D + 4 * c) * (int)sizeof(float), 0, B8_COHERENT));
    }
  }
  __device__ __forceinline__ void add(const B8Attn& p, int s0, float& m, float& l, f32x4& acc) {
    float to = m;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (s0 + i * SPLIT_LANES >= p.S) ml[i] = f32x2{REF_INIT, 0.f}, v[i] = f32x4{0, 0, 0, 0};
      to = max_of(to, ml[i][0]);
    }
    const float f0 = fast_exp2(m - to);
    acc *= f0;
    l *= f0;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float f = fast_exp2(ml[i][0] - to);
      acc += v[i] * f;
      l = fmaf(ml[i][1], f, l);
    }
    m = to;
  }
};
template <int D>
__device__ __forceinline__ void b8_add_splits(const B8Attn& p, __amdgpu_buffer_rsrc_t racc, __amdgpu_buffer_rsrc_t rml, int first, int j,
                                              int c, float* o, f32x2* ml_out) {
  float m = REF_INIT, l = 0.f;
  f32x4 acc = {0, 0, 0, 0};
  for (int s0 = j; s0 < p.S; s0 += SPLIT_LANES * SPLIT_BATCH) {
    B8Splits<D, SPLIT_BATCH> some;
    some.load(p, racc, rml, first, s0, c);
    some.add(p, s0, m, l, acc);
  }
  *reinterpret_cast<f32x4*>(o) = acc;
  if (c == 0) *ml_out = f32x2{m, l};
}
// The split lanes' sums (o_lane and ml_lane apart from lane to lane) added, the row finished.
template <int D>
__device__ __forceinline__ void b8_finish_row(const B8Attn& p, int h, int row, int c, const float* o, const f32x2* ml, int o_lane,
                                              int ml_lane) {
  const float gate = b8_gate(p, h, row);
  float m = REF_INIT, l = 0.f;
  f32x4 acc = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < SPLIT_LANES; ++w) m = max_of(m, ml[w * ml_lane][0]);
#pragma unroll
  for (int w = 0; w < SPLIT_LANES; ++w) {
    const float f = fast_exp2(ml[w * ml_lane][0] - m);
    acc += *reinterpret_cast<const f32x4*>(o + w * o_lane) * f;
    l = fmaf(ml[w * ml_lane][1], f, l);
  }
  b8_store<D>(p, h, row, c, acc, m, l, gate);
}

// One workgroup per (KV head, key split, row group), the split's pages spread evenly over its waves. Splits go to the
// workspace, where the last of them (RB = 1) or a second kernel adds them; a single split is finished here. Bound by first loads,
// the sums and bytes for one row group (32768 keys of 8 heads of 64, 64 rows: 13.4-14.3 us) and by issue for more, since every
// row group loads and converts a page anew. D = 64, e4m3: 65 vector instructions a page and 16 rows, of them 8 products, 8
// exponentials and 13 conversions (40 a page, for three row blocks); products hardly overlap with the others (131072 keys of 8
// heads of 64, 132 rows: 58-63 us, 560-610 TFLOP/s, vector units busy 60 % of it, matrix cores 26 %). D = 128, int8: 156, of
// them 16 products and 88 conversions (176 a page, for two row blocks), and 36 rows are computed as 64 (131072 keys of 4 heads of
// 128: 34-35 us, 134 MB, 3.9 TB/s; vector units busy 44 %).
template <int D, int RB, bool FP8>
__global__ __launch_bounds__(64 * b8_waves(D, RB), b8_waves(D, RB) / 4) void attn_b8_kernel(B8Attn p) {
  constexpr int ND = D / 16, NW = b8_waves(D, RB), ROWS = 16 * RB, NT = 64 * NW;
  __shared__ float s_o[NW][ROWS][D + 4];  // (rows 4 banks apart)
  __shared__ f32x2 s_ml[NW][ROWS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const int h = blockIdx.y, sp = blockIdx.x, row0 = blockIdx.z * ROWS;
  // wave gw of the head's S NW waves: pps pages, one more for the first `more` waves
  const int gw = sp * NW + wave;
  const int w0 = p.page0 + gw * p.pps + min(gw, p.more), w1 = w0 + p.pps + (gw < p.more ? 1 : 0);

  int pgl = b8_page(p.c, min(w0 + lane, p.page0 + p.npages - 1));  // lane i knows page b0 + i
  half8 q[RB][D / 32];
  int tok[RB];
  b8_load_q<D, RB>(p, h, row0, lane, q, tok);
  B8Rows<D, RB> st;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    st.ref[rb] = REF_INIT;
    st.l[rb] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) st.o[rb][d] = f32x4{0, 0, 0, 0};
  }

  for (int b0 = w0; b0 < w1; b0 += 64) {
    const int nb = min(64, w1 - b0);
    if (b0 > w0) pgl = b8_page(p.c, min(b0 + lane, w1 - 1));
    const size_t sat = (size_t)max(pgl, 0) * p.c.KVH + h;
    B8Tile<D> t[2];
    b8_load_tile<D>(p, h, __builtin_amdgcn_readlane(pgl, 0), lane, t[0]);
    const float ksl = ldg(p.c.ks + sat) * p.c2, vat = ldg(p.c.vs + sat);
    const float vsl = pgl < 0 ? 0.f : vat;  // (what an absent page's lane loaded is another page's: infinite, it made NaN of -inf)
    // log2 vs, and 1 / vs as its very inverse. A block of zeros (scale 0), which counts in the sum alone, takes one below every
    // scale that holds anything: it moves no reference above what a later block of small values needs.
    const float lvl = vsl > 1e-30f ? __builtin_amdgcn_logf(vsl) : ZERO_LOG2;
    const float ivl = fast_exp2(-lvl);
    // the next page's loads are in flight while a page is worked on (past the last one: that page again, from L2)
    auto step = [&](int i, const B8Tile<D>& now, B8Tile<D>& next) {
      b8_load_tile<D>(p, h, __builtin_amdgcn_readlane(pgl, min(i + 1, nb - 1)), lane, next);
      b8_page<D, RB, FP8>(p, now, q, tok, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ksl), i)),
                          __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lvl), i)),
                          __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ivl), i)),
                          __builtin_amdgcn_readlane(pgl, i) < 0 ? -1 : b0 + i, lane, st);
    };
    // Of the waves of a SIMD the oldest would run ahead and leave the others to finish alone: who is further on yields.
    __builtin_amdgcn_s_setprio(3);
    for (int i = 0; i < nb; i += 2) {
      if (4 * i >= nb) __builtin_amdgcn_s_setprio(2);
      if (2 * i >= nb) __builtin_amdgcn_s_setprio(1);
      if (4 * i >= 3 * nb) __builtin_amdgcn_s_setprio(0);
      step(i, t[0], t[1]);
      if (i + 1 < nb) step(i + 1, t[1], t[0]);
    }
  }

  // Every wave's sums into LDS at once, then each thread adds up some rows' quads, rescaled to the row's largest reference,
  // in wave order. (Row block by row block with 16 rows of LDS: two more barriers and a drain each; 16 tokens of
  // 32768 keys took 17.5 us instead of 15.2.)
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const float l = row_sum(st.l[rb]);
    if (g == 0) s_ml[wave][16 * rb + n] = f32x2{st.ref[rb], l};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < ND; d += 4)
        *reinterpret_cast<f32x4*>(&s_o[wave][16 * rb + n][ND * (4 * g + i) + d]) =
            f32x4{st.o[rb][d][i], st.o[rb][d + 1][i], st.o[rb][d + 2][i], st.o[rb][d + 3][i]};
  }
  constexpr int QUADS = D / 4, PER = NT / QUADS;  // rows side by side
  const int c = threadIdx.x % QUADS;
  float gate[(ROWS + PER - 1) / PER];
  if (p.S == 1)
#pragma unroll
    for (int k = 0; k < (ROWS + PER - 1) / PER; ++k) gate[k] = b8_gate(p, h, min(row0 + (int)threadIdx.x / QUADS + k * PER, p.R - 1));
  // the row group's part of the workspace (rows past the last have none; under 2 GiB: at most 64 rows and 4096 splits)
  const size_t first = ((size_t)h * p.R + row0) * p.S;
  const int held = min(ROWS, p.R - row0) * p.S;
  const __amdgpu_buffer_rsrc_t racc =
      __builtin_amdgcn_make_buffer_rsrc((void*)(p.part_acc + first * D), (short)0, held * D * (int)sizeof(float), 0x00020000);
  const __amdgpu_buffer_rsrc_t rml =
      __builtin_amdgcn_make_buffer_rsrc((void*)(p.part_ml + first), (short)0, held * (int)sizeof(f32x2), 0x00020000);
  lds_barrier();
#pragma unroll
  for (int k = 0; k < (ROWS + PER - 1) / PER; ++k) {
    const int r = threadIdx.x / QUADS + k * PER, row = row0 + r;
    if (r >= ROWS || row >= p.R) continue;
    f32x2 ml[NW];
    float m = REF_INIT, l = 0.f;
    f32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      ml[w] = s_ml[w][r];
      m = max_of(m, ml[w][0]);
    }
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = fast_exp2(ml[w][0] - m);
      l = fmaf(ml[w][1], f, l);
      acc += *reinterpret_cast<const f32x4*>(&s_o[w][r][4 * c]) * f;
    }
    if (p.S == 1) {
      b8_store<D>(p, h, row, c, acc, m, l, gate[k]);
    } else {
      const uint32_t at = (uint32_t)(r * p.S + sp);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc), racc, (int)((at * D + 4 * c) * sizeof(float)), 0, B8_COHERENT);
      if (c == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{m, l}), rml, (int)(at * sizeof(f32x2)), 0, B8_COHERENT);
    }
  }
  if constexpr (RB == 1) {
    // The last split of a row group to arrive adds all of them. Sums are stored and loaded device-coherent; every store of a
    // split is complete (vmcnt 0, then the workgroup's barrier) before its arrival is counted, and the last one's loads come
    // after its own count. It leaves the counter at zero.
    if (!p.arrivals) return;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    __shared__ int last_s;
    if (threadIdx.x == 0) {
      uint32_t* counter = p.arrivals + h * p.RG + blockIdx.z;
      last_s = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(p.S - 1);
      if (last_s) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last_s) return;
    constexpr int RP = PER / SPLIT_LANES, ROUNDS = (ROWS + RP - 1) / RP, FEW = 2;  // rows side by side
    static_assert(PER % SPLIT_LANES == 0 && NW >= SPLIT_LANES, "the split lanes' sums fit where the waves' were");
    const int u = threadIdx.x / QUADS, j = u / RP;
    if (p.S <= FEW * SPLIT_LANES) {  // the sums of all rows in flight at once (8 tokens, 16/4/128, 1001 keys: 14.0 -> 11.0 us)
      B8Splits<D, FEW> some[ROUNDS];
#pragma unroll
      for (int k = 0; k < ROUNDS; ++k) some[k].load(p, racc, rml, (k * RP + u % RP) * p.S, j, c);
#pragma unroll
      for (int k = 0; k < ROUNDS; ++k) {
        const int r = k * RP + u % RP;
        if (r >= ROWS) continue;
        float m = REF_INIT, l = 0.f;
        f32x4 acc = {0, 0, 0, 0};
        some[k].add(p, j, m, l, acc);
        *reinterpret_cast<f32x4*>(&s_o[j][r][4 * c]) = acc;
        if (c == 0) s_ml[j][r] = f32x2{m, l};
      }
    } else {
#pragma unroll 1
      for (int r = u % RP; r < ROWS && row0 + r < p.R; r += RP) b8_add_splits<D>(p, racc, rml, r * p.S, j, c, &s_o[j][r][4 * c], &s_ml[j][r]);
    }
    lds_barrier();
    for (int r = u; r < ROWS && row0 + r < p.R; r += PER)
      b8_finish_row<D>(p, h, row0 + r, c, &s_o[0][r][4 * c], &s_ml[0][r], ROWS * (D + 4), ROWS);
  }
}

// One workgroup for some rows of a KV head: the splits' sums added and finished. A chain of two loads: 4.0 us for 36 rows of 32
// splits (D = 128), 4.8 for 132 rows of 10 (D = 64).
template <int D>
__global__ __launch_bounds__(256) void attn_b8_merge_kernel(B8Attn p) {
  constexpr int Q = D / 4, RP = 256 / Q / SPLIT_LANES;
  __shared__ float s_acc[SPLIT_LANES][RP][D];
  __shared__ f32x2 s_ml[SPLIT_LANES][RP];
  const int h = blockIdx.y, c = threadIdx.x % Q, u = threadIdx.x / Q, r = u % RP, j = u / RP, row = blockIdx.x * RP + r;
  const size_t first = ((size_t)h * p.R + blockIdx.x * RP) * p.S;
  const int held = min(RP, p.R - (int)blockIdx.x * RP) * p.S;
  const __amdgpu_buffer_rsrc_t racc =
      __builtin_amdgcn_make_buffer_rsrc((void*)(p.part_acc + first * D), (short)0, held * D * (int)sizeof(float), 0x00020000);
  const __amdgpu_buffer_rsrc_t rml =
      __builtin_amdgcn_make_buffer_rsrc((void*)(p.part_ml + first), (short)0, held * (int)sizeof(f32x2), 0x00020000);
  if (row < p.R) b8_add_splits<D>(p, racc, rml, r * p.S, j, c, &s_acc[j][r][4 * c], &s_ml[j][r]);
  lds_barrier();
  if (row < p.R && j == 0) b8_finish_row<D>(p, h, row, c, &s_acc[0][r][4 * c], &s_ml[0][r], RP * D, RP);
}

// ---------------------------------------------------------------- accounts of attention weight
// mass_out[h][p] = (p < a ? mass_in[h][p] : 0) + sum over the rows of 2^(x - lse log2(e)), p < a + rows. A wave owns whole
// pages, so every key's sum is one wave's, in a fixed order and without atomics. K alone is read. The score product has its
// operands the other way round than the attention's (A = Q, B = K): a lane holds one key's scores of rows 4 g + i, adds them
// up in place over all row blocks, and only the four lanes of a key are added across (sums over the rows' lanes instead, with
// A = K, are eight row reductions a page: 39 us at 128k keys and 64 rows a head, 31 so). Bound by K's bytes and a fixed 4 us
// (131088 keys of 8 heads of 64, 64 rows: 21.4-22.0 us, 76 MB; 4107 keys 5.0). K is read of pages out of sight too.
template <int D, int RB, bool FP8>
__global__ __launch_bounds__(64 * MASS_WAVES, 2) void mass_b8_kernel(B8Attn p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const int h = blockIdx.y;
  const int rows = p.rows ? min(max(ldc(p.rows), 0), p.M) : p.M;
  const int end = p.page0 + p.npages;
  const int w0 = min(end, p.page0 + ((int)blockIdx.x * MASS_WAVES + wave) * p.pps), w1 = min(end, w0 + p.pps);
  const int live = p.a + rows, R = rows * p.G;
  const float* in = p.mass_in ? p.mass_in + (size_t)h * p.mass_stride : nullptr;
  float* out = p.mass_out + (size_t)h * p.mass_stride;
  // Every group of 16 RB rows in turn over the wave's pages: the first group stores in + sum, later ones add to that.
  for (int row0 = 0; row0 == 0 || row0 < R; row0 += 16 * RB) {
    half8 q[RB][D / 32];
    int tok[RB];
    b8_load_q<D, RB>(p, h, row0, lane, q, tok);
    // A row past the rows, or with lse -inf, adds nothing: l2 is -inf and its q zeros, so that its weights are 2^(0 - inf)
    // whatever q holds (a rejected draft's may be infinite or no number, and so would the score be).
    auto draws = [&](int row, float l) { return row < R && l != -INFINITY; };
    auto lse_of = [&](int row) {
      const int rc = min(row, p.R - 1), t = div_by(rc, p.g_div);
      return ldg(p.lse_in + (size_t)t * p.QH + h * p.G + rc - t * p.G);
    };
    float own[RB];  // of the row whose q the lane holds
    f32x4 l2[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      own[rb] = lse_of(row0 + 16 * rb + n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = row0 + 16 * rb + 4 * g + i;
        const float l = lse_of(row);
        l2[rb][i] = draws(row, l) ? l * -1.44269504088896341f : -INFINITY;
      }
    }
    for (int b0 = w0; b0 < w1; b0 += 64) {
      const int nb = min(64, w1 - b0);
      const int pgl = b8_page(p.c, b0 + min(lane, nb - 1));
      const float ksl = ldg(p.c.ks + (size_t)max(pgl, 0) * p.c.KVH + h) * p.c2;
      u32x4 k[2][2][D / 64];
      float old[2];
      // lane (n, g), g < 2, stores key 16 g + n
      auto load = [&](int i, u32x4 (&t)[2][D / 64], float& was) {
        const int kp = (b0 + i) * PAGE + 16 * (g & 1) + n;
        b8_load_k<D>(b8_block<D>(p.c.k, p.c.KVH, h, __builtin_amdgcn_readlane(pgl, i)), lane, t);
        const float* from = row0 ? out : in;
        was = from && kp < (row0 ? live : p.a) ? ldg(from + kp) : 0.f;
      };
      load(0, k[0], old[0]);
      if (b0 == w0)  // (behind the first page's loads: ahead of them it held them back by 0.5 us)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          if (!draws(row0 + 16 * rb + n, own[rb]))
#pragma unroll
            for (int e = 0; e < D / 32; ++e) q[rb][e] = half8{0, 0, 0, 0, 0, 0, 0, 0};
      auto step = [&](int i, const u32x4 (&now)[2][D / 64], float was, u32x4 (&next)[2][D / 64], float& then) {
        load(min(i + 1, nb - 1), next, then);
        const int lp = b0 + i;
        float acc[2] = {0.f, 0.f};
        if (__builtin_amdgcn_readlane(pgl, i) >= 0 && lp >= p.seen_lo && R > 0) {
          const float ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ksl), i));
          f32x4 x[RB][2];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            half8 kf[D / 32];
            b8_k_operand<D, FP8>(now[b], kf);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
              f32x4 s = {0, 0, 0, 0};
#pragma unroll
              for (int e = 0; e < D / 32; ++e) s = mfma16x16x32(q[rb][e], kf[e], s);
#pragma unroll
              for (int i = 0; i < 4; ++i) x[rb][b][i] = fmaf(s[i], ks, l2[rb][i]);
            }
          }
          if (lp < p.full_lo || lp >= p.full_hi) {
            int pos = lp * PAGE;
            asm volatile("" : "+s"(pos));  // (keeps the comparisons in this branch: they were made for every page)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const B8Sight sight = b8_sight(p, div_by(min(row0 + 16 * rb + 4 * g + i, p.R - 1), p.g_div));
#pragma unroll
                for (int b = 0; b < 2; ++b) x[rb][b][i] = sight.sees(pos + 16 * b + n) ? x[rb][b][i] : -INFINITY;
              }
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            f32x4 sum = {0, 0, 0, 0};
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
              for (int i = 0; i < 4; ++i) sum[i] += fast_exp2(x[rb][b][i]);
            acc[b] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
          }
        }
        const float v0 = row_sum(acc[0]), v1 = row_sum(acc[1]);  // (the exchanges take every lane: no branch around them)
        const int kp = lp * PAGE + 16 * (g & 1) + n;
        if (g < 2 && kp < live) out[kp] = was + (g ? v1 : v0);
      };
      __builtin_amdgcn_s_setprio(3);  // (as in the attention: who is further on yields)
      for (int i = 0; i < nb; i += 2) {
        if (4 * i >= nb) __builtin_amdgcn_s_setprio(2);
        if (2 * i >= nb) __builtin_amdgcn_s_setprio(1);
        if (4 * i >= 3 * nb) __builtin_amdgcn_s_setprio(0);
        step(i, k[0], old[0], k[1], old[1]);
        if (i + 1 < nb) step(i + 1, k[1], old[1], k[0], old[0]);
      }
    }
  }
}

// ---------------------------------------------------------------- plans and launches
constexpr int B8_ROW_BLOCKS = 4;  // most 16-row blocks of a row group (2 at D = 128)

// Which pages any row sees, and which every row sees whole.
static void b8_range(B8Attn& p, int D) {
  const int lo = std::min(p.a, std::max(p.start, p.window > 0 ? p.a - p.window + 1 : 0));  // first key any row sees
  p.page0 = lo / PAGE;
  p.npages = (p.a + p.M - 1) / PAGE + 1 - p.page0;
  const int whole = std::max(p.start, p.window > 0 ? p.a + p.M - p.window : 0);            // first context key all rows see
  p.full_lo = whole / PAGE + (whole % PAGE > 0);
  p.full_hi = p.a / PAGE;
  p.c2 = 1.4426950408889634f / std::sqrt((float)D);
}

void b8_attn_plan(B8Attn& p, int D, int splits, int cus) {
  p.R = p.G * p.M;
  p.g_div = div_magic((uint32_t)p.G);
  b8_range(p, D);
  const int blocks = (p.R + 15) / 16, most = D == 64 ? B8_ROW_BLOCKS : 2;
  p.RG = (blocks + most - 1) / most;
  p.rb = (blocks + p.RG - 1) / p.RG;
  // Few pages: a row block a workgroup, up to two pages a wave in one split (16 tokens, 32/8/64 heads, 500 keys: 5.7 us, 7.6 with
  // a page a wave; three and four a wave lose to splits at 16/4/128, 1001 keys 11.6 against 10.9), then splits of a page a wave
  // as far as there are CUs -- at D = 64 up to four pages a wave (1000 keys 9.8 -> 8.0 us against row groups of four blocks,
  // 4000 10.3 -> 8.9, 8000 11.5 -> 10.4, 16000 13.1 -> 12.7), at D = 128 to one (8 tokens, 16/4/128: 250 keys 10.5 -> 7.0,
  // 1001 10.7 -> 10.9 but without a second launch, 16000 13.1 -> 14.2 with two).
  const int w1 = b8_waves(D, 1), most1 = cus / (p.c.KVH * blocks);
  if (splits == 0 && most1 > 0 && p.npages <= (D == 64 ? 4 : 1) * w1 * most1) {
    p.rb = 1;
    p.RG = blocks;
    splits = p.npages <= 2 * w1 ? 1 : std::min(most1, (p.npages + w1 - 1) / w1);
  }
  const int waves = b8_waves(D, p.rb);
  int S = splits > 0 ? splits : std::max(1, cus / (p.c.KVH * p.RG));
  S = std::max(1, std::min(std::min(S, 4096), (p.npages + waves - 1) / waves));
  p.S = S;
  // The last split to arrive adds the others (if the caller has counters) where they are little to read for one workgroup: a
  // token of 32768 keys takes 12.8 us instead of 11.9 with a second launch, whose caller spends 4 more on it; 32 rows of
  // 131063 keys in one workgroup 46 against 38.
  if (S == 1 || p.rb > 1 || std::min(p.R, 16) * S * D * (int)sizeof(float) > B8_FUSED_BYTES) p.arrivals = nullptr;
  p.pps = p.npages / (S * waves);
  p.more = p.npages % (S * waves);
}

size_t b8_attn_workspace(const B8Attn& p, int D) {
  if (p.S == 1) return 0;
  const size_t rows = (size_t)p.c.KVH * p.R * p.S;
  return rows * D * sizeof(float) + rows * sizeof(f32x2);
}

template <int D, int RB, bool FP8>
static void attn_b8_rows(const B8Attn& p, hipStream_t s) {
  hipLaunchKernelGGL((attn_b8_kernel<D, RB, FP8>), dim3(p.S, p.c.KVH, p.RG), dim3(64 * b8_waves(D, RB)), 0, s, p);
}
template <int D, bool FP8>
static void attn_b8_by_rows(const B8Attn& p, hipStream_t s) {
  if (p.rb == 1) return attn_b8_rows<D, 1, FP8>(p, s);
  if (p.rb == 2) return attn_b8_rows<D, 2, FP8>(p, s);
  if constexpr (D == 64) {
    if (p.rb == 3) return attn_b8_rows<D, 3, FP8>(p, s);
    return attn_b8_rows<D, 4, FP8>(p, s);
  }
}

int b8_attn_launch(const B8Attn& p, int D, bool fp8, hipStream_t s) {
  if (D == 64) fp8 ? attn_b8_by_rows<64, true>(p, s) : attn_b8_by_rows<64, false>(p, s);
  else fp8 ? attn_b8_by_rows<128, true>(p, s) : attn_b8_by_rows<128, false>(p, s);
  if (const int rc = (int)hipGetLastError()) return rc;
  if (p.S == 1 || p.arrivals) return 0;
  const int rows = 256 / (D / 4) / SPLIT_LANES;
  const dim3 grid((p.R + rows - 1) / rows, p.c.KVH);
  if (D == 64) hipLaunchKernelGGL(attn_b8_merge_kernel<64>, grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL(attn_b8_merge_kernel<128>, grid, dim3(256), 0, s, p);
  return (int)hipGetLastError();
}

template <int D, bool FP8>
static void mass_b8_by_rows(const B8Attn& p, dim3 grid, hipStream_t s) {
  const dim3 block(64 * MASS_WAVES);
  switch (p.rb) {
    case 1: hipLaunchKernelGGL((mass_b8_kernel<D, 1, FP8>), grid, block, 0, s, p); break;
    case 2: hipLaunchKernelGGL((mass_b8_kernel<D, 2, FP8>), grid, block, 0, s, p); break;
    case 3: hipLaunchKernelGGL((mass_b8_kernel<D, 3, FP8>), grid, block, 0, s, p); break;
    default: hipLaunchKernelGGL((mass_b8_kernel<D, 4, FP8>), grid, block, 0, s, p); break;
  }
}

int b8_mass_launch(const B8Attn& q, int D, bool fp8, int cus, hipStream_t s) {
  B8Attn p = q;
  p.R = p.G * p.M;
  p.rb = std::min(B8_ROW_BLOCKS, (p.R + 15) / 16);
  p.g_div = div_magic((uint32_t)p.G);
  b8_range(p, D);
  p.seen_lo = p.page0;
  p.page0 = 0;  // every account is carried over, those of keys out of sight too
  p.npages = (p.a + p.M - 1) / PAGE + 1;
  // as many pages a wave as let every workgroup start at once (131088 keys, 64 rows a head, when a page still cost more: 26.0 us,
  // 27.8 with a few workgroups over)
  const int64_t waves = (int64_t)cus * (p.rb > 2 ? 12 : 16);
  p.pps = (int)std::max<int64_t>(1, ((int64_t)p.npages * p.c.KVH + waves - 1) / waves);
  const dim3 grid((p.npages + p.pps * MASS_WAVES - 1) / (p.pps * MASS_WAVES), p.c.KVH);
  if (D == 64) fp8 ? mass_b8_by_rows<64, true>(p, grid, s) : mass_b8_by_rows<64, false>(p, grid, s);
  else fp8 ? mass_b8_by_rows<128, true>(p, grid, s) : mass_b8_by_rows<128, false>(p, grid, s);
  return (int)hipGetLastError();
}

}  // namespace dspark
