// The 8-bit block-scaled K/V cache: appending, reading back and evicting.
//
// A block is the 32 positions of one (page, KV head), of K or of V: 32 x D one-byte codes, rows of D bytes in position
// order, and one fp32 scale; value = code * scale (b8.h has the arithmetic). Rows are kept whole and in order -- the
// attention transposes V in registers, by D / 8 of the 220 to 370 vector instructions that a page costs a wave -- so that a
// position is D contiguous bytes to the writer, the reader and the eviction.
#include "b8.h"
#include "dspark.h"

namespace dspark {

constexpr int WPB = 4;  // waves per workgroup; a wave owns one block

// ---------------------------------------------------------------- append
// One wave per (page, K or V, head): the block's new rows are read once (16 bytes a lane, every load in flight before the
// first is used), their largest finite magnitude gives the scale, and the codes are stored 8 bytes a lane. Only the first
// page can hold earlier rows (pos0 inside it): they stay, re-coded where the scale grew. Slots behind the last row are
// cleared. Bound by the rows' fp16 bytes for prompts (32768 rows of 4 heads of 128: 21.4 us, 100.7 MB read and written, 4.7 TB/s)
// and by one chain (table, rows, reduction, store) for a block (16 rows of 8 heads of 64: 3.1 us, 8192 of them 11.6).
template <int D, bool FP8>
__global__ __launch_bounds__(64 * WPB) void kv_write_b8_kernel(B8Write p, int nwaves) {
  constexpr int LPR = D / 8, RPI = 64 / LPR, NI = PAGE / RPI;  // lanes per row, rows per instruction, instructions
  const int w = blockIdx.x * WPB + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (w >= nwaves) return;
  const int KVH = p.c.KVH, h = w % KVH, kv = (w / KVH) & 1, lp = p.pos0 / PAGE + w / (2 * KVH);
  const int pg = b8_page(p.c, lp);
  if (pg < 0) return;
  const size_t blk = (size_t)pg * KVH + h;
  const _Float16* src = (kv ? p.v : p.k) + (size_t)h * D;
  uint8_t* dst = (kv ? p.c.v : p.c.k) + blk * (PAGE * D);
  float* scale = (kv ? p.c.vs : p.c.ks) + blk;
  const int base = lp * PAGE - p.pos0;  // row of x that slot 0 takes
  const int r = lane / LPR, c = lane % LPR;
  half8 x[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row = min(max(base + r + RPI * i, 0), p.n - 1);
    x[i] = as_half8(ldg(reinterpret_cast<const u32x4*>(src + (size_t)row * p.row_stride + 8 * c)));
  }
  const bool entered = base < 0;  // the page holds earlier rows
  const float was = entered ? ldg(scale) : 0.f;
  // Largest magnitude: for non-negative halves the order of the patterns is that of the values, so two are compared by one
  // packed maximum. Patterns from 0x7c00 on are infinities and NaN: only if there is one are the finite values picked out.
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 most = {0, 0};
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row = base + r + RPI * i;
    u32x4 w;
    __builtin_memcpy(&w, &x[i], 16);
    if (row < 0 || row >= p.n) w = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w[j] & 0x7fff7fffu));
  }
  uint32_t top = wave_max_u32(max((uint32_t)most[0], (uint32_t)most[1]));
  const bool any = top >= 0x7c00u;
  if (any) {
    top = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = base + r + RPI * i;
      if (row >= 0 && row < p.n)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t b = __builtin_bit_cast(uint16_t, (_Float16)x[i][j]) & 0x7fffu;
          top = max(top, b < 0x7c00u ? b : 0u);
        }
    }
    top = wave_max_u32(top);
  }
  const float s = fmaxf(was, b8_scale<FP8>((float)__builtin_bit_cast(_Float16, (uint16_t)top)));
  const float inv = b8_inv(s);
  if (lane == 0) *scale = s;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int slot = r + RPI * i, row = base + slot;
    u32x2* at = reinterpret_cast<u32x2*>(dst + slot * D + 8 * c);
    u32x2 y;
    if (row >= 0) {
      const half8 v = x[i];
      if (any) {
        y[0] = b8_code4<FP8, true>((float)v[0], (float)v[1], (float)v[2], (float)v[3], s, inv);
        y[1] = b8_code4<FP8, true>((float)v[4], (float)v[5], (float)v[6], (float)v[7], s, inv);
      } else {
        y[0] = b8_code4<FP8, false>((float)v[0], (float)v[1], (float)v[2], (float)v[3], s, inv);
        y[1] = b8_code4<FP8, false>((float)v[4], (float)v[5], (float)v[6], (float)v[7], s, inv);
      }
      if (row >= p.n) y = u32x2{0, 0};
      *at = y;
    } else if (s != was) {
      y = ldg(at);
      y[0] = b8_recode4<FP8>(y[0], was, s, inv);
      y[1] = b8_recode4<FP8>(y[1], was, s, inv);
      *at = y;
    }
  }
}

// ---------------------------------------------------------------- read back
// One wave per (page, K or V, head): 4 codes a lane, so that a store is 1 KB of whole row pieces. Bound by what it writes, four
// times what it reads (32768 rows of 4 heads of 128: 25.4 us, 167.8 MB, 6.6 TB/s).
template <int D, bool FP8>
__global__ __launch_bounds__(64 * WPB) void kv_read_b8_kernel(B8Read p, int nwaves) {
  constexpr int LPR = D / 4, RPI = 64 / LPR, NI = PAGE / RPI;
  const int w = blockIdx.x * WPB + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (w >= nwaves) return;
  const int KVH = p.c.KVH, h = w % KVH, kv = (w / KVH) & 1, lp = p.pos0 / PAGE + w / (2 * KVH);
  const int pg = b8_page(p.c, lp);
  const size_t blk = (size_t)max(pg, 0) * KVH + h;
  const uint8_t* src = (kv ? p.c.v : p.c.k) + blk * (PAGE * D);
  const float s = pg < 0 ? 0.f : ldg((kv ? p.c.vs : p.c.ks) + blk);
  float* out = (kv ? p.v : p.k) + (size_t)h * D;
  const int base = lp * PAGE - p.pos0, r = lane / LPR, c = lane % LPR;
  uint32_t y[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) y[i] = pg < 0 ? 0u : ldg(reinterpret_cast<const uint32_t*>(src + (r + RPI * i) * D + 4 * c));
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row = base + r + RPI * i;
    if (row >= 0 && row < p.n)
      *reinterpret_cast<f32x4*>(out + (size_t)row * p.row_stride + 4 * c) = b8_value4<FP8>(y[i]) * s;
  }
}

// ---------------------------------------------------------------- eviction
// Order of the accounts: as the values are, NaN below all of them, -0 as 0.
__device__ __forceinline__ uint32_t mass_key(float v) { return v != v ? 0u : argmax_ord(v + 0.f); }

constexpr int SEL_T = 1024, SEL_W = SEL_T / 64, SEL_BINS = 2048;
// Radix selection over the keys' bits 31-21, 20-10 and 9-0.
constexpr int sel_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
constexpr int sel_bins(int pass) { return pass == 2 ? 1024 : 2048; }

// Inclusive sum over the lanes of a row of 16 up to this one, and over the lanes of the wave up to this one.
template <int N>
__device__ __forceinline__ uint32_t row_shr_add(uint32_t v) {
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x110 + N, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t row_scan(uint32_t v) { return row_shr_add<8>(row_shr_add<4>(row_shr_add<2>(row_shr_add<1>(v)))); }
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = row_scan(v);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // row 0's last lane to row 1, 2's to 3
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);  // lane 31 to rows 2 and 3
}
__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
  return wave_butterfly(v, [](uint32_t a, uint32_t b) { return a + b; });
}

// Where the need-th largest of the counted keys lies: its bin and how many lie in higher bins. Thread t holds the counts n1, n0
// of bins b1 = bins - 1 - 2 t and b1 - 1 (0 past the bins); 1 <= need <= the number counted.
struct SelLds {
  uint32_t wsum[SEL_W];
  uint32_t found[2];
};
__device__ __forceinline__ void sel_find(SelLds& s, int bins, uint32_t n1, uint32_t n0, uint32_t need, uint32_t& bin,
                                         uint32_t& above) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t sum = wave_scan(n1 + n0);
  if (lane == 63) s.wsum[wave] = sum;
  __syncthreads();
  const uint32_t upto = row_scan(s.wsum[lane % SEL_W]);
  const uint32_t before = sum - n1 - n0 + (wave ? (uint32_t)__builtin_amdgcn_readlane((int)upto, max(wave - 1, 0)) : 0u);
  const int b1 = bins - 1 - 2 * tid;
  if (before < need && need <= before + n1 + n0) {
    const bool low = need > before + n1;
    s.found[0] = (uint32_t)(b1 - low);
    s.found[1] = before + (low ? n1 : 0u);
  }
  __syncthreads();
  bin = s.found[0];
  above = s.found[1];
}

__device__ __forceinline__ void sel_edges(const B8Evict& p, int32_t* kept, int first, int step) {
  for (int i = first; i < p.sinks; i += step) kept[i] = i;
  for (int i = first; i < p.recent; i += step) kept[p.keep - p.recent + i] = p.T - p.recent + i;
}

// A wave's 64 NPL keys: u[4 j + e] of position i0 + 256 j + 4 lane + e, so that a lane's four are one load and places come from
// one scan over the lanes for 256 positions.
template <int NPL>
__device__ __forceinline__ void sel_load(const float* mass, int i0, int N, uint32_t (&u)[NPL]) {
  typedef __attribute__((address_space(1))) const f32x4 __attribute__((aligned(4))) GV;  // the accounts' rows start at any word
  f32x4 v[NPL / 4];
#pragma unroll
  for (int j = 0; j < NPL / 4; ++j) {
    const int i = i0 + 256 * j + 4 * (threadIdx.x & 63);
    if (i + 4 <= N) {
      v[j] = *(GV*)(mass + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = i + e < N ? ldg(mass + i + e) : 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < NPL; ++k) u[k] = mass_key(v[k / 4][k % 4]);
}
__device__ __forceinline__ int sel_pos(int i0, int k) { return i0 + 256 * (k / 4) + 4 * (int)(threadIdx.x & 63) + k % 4; }
// A lane's keys above the threshold (low half) and equal to it (high half) among its four of group j.
template <int NPL>
__device__ __forceinline__ uint32_t sel_mark(const uint32_t (&u)[NPL], int j, int i0, int N, uint32_t thr) {
  uint32_t c = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t x = u[4 * j + e];
    c += sel_pos(i0, 4 * j + e) < N ? (x > thr ? 1u : 0u) + (x == thr ? 0x10000u : 0u) : 0u;
  }
  return c;
}
template <int NPL>
__device__ __forceinline__ uint32_t sel_count(const uint32_t (&u)[NPL], int i0, int N, uint32_t thr) {
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < NPL / 4; ++j) c += sel_mark<NPL>(u, j, i0, N, thr);
  return wave_total(c);
}
// Stores the kept ones: a key above the threshold, or one of the first `need` equal to it, goes to place
// sinks + (keys above before it) + min(need, equal ones before it); gt, eq: those before the wave's first.
template <int NPL>
__device__ __forceinline__ void sel_emit(const uint32_t (&u)[NPL], int i0, int N, uint32_t thr, uint32_t need, uint32_t gt, uint32_t eq,
                                         int sinks, int32_t* kept) {
#pragma unroll
  for (int j = 0; j < NPL / 4; ++j) {
    if (i0 + 256 * j >= N) break;
    const uint32_t c = sel_mark<NPL>(u, j, i0, N, thr), upto = wave_scan(c);
    uint32_t g = gt + ((upto - c) & 0xffffu), q = eq + ((upto - c) >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = sel_pos(i0, 4 * j + e);
      const bool above = i < N && u[4 * j + e] > thr, same = i < N && u[4 * j + e] == thr;
      if (above || (same && q < need)) kept[sinks + g + min(q, need)] = sinks + i;
      g += above;
      q += same;
    }
    const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    gt += all & 0xffffu;
    eq += all >> 16;
  }
}
// The counts of the waves before this one (wc: every wave's, complete and visible), and of all of them.
__device__ __forceinline__ uint32_t sel_before(const uint32_t* wc, int wave, uint32_t& all) {
  const uint32_t upto = row_scan(wc[threadIdx.x % SEL_W]);
  all = (uint32_t)__builtin_amdgcn_readlane((int)upto, SEL_W - 1);
  return wave ? (uint32_t)__builtin_amdgcn_readlane((int)upto, max(wave - 1, 0)) : 0u;
}

// One workgroup per KV head finds the keep - sinks - recent largest accounts of up to 1024 NPL middle positions, held in
// registers, and lists what is kept in position order. Bound by its chain of phases (three digits of clear, count, scan):
// 9.9-10.1 us for 8449 positions.
template <int NPL>
__global__ __launch_bounds__(SEL_T) void evict_select_kernel(B8Evict p) {
  __shared__ SelLds s;
  __shared__ __align__(16) uint32_t hist[SEL_BINS];
  __shared__ uint32_t wc[SEL_W];
  const int h = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float* mass = p.mass + (size_t)h * p.mass_stride + p.sinks;
  int32_t* kept = p.kept + (size_t)h * p.keep;
  const int N = p.T - p.sinks - p.recent, k = p.keep - p.sinks - p.recent;
  const int per = (N + 256 * SEL_W - 1) / (256 * SEL_W) * 256, i0 = wave * per, hi = min(N, i0 + per);  // whole groups a wave
  uint32_t u[NPL];
  sel_load<NPL>(mass, i0, hi, u);
  sel_edges(p, kept, tid, SEL_T);
  if (k <= 0) return;
  uint32_t thr = 0, mask = 0, need = (uint32_t)k;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = sel_shift(pass), bins = sel_bins(pass);
    for (int i = tid; i < bins; i += SEL_T) hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (sel_pos(i0, j) < hi && (u[j] & mask) == thr) atomicAdd(&hist[(u[j] >> shift) & (bins - 1)], 1u);
    __syncthreads();
    const u32x2 n = 2 * tid < bins ? *reinterpret_cast<const u32x2*>(&hist[bins - 2 - 2 * tid]) : u32x2{0, 0};
    uint32_t bin, above;
    sel_find(s, bins, n[1], n[0], need, bin, above);
    thr |= bin << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    need -= above;
  }
  const uint32_t c = sel_count<NPL>(u, i0, hi, thr);
  if (lane == 0) wc[wave] = c;
  __syncthreads();
  uint32_t all;
  const uint32_t before = sel_before(wc, wave, all);  // (up to 16384 of each: the halves do not meet)
  sel_emit<NPL>(u, i0, hi, thr, need, before & 0xffffu, before >> 16, p.sinks, kept);
}

// More positions: `parts` workgroups a head, each a contiguous range of them (whole tiles of 8192), and a launch for each
// digit. A workgroup stores its own histogram; the next launch's workgroups each add up all of the head's (from L2), find the
// digit, and count the next one among their keys that match so far. The last launch knows from the parts' counts where each
// part's first kept key goes. No atomics in memory, and no state from one call to the next. Each launch is a chain (histograms
// or keys, counts in LDS, a scan, a store): 3.4-3.7 us, then 5.6-6.1 each, for 130044 positions of 4 heads.
constexpr int SEL_NPL = 8, SEL_TILE = SEL_T * SEL_NPL, SEL_PARTS = 32;
struct SelHead {  // a head's part of the workspace, a u32 each
  uint32_t hist[3][SEL_PARTS][SEL_BINS];
  uint32_t above[2][SEL_PARTS];  // a part's keys over the threshold by digit 0, by digit 1
  uint32_t state[2][2];          // after digit 0 and 1: threshold so far, keys still needed at it
};
template <int PASS>
__global__ __launch_bounds__(SEL_T) void evict_pass_kernel(B8Evict p, SelHead* ws, int parts, int per) {
  __shared__ SelLds s;
  __shared__ __align__(16) uint32_t hist[SEL_BINS];
  __shared__ uint32_t wc[SEL_W];
  __shared__ uint32_t red[2];
  const int h = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  SelHead& w = ws[h];
  const float* mass = p.mass + (size_t)h * p.mass_stride + p.sinks;
  int32_t* kept = p.kept + (size_t)h * p.keep;
  const int N = p.T - p.sinks - p.recent;
  const int lo = part * per, hi = min(N, lo + per);
  uint32_t u[SEL_NPL];
  const int w0 = wave * 64 * SEL_NPL;
  sel_load<SEL_NPL>(mass, lo + w0, N, u);  // the first tile's keys, in flight while the digit is found
  uint32_t thr = 0, mask = 0, need = (uint32_t)(p.keep - p.sinks - p.recent);
  uint32_t gt = 0, eq = 0;  // PASS 3: kept and equal keys in the parts before
  if constexpr (PASS > 0) {  // the digit of the launch before
    constexpr int prev = PASS - 1, bins = sel_bins(prev);
    if (PASS > 1) {
      thr = ldg(&w.state[PASS - 2][0]);
      need = ldg(&w.state[PASS - 2][1]);
      mask = (uint32_t)(sel_bins(0) - 1) << sel_shift(0);
    }
    if (tid < 2) red[tid] = 0;
    // this thread's two bins in every part: all of them, this part's own, and those of the parts before it
    u32x2 all = {0, 0}, mine = {0, 0}, ahead = {0, 0};
    if (2 * tid < bins) {
      const u32x2* at = reinterpret_cast<const u32x2*>(&w.hist[prev][0][bins - 2 - 2 * tid]);
#pragma unroll 16
      for (int q = 0; q < parts; ++q) {
        const u32x2 n = ldg(at + (size_t)q * (SEL_BINS / 2));
        all += n;
        if (q == part) mine = n;
        if (q < part) ahead += n;
      }
    }
    uint32_t bin, above;
    sel_find(s, bins, all[1], all[0], need, bin, above);
    thr |= bin << sel_shift(prev);
    need -= above;
    mask |= (uint32_t)(bins - 1) << sel_shift(prev);
    const uint32_t b1 = (uint32_t)(bins - 1 - 2 * tid);
    if (2 * tid < bins) {
      const u32x2 n = PASS < 3 ? mine : ahead;
      gt = (b1 > bin ? n[1] : 0u) + (b1 - 1 > bin ? n[0] : 0u);
      eq = (b1 == bin ? n[1] : 0u) + (b1 - 1 == bin ? n[0] : 0u);
    }
    if (PASS == 3 && tid < part) gt += ldg(&w.above[0][tid]) + ldg(&w.above[1][tid]);
    gt = wave_total(gt);
    eq = wave_total(eq);
    if (lane == 0 && gt) atomicAdd(&red[0], gt);
    if (lane == 0 && eq) atomicAdd(&red[1], eq);
    __syncthreads();
    gt = red[0];
    eq = red[1];
    if (PASS < 3 && tid == 0) {
      w.above[PASS - 1][part] = gt;  // keys of this part that the digit puts over the threshold
      if (part == 0) {
        w.state[PASS - 1][0] = thr;
        w.state[PASS - 1][1] = need;
      }
    }
  }
  if constexpr (PASS < 3) {
    constexpr int bins = sel_bins(PASS), shift = sel_shift(PASS);
    for (int i = tid; i < bins; i += SEL_T) hist[i] = 0;
    __syncthreads();
    for (int t0 = lo; t0 < hi; t0 += SEL_TILE) {
      if (t0 > lo) sel_load<SEL_NPL>(mass, t0 + w0, N, u);
#pragma unroll
      for (int j = 0; j < SEL_NPL; ++j)
        if (sel_pos(t0 + w0, j) < hi && (u[j] & mask) == thr) atomicAdd(&hist[(u[j] >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int i = tid; i < bins; i += SEL_T) w.hist[PASS][part][i] = hist[i];
  } else {
    if (part == 0) sel_edges(p, kept, tid, SEL_T);
    for (int t0 = lo; t0 < hi; t0 += SEL_TILE) {
      if (t0 > lo) sel_load<SEL_NPL>(mass, t0 + w0, N, u);
      const uint32_t c = sel_count<SEL_NPL>(u, t0 + w0, hi, thr);
      if (lane == 0) wc[wave] = c;
      __syncthreads();
      uint32_t all;
      const uint32_t before = sel_before(wc, wave, all);
      sel_emit<SEL_NPL>(u, t0 + w0, hi, thr, need, gt + (before & 0xffffu), eq + (before >> 16), p.sinks, kept);
      gt += all & 0xffffu;  // on to the next tile
      eq += all >> 16;
      __syncthreads();
    }
  }
}

__global__ __launch_bounds__(SEL_T) void evict_edges_kernel(B8Evict p) {
  sel_edges(p, p.kept + (size_t)blockIdx.x * p.keep, threadIdx.x, SEL_T);
}

// One wave per (destination page, K or V, head): 32 kept rows gathered 16 bytes a lane into one block. Its scale is the
// largest of its rows' scales: rows that had it keep their codes, the others are re-coded to it. Bound by the chain kept ->
// table -> rows and the gather (16384 rows of 4 heads of 128: 8.8-9.0 us, 37 MB, 4.2 TB/s; 8192 of 8 heads of 64, int8: 9.8-10.1; with the
// rows' loads ahead of the scales' use the same).
template <int D, bool FP8>
__global__ __launch_bounds__(64 * WPB) void evict_move_kernel(B8Evict p, int nwaves) {
  constexpr int LPR = D / 16, RPI = 64 / LPR, NI = PAGE / RPI;
  const int w = blockIdx.x * WPB + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (w >= nwaves) return;
  const int KVH = p.src.KVH, h = w % KVH, kv = (w / KVH) & 1, lp = w / (2 * KVH);
  const int slot0 = lp * PAGE, live = min(PAGE, p.keep - slot0);
  // lane i < 32 knows row i's source
  const bool mine = lane < live;
  const int pos = ldg(p.kept + (size_t)h * p.keep + slot0 + min(lane, live - 1));
  const int pg = b8_page(p.src, pos / PAGE);
  const float s_from = mine && pg >= 0 ? ldg((kv ? p.src.vs : p.src.ks) + (size_t)pg * KVH + h) : 0.f;
  if (kv == 0 && mine) p.mass_out[(size_t)h * p.mass_out_stride + slot0 + lane] = ldg(p.mass + (size_t)h * p.mass_stride + pos);
  const int dpg = b8_page(p.dst, lp);
  if (dpg < 0) return;
  const size_t blk = (size_t)dpg * KVH + h;
  const float s = wave_max(s_from), inv = b8_inv(s);
  if (lane == 0) *((kv ? p.dst.vs : p.dst.ks) + blk) = s;
  const uint8_t* from = kv ? p.src.v : p.src.k;
  uint8_t* to = (kv ? p.dst.v : p.dst.k) + blk * (PAGE * D);
  const int r = lane / LPR, c = lane % LPR;
  u32x4 y[NI];
  float sf[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row = r + RPI * i;
    const int rp = __shfl(pos, row), rpg = __shfl(pg, row);
    sf[i] = __shfl(s_from, row);
    y[i] = u32x4{0, 0, 0, 0};
    if (row < live && rpg >= 0)
      y[i] = ldg(reinterpret_cast<const u32x4*>(from + ((size_t)rpg * KVH + h) * (PAGE * D) + (rp % PAGE) * D + 16 * c));
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    if (sf[i] != s)
#pragma unroll
      for (int j = 0; j < 4; ++j) y[i][j] = b8_recode4<FP8>(y[i][j], sf[i], s, inv);
    *reinterpret_cast<u32x4*>(to + (r + RPI * i) * D + 16 * c) = y[i];
  }
}

// ---------------------------------------------------------------- launches
template <typename F>
static int by_kind(int D, bool fp8, F f) {
  if (D == 64) fp8 ? f(std::integral_constant<int, 64>(), std::true_type()) : f(std::integral_constant<int, 64>(), std::false_type());
  else fp8 ? f(std::integral_constant<int, 128>(), std::true_type()) : f(std::integral_constant<int, 128>(), std::false_type());
  return (int)hipGetLastError();
}
static int waves_of(int pos0, int n, int KVH) { return ((pos0 + n - 1) / PAGE - pos0 / PAGE + 1) * 2 * KVH; }

int b8_write_launch(const B8Write& p, int D, bool fp8, hipStream_t s) {
  if (p.n == 0) return 0;
  const int nw = waves_of(p.pos0, p.n, p.c.KVH);
  return by_kind(D, fp8, [&](auto d, auto f) {
    hipLaunchKernelGGL((kv_write_b8_kernel<decltype(d)::value, decltype(f)::value>), dim3((nw + WPB - 1) / WPB), dim3(64 * WPB),
                       0, s, p, nw);
  });
}
int b8_read_launch(const B8Read& p, int D, bool fp8, hipStream_t s) {
  if (p.n == 0) return 0;
  const int nw = waves_of(p.pos0, p.n, p.c.KVH);
  return by_kind(D, fp8, [&](auto d, auto f) {
    hipLaunchKernelGGL((kv_read_b8_kernel<decltype(d)::value, decltype(f)::value>), dim3((nw + WPB - 1) / WPB), dim3(64 * WPB), 0,
                       s, p, nw);
  });
}
// Up to 16384 middle positions in one launch, from 16 keys a lane; more by parts. (One workgroup a head with passes over memory
// for every length took 18 us for 8449 positions and 160 for 130044, against 9.9 and 20.6.)
constexpr int SEL_ONE = 16 * SEL_T;
size_t b8_evict_workspace(int KVH, int length) { return length > SEL_ONE ? (size_t)KVH * sizeof(SelHead) : 0; }

int b8_evict_launch(const B8Evict& p, int D, bool fp8, void* ws, hipStream_t s) {
  const int N = p.T - p.sinks - p.recent, KVH = p.src.KVH;
  if (N <= 4 * SEL_T) {
    hipLaunchKernelGGL(evict_select_kernel<4>, dim3(KVH), dim3(SEL_T), 0, s, p);
  } else if (N <= SEL_ONE) {
    hipLaunchKernelGGL(evict_select_kernel<16>, dim3(KVH), dim3(SEL_T), 0, s, p);
  } else {
    const int tiles = (N + SEL_TILE - 1) / SEL_TILE, each = (tiles + SEL_PARTS - 1) / SEL_PARTS;
    const int parts = (tiles + each - 1) / each, per = each * SEL_TILE;
    SelHead* w = static_cast<SelHead*>(ws);
    const dim3 grid(parts, KVH), block(SEL_T);
    if (p.keep > p.sinks + p.recent) {
      hipLaunchKernelGGL(evict_pass_kernel<0>, grid, block, 0, s, p, w, parts, per);
      hipLaunchKernelGGL(evict_pass_kernel<1>, grid, block, 0, s, p, w, parts, per);
      hipLaunchKernelGGL(evict_pass_kernel<2>, grid, block, 0, s, p, w, parts, per);
      hipLaunchKernelGGL(evict_pass_kernel<3>, grid, block, 0, s, p, w, parts, per);
    } else {  // nothing of the middle is kept
      hipLaunchKernelGGL(evict_edges_kernel, dim3(KVH), block, 0, s, p);
    }
  }
  if (const int rc = (int)hipGetLastError()) return rc;
  const int nw = (p.keep + PAGE - 1) / PAGE * 2 * p.src.KVH;
  return by_kind(D, fp8, [&](auto d, auto f) {
    hipLaunchKernelGGL((evict_move_kernel<decltype(d)::value, decltype(f)::value>), dim3((nw + WPB - 1) / WPB), dim3(64 * WPB), 0,
                       s, p, nw);
  });
}

}  // namespace dspark
