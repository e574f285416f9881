// The 8-bit block-scaled K/V cache: appending, reading back and evicting.
//
// A block is the 32 positions of one (page, KV head), of K or of V: 32 x D one-byte codes, rows of D bytes in position
// order, and one fp32 scale; value = code * scale (b8.h has the arithmetic). Rows are kept whole and in order -- the
// attention transposes V in registers, which costs it under a tenth of its issue -- so that a position is D contiguous
// bytes to the writer, the reader and the eviction.
#include "b8.h"
#include "dspark.h"

namespace dspark {

constexpr int WPB = 4;  // waves per workgroup; a wave owns one block

// ---------------------------------------------------------------- append
// One wave per (page, K or V, head): the block's new rows are read once (16 bytes a lane, every load in flight before the
// first is used), their largest finite magnitude gives the scale, and the codes are stored 8 bytes a lane. Only the first
// page can hold earlier rows (pos0 inside it): they stay, re-coded where the scale grew. Slots behind the last row are
// cleared. Bound by the rows' fp16 bytes for prompts and by one chain (table, rows, reduction, store) for a block.
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
  uint32_t top = 0;  // largest finite magnitude: for non-negative halves the order of the patterns is that of the values
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
      y[0] = b8_code4<FP8>((float)v[0], (float)v[1], (float)v[2], (float)v[3], s, inv);
      y[1] = b8_code4<FP8>((float)v[4], (float)v[5], (float)v[6], (float)v[7], s, inv);
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
// One wave per (page, K or V, head): 4 codes a lane, so that a store is 1 KB of whole row pieces.
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

constexpr int SEL_T = 1024, SEL_W = SEL_T / 64;

// One workgroup per KV head finds the keep - sinks - recent largest accounts of the middle positions and lists what is
// kept in position order. The threshold (the least kept key) by radix selection over 11, 11 and 10 bits with LDS
// histograms; of the keys equal to it the first positions are kept. Wave w owns a contiguous range of positions, 64 in
// a row at a time, so that the places come from ballots and one scan over the waves.
__global__ __launch_bounds__(SEL_T) void evict_select_kernel(B8Evict p) {
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t wsum[SEL_W];
  __shared__ uint32_t found[2];  // digit, keys above it
  __shared__ uint32_t wgt[SEL_W], weq[SEL_W];
  const int h = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* mass = p.mass + (size_t)h * p.mass_stride + p.sinks;
  int32_t* kept = p.kept + (size_t)h * p.keep;
  const int N = p.T - p.sinks - p.recent, k = p.keep - p.sinks - p.recent;
  for (int i = tid; i < p.sinks; i += SEL_T) kept[i] = i;
  for (int i = tid; i < p.recent; i += SEL_T) kept[p.keep - p.recent + i] = p.T - p.recent + i;
  if (k <= 0) return;
  uint32_t prefix = 0, mask = 0;  // the threshold's bits found so far
  uint32_t need = (uint32_t)k;    // how many of the keys with that prefix are kept
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < bins; i += SEL_T) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < N; i += SEL_T) {
      const uint32_t u = mass_key(ldg(mass + i));
      if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    // thread t owns bins 2 t, 2 t + 1 counted from the top; an inclusive scan over the threads
    const int b1 = bins - 1 - 2 * tid, b0 = b1 - 1;
    const uint32_t n1 = b1 >= 0 ? hist[b1] : 0u, n0 = b0 >= 0 ? hist[b0] : 0u;
    uint32_t sum = n1 + n0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 63) wsum[wave] = sum;
    __syncthreads();
    uint32_t before = sum - n1 - n0;
    for (int w = 0; w < wave; ++w) before += wsum[w];
    if (before < need && need <= before + n1) {
      found[0] = (uint32_t)b1;
      found[1] = before;
    } else if (before + n1 < need && need <= before + n1 + n0) {
      found[0] = (uint32_t)b0;
      found[1] = before + n1;
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    need -= found[1];
  }
  // every key above the threshold, and the first `need` of those equal to it
  const int per = ((N + SEL_W - 1) / SEL_W + 63) / 64 * 64;
  const int lo = min(N, wave * per), hi = min(N, lo + per);
  uint32_t gt = 0, eq = 0;
  for (int i = lo + lane; i - lane < hi; i += 64) {
    const uint32_t u = i < hi ? mass_key(ldg(mass + i)) : 0u;
    gt += __popcll(__ballot(i < hi && u > prefix));
    eq += __popcll(__ballot(i < hi && u == prefix));
  }
  if (lane == 0) {
    wgt[wave] = gt;
    weq[wave] = eq;
  }
  __syncthreads();
  uint32_t at = 0, used = 0;
  for (int w = 0; w < wave; ++w) {
    const uint32_t e = min(weq[w], need - used);
    at += wgt[w] + e;
    used += e;
  }
  const uint64_t below = (1ull << lane) - 1;
  for (int i = lo + lane; i - lane < hi; i += 64) {
    const uint32_t u = i < hi ? mass_key(ldg(mass + i)) : 0u;
    const uint64_t be = __ballot(i < hi && u == prefix);
    const bool take = i < hi && (u > prefix || (u == prefix && used + __popcll(be & below) < need));
    const uint64_t bt = __ballot(take);
    if (take) kept[p.sinks + at + __popcll(bt & below)] = p.sinks + i;
    at += __popcll(bt);
    used = min(need, used + (uint32_t)__popcll(be));
  }
}

// One wave per (destination page, K or V, head): 32 kept rows gathered 16 bytes a lane into one block. Its scale is the
// largest of its rows' scales: rows that had it keep their codes, the others are re-coded to it.
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
int b8_evict_launch(const B8Evict& p, int D, bool fp8, hipStream_t s) {
  hipLaunchKernelGGL(evict_select_kernel, dim3(p.src.KVH), dim3(SEL_T), 0, s, p);
  if (const int rc = (int)hipGetLastError()) return rc;
  const int nw = (p.keep + PAGE - 1) / PAGE * 2 * p.src.KVH;
  return by_kind(D, fp8, [&](auto d, auto f) {
    hipLaunchKernelGGL((evict_move_kernel<decltype(d)::value, decltype(f)::value>), dim3((nw + WPB - 1) / WPB), dim3(64 * WPB), 0,
                       s, p, nw);
  });
}

}  // namespace dspark
