// Rotary positions of a batch's q and k rows, and its K and V rows into the fp16 pages by slot.
//
// A pair (x_i, x_j) turns by the angle p f: y_i = s (x_i cos - x_j sin), y_j = s (x_j cos + x_i sin). The angle is taken in
// turns, p (f / 2 pi) in 64 bits, less its nearest whole number (exact), then as a quarter turn and a rest within an eighth,
// whose sine and cosine are their series in 64 bits (the first term left out is under 2e-14): fp32 loses the angle itself
// from some ten thousand positions on. 64-bit multiply-adds run at the rate of 32-bit ones here, and an angle serves every
// head of its token: a workgroup computes its tokens' sines and cosines once, into LDS.
//
// Bound by memory: each value is read and written once, in pieces of 16 bytes where sizes and addresses allow (VEC), else value
// by value. A unit of work is a piece (half layout: the piece and its partner rot / 2 further) or a piece of what is not turned.
// Measured: 4099 tokens of 16 + 4 heads of 128 in fp32, 84 MB, 13.5 us (6.2 TB/s: partly from the 256 MB cache); 8192 tokens of 16 + 4
// heads of 128 in fp16 with K and V into pages, 101 MB, 22 us (26 from memory alone, 3.9 TB/s); 8 tokens 3.9 us.
//
// Into the pages go workgroups of a KV head and 32 tokens, side by side in the lanes: tokens of a run lie in consecutive slots,
// which K's operand order keeps 16 bytes apart and V's transposed rows 2, so that a wave's store covers whole lines (a token's row
// after another's 2-byte stores 64 bytes apart: 63 us instead of 22). V's rows turn in LDS.
#include "batch.h"

#include <algorithm>

#include "dspark.h"

namespace dspark {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_TOKENS = 8;  // of a workgroup at most
constexpr int ROPE_RUN = 32;    // of a workgroup that fills pages

__device__ __forceinline__ float rope_to_f32(float x) { return x; }
__device__ __forceinline__ float rope_to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float rope_to_f32(__bf16 x) { return (float)x; }

// (cos, sin) of `turns` turns times scale.
__device__ __forceinline__ f32x2 rope_cos_sin(double turns, double scale, bool inverse) {
  const double r = turns - rint(turns);
  const double quarter = rint(4 * r);
  const double a = (r - 0.25 * quarter) * 6.283185307179586476925, b = a * a;  // |a| <= pi / 4
  const double s = a * fma(b, fma(b, fma(b, fma(b, fma(b, fma(b, 1.0 / 6227020800.0, -1.0 / 39916800.0), 1.0 / 362880.0), -1.0 / 5040.0), 1.0 / 120.0), -1.0 / 6.0), 1.0);
  const double c = fma(b, fma(b, fma(b, fma(b, fma(b, fma(b, fma(b, -1.0 / 87178291200.0, 1.0 / 479001600.0), -1.0 / 3628800.0), 1.0 / 40320.0), -1.0 / 720.0), 1.0 / 24.0), -0.5), 1.0);
  const int q = (int)quarter & 3;  // (-2 .. 2, or of a NaN anything: the values are NaN)
  double cs = q & 1 ? s : c, sn = q & 1 ? c : s;
  if (q == 1 || q == 2) cs = -cs;
  if (q >= 2) sn = -sn;
  return f32x2{(float)(cs * scale), (float)((inverse ? -sn : sn) * scale)};
}

template <typename T, int VEC>
struct RopePiece {
  T x[VEC];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC * sizeof(T) == 16) {
      const u32x4 u = ldg(reinterpret_cast<const u32x4*>(p));
      __builtin_memcpy(x, &u, 16);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VEC * sizeof(T) == 16) {
      u32x4 u;
      __builtin_memcpy(&u, x, 16);
      *reinterpret_cast<u32x4*>(p) = u;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) p[i] = x[i];
    }
  }
};

// The sines and cosines of tokens t0 .. t0 + nt - 1: cs[t][rot / 2], tokens `pitch` apart.
__device__ __forceinline__ void rope_angles(const RopeBatch& p, f32x2* cs, int pitch, int t0, int nt) {
  const int P = p.rot / 2;
  for (int e = threadIdx.x; e < nt * P; e += ROPE_THREADS) {
    const int t = e / P, i = e - t * P;
    cs[t * pitch + i] = rope_cos_sin((double)ldg(p.pos + t0 + t) * (ldg(p.freq + i) * 0.15915494309189533577), p.scale, p.inverse != 0);
  }
}

// Unit u of a head's row: loaded, then turned by its token's c and stored to dst + at(d). VEC: values of a piece, 16 bytes' worth or
// (sizes or addresses off 16 bytes) 1, interleaved pairs 2.
template <typename T, int VEC, bool IL>
struct RopeUnit {
  RopePiece<T, VEC> a, b;  // (b: the half layout's partner)
  int d;
  bool turns, stays;
  __device__ __forceinline__ void load(const RopeBatch& p, int u, const T* src, bool in_place) {
    const int P = p.rot / 2, turning = IL ? p.rot / VEC : P / VEC;  // units of a head: what turns first, then the rest
    turns = u < turning;
    d = turns ? u * VEC : p.rot + (u - turning) * VEC;
    stays = !turns && in_place;
    if (stays) return;
    a.load(src + d);
    if (!IL && turns) b.load(src + P + d);
  }
  template <typename At>
  __device__ __forceinline__ void store(const RopeBatch& p, const f32x2* c, T* dst, At at) {
    const int P = p.rot / 2;
    if (stays) return;
    if (!turns) {
      a.store(dst + at(d));
    } else if constexpr (IL) {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {
        const f32x2 w = c[d / 2 + i / 2];
        const float xi = rope_to_f32(a.x[i]), xj = rope_to_f32(a.x[i + 1]);
        a.x[i] = (T)(xi * w[0] - xj * w[1]);
        a.x[i + 1] = (T)(xj * w[0] + xi * w[1]);
      }
      a.store(dst + at(d));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const f32x2 w = c[d + i];
        const float xi = rope_to_f32(a.x[i]), xj = rope_to_f32(b.x[i]);
        a.x[i] = (T)(xi * w[0] - xj * w[1]);
        b.x[i] = (T)(xj * w[0] + xi * w[1]);
      }
      a.store(dst + at(d));
      b.store(dst + at(P + d));
    }
  }
};

// K and V of KV head h, tokens t0 .. t0 + nt - 1 (nt <= ROPE_RUN), into the pages.
template <int VEC, bool IL>
__device__ __forceinline__ void rope_pages(const RopeBatch& p, f32x2* cs, int h, int t0, int nt) {
  // (lanes are tokens: angles of two words an odd number of them apart, V's rows an odd number of words)
  const int angles = p.rot / 2 | 1, per = p.D / 8, pitch = p.D + 2;
  _Float16* turn = reinterpret_cast<_Float16*>(cs + ROPE_RUN * angles);
  // K's first pieces are on their way while V's rows and the angles are laid down
  const int tk = threadIdx.x % ROPE_RUN, u0 = threadIdx.x / ROPE_RUN;
  const _Float16* k = static_cast<const _Float16*>(p.k.x) + (size_t)(t0 + min(tk, nt - 1)) * p.k.x_stride + (size_t)h * p.D;
  const int64_t slot = ldg(p.slots + t0 + min(tk, nt - 1));
  RopeUnit<_Float16, VEC, IL> now, next;
  if (u0 < p.uph) now.load(p, u0, k, false);
  for (int e = threadIdx.x; e < nt * per; e += ROPE_THREADS) {
    const int t = e / per, d = (e - t * per) * 8;
    const _Float16* src = static_cast<const _Float16*>(p.v.x) + (size_t)(t0 + t) * p.v.x_stride + (size_t)h * p.D + d;
    uint32_t x[4];
    if (p.v_wide) {
      const u32x4 u = ldg(reinterpret_cast<const u32x4*>(src));
      __builtin_memcpy(x, &u, 16);
    } else {
      __builtin_memcpy(x, src, 16);
    }
    uint32_t* to = reinterpret_cast<uint32_t*>(turn + t * pitch + d);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = x[i];
  }
  rope_angles(p, cs, angles, t0, nt);
  __syncthreads();
  if (tk >= nt || slot < 0 || slot >= p.n_slots) return;
  const size_t block = (size_t)((slot / PAGE) * p.KVH + h) * (PAGE * p.D);
  const int at_slot = (int)(slot % PAGE);
  // (a piece of up to 8 values from a multiple of its size lies together in K's page)
  for (int u = u0; u < p.uph; u += ROPE_THREADS / ROPE_RUN) {
    if (u + ROPE_THREADS / ROPE_RUN < p.uph) next.load(p, u + ROPE_THREADS / ROPE_RUN, k, false);
    now.store(p, cs + tk * angles, p.kp + block, [&](int d) { return k_page_elem(at_slot, d, p.D); });
    now = next;
  }
  for (int d = u0; d < p.D; d += ROPE_THREADS / ROPE_RUN) p.vp[block + v_page_elem(at_slot, d)] = turn[tk * pitch + d];
}

template <typename T, int VEC, bool IL>
__global__ __launch_bounds__(ROPE_THREADS) void rope_kernel(RopeBatch p) {
  extern __shared__ f32x2 cs[];  // [tokens][rot / 2]
  int wg = (int)blockIdx.x;
  if constexpr (__is_same(T, _Float16)) {
    if (wg < p.fill) {
      const int run = wg / p.KVH, t0 = run * ROPE_RUN;
      rope_pages<VEC, IL>(p, cs, wg - run * p.KVH, t0, min(ROPE_RUN, p.n - t0));
      return;
    }
    wg -= p.fill;
  }
  const int t0 = wg * p.tok, nt = min(p.tok, p.n - t0);
  // a unit's loads are on their way while the angles, then the unit before are worked on (in place too: no unit reads what another writes)
  struct Place {
    const T* src;
    T* dst;
    int u, tl;
  };
  auto place = [&](int e) {
    const int tl = p.tok == 1 ? 0 : div_by(e, p.upt_div), r = e - tl * p.upt;
    int h = div_by(r, p.uph_div);
    const int u = r - h * p.uph;
    const bool in_q = h < p.q.heads;
    const RopeTensor& x = in_q ? p.q : p.k;
    if (!in_q) h -= p.q.heads;
    const size_t t = t0 + tl;
    return Place{static_cast<const T*>(x.x) + t * x.x_stride + (size_t)h * p.D, static_cast<T*>(x.y) + t * x.y_stride + (size_t)h * p.D, u, tl};
  };
  const int units = nt * p.upt;
  RopeUnit<T, VEC, IL> now, next;
  Place here = {}, there = {};
  if ((int)threadIdx.x < units) {
    here = place(threadIdx.x);
    now.load(p, here.u, here.src, here.src == here.dst);
  }
  rope_angles(p, cs, p.rot / 2, t0, nt);
  __syncthreads();
  for (int e = threadIdx.x; e < units; e += ROPE_THREADS) {
    if (e + ROPE_THREADS < units) {
      there = place(e + ROPE_THREADS);
      next.load(p, there.u, there.src, there.src == there.dst);
    }
    now.store(p, cs + here.tl * (p.rot / 2), here.dst, [](int d) { return d; });
    here = there;
    now = next;
  }
}

int rope_batch_launch(RopeBatch& p, int type, bool interleaved, hipStream_t s) {
  const int size = type == DSPARK_F32 ? 4 : 2, vec16 = 16 / size;
  // whole 16-byte pieces everywhere: the head and its turned part (half layout: half of it) in pieces, rows and heads on
  // 16-byte boundaries (D a multiple of a piece keeps every head on one)
  bool wide = p.D % vec16 == 0 && p.rot % vec16 == 0 && (interleaved || p.rot / 2 % vec16 == 0);
  for (const RopeTensor* x : {&p.q, &p.k}) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(x->x) | reinterpret_cast<uintptr_t>(x->y) |
                           (uintptr_t)(x->x_stride * size) | (uintptr_t)(x->y_stride * size);
    if (x->heads && bits & 15) wide = false;
  }
  const int vec = wide ? vec16 : interleaved ? 2 : 1;
  p.uph = interleaved ? p.D / vec : p.rot / 2 / vec + (p.D - p.rot) / vec;
  p.upt = (p.q.heads + (p.kp ? 0 : p.k.heads)) * p.uph;
  p.uph_div = div_magic(p.uph);
  p.upt_div = div_magic(max(p.upt, 1));
  // tokens of a workgroup: several where that leaves over 4 workgroups a CU, whose one round of angles then serves more work, and where
  // the division by upt is exact (a token alone may have more units than that)
  p.tok = 1;
  while (p.tok < ROPE_TOKENS && (p.n + 2 * p.tok - 1) / (2 * p.tok) >= 1024 && (int64_t)2 * p.tok * p.upt * p.upt < (int64_t)1 << 32) p.tok *= 2;
  p.fill = p.kp ? (p.n + ROPE_RUN - 1) / ROPE_RUN * p.KVH : 0;
  p.v_wide = !((reinterpret_cast<uintptr_t>(p.v.x) | (uintptr_t)(p.v.x_stride * 2)) & 15);
  const dim3 grid((p.upt ? (p.n + p.tok - 1) / p.tok : 0) + p.fill), block(ROPE_THREADS);
  size_t lds = (size_t)p.tok * (p.rot / 2) * sizeof(f32x2);
  if (p.fill) lds = std::max(lds, (size_t)ROPE_RUN * (p.rot / 2 + 1) * sizeof(f32x2) + (size_t)ROPE_RUN * (p.D + 2) * 2);
#define ROPE_GO(T, V, IL) hipLaunchKernelGGL((rope_kernel<T, V, IL>), grid, block, lds, s, p)
#define ROPE_TYPE(T, V16)                    \
  if (wide && interleaved) ROPE_GO(T, V16, true);  \
  else if (wide) ROPE_GO(T, V16, false);     \
  else if (interleaved) ROPE_GO(T, 2, true); \
  else ROPE_GO(T, 1, false)
  if (type == DSPARK_F32) {
    ROPE_TYPE(float, 4);
  } else if (type == DSPARK_BF16) {
    ROPE_TYPE(__bf16, 8);
  } else {
    ROPE_TYPE(_Float16, 8);
  }
#undef ROPE_TYPE
#undef ROPE_GO
  return (int)hipGetLastError();
}

}  // namespace dspark
