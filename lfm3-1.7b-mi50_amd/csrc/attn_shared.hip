// Verify attention of a batch of sequences behind a shared prefix (fp16 pages): the prefix's keys are read once for the rows of
// all sequences, each sequence's own keys for its rows.
//
// o = sum_j P_j v_j / l with P_j = 2^(c q.k_j - m), c = log2(e) / sqrt(D), l = sum_j P_j and m the row's running reference (it
// moves only when a score passes it by more than TAU, so P <= 2^TAU and a page mostly needs no rescale). It is set BASE below the
// largest score: fp16 then holds weights down to 2^-31 of the largest, and a long tail of keys far below one of them keeps its
// share (with the reference at the largest itself a weight of 2^-26 is nothing, 2^17 such keys 2^-9 of the whole). Tiles are those
// of the page format: S^T[keys][rows] = K Q^T, a lane holds one row's scores of eight keys, which in this order are its operand of
// O^T += V^T P^T; row sums are added up before that. Scores, sums and outputs are fp32, P is rounded to fp16 once (V's
// products take fp16 operands; sums of the rounded P by a product with ones cost lse its digits past 2^-11, and a long call 229 us
// instead of 224); q is taken as it is, the scale in the exponent's multiply-add (scaled in fp16 it would be rounded).
//
// Work: one launch over two kinds of workgroups. Prefix: a KV head, a block of its rows (all sequences' side by side: 16 to 128)
// and a range of prefix pages. Own: a KV head, a sequence, a block of its rows and a range of its pages. Either streams pages
// through a two-slot ring in LDS by direct-to-LDS loads, one slot ahead; its waves are row waves (every wave all pages of a slot)
// or, with few rows, page waves (each a page of the slot), whose sums meet in LDS. Partial sums go to the workspace, a second
// launch adds a row's in split order: no atomics, the same bits every call.
//
// What bounds it. Few rows: the chain of launch, table, first pages, sums and second launch (4 rows of 1001 + 37 keys, 4 x 128: 7.1 + 4.1
// us). A long prefix of 128 rows (8 x 64, 32768 keys and 32 sequences' own): 82 MB fetched in 26 us, 3.2 TB/s, ~4 of them before the
// first page is there. Many rows: issue; 640 rows of each head x 131072 keys of 8 x 64 take 212-235 us, 740-810 TFLOP/s. A page of
// 32 rows costs a wave some 110 vector instructions beside 16 products of matrix instructions (16 exponentials, multiply-adds,
// additions, 14 maxima, 16 roundings, addresses and bookkeeping), which follow each other in its program and hardly run side by side:
// matrix cores 36 %, vector units 68 % of the time at a clock of 1.7-2.1 GHz. That is the schedule's limit, neither unit's own.
// With a window the prefix is split as without one and the workgroups before it find nothing to do: 32 rows of 131072 keys, 4096 of
// them seen, take 77 us, all of them 84, a prefix of 4096 keys 20. Measured and not kept, of many rows: a third or fourth slot in the ring
// (229 -> 225 us, shorter calls slower), two pages' softmax at once (237, spills at D = 128), four row blocks a wave, wave priorities,
// one workgroup of 64 rows instead of two of 32 for a sequence's own keys (27.7 -> 27.7 at 36 rows a sequence).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "batch.h"
#include "dspark.h"

namespace dspark {

constexpr float SA_TAU = 15.f, SA_BASE = 7.f;  // (2^15 < 65504)
constexpr int SA_THREADS = 256;

// The row-wave form's ring: two slots of two pages. At D = 64 that leaves room for four workgroups a CU, at 128 for two, as many as the
// registers do.
constexpr int SA_NP = 2;
constexpr int sa_slot(int D) { return SA_NP * PAGE * D * 4; }
constexpr int sa_waves(int D) { return D == 64 ? 4 : 2; }  // of a SIMD
// The two slots are two LDS objects: the compiler then knows that loads in flight into one do not touch what is read from the other
// (in one array it waits for all loads before the first read of a step). The page-wave form keeps K in the first, V in the second.
static_assert(sa_slot(128) == 4 * PAGE * 128 * 2 && sa_slot(64) == 2 * 32 * 64 * 4, "four page waves' K; two waves' sums of 32 rows");

// Which keys the lane's rows see: lo <= key <= hi, and the pages on which every row of the wave sees all keys.
template <int QB>
struct SaMask {
  int lo[QB], hi[QB];
  int full_lo, full_hi;  // wave-uniform
};

template <int D, int QB>
struct SaState {
  f32x4 o[QB][D / 16];
  float l[QB];    // of the lane's keys: a row's four lanes add theirs at the end (sa_sum)
  float m[QB];    // reference in log2 units, 0 before the row's first key
  float thr[QB];  // an exponent above this moves it: TAU, -inf before the first key
};

// Scores of one page for the wave's row blocks, from K at `kt` in LDS (operand order).
template <int D, int QB>
__device__ __forceinline__ void sa_scores(const char* kt, const half8 (&q)[QB][D / 32], f32x4 (&s)[QB][2], int lane) {
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) s[qb][0] = s[qb][1] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks) {
    const half8 k0 = *reinterpret_cast<const half8*>(kt + ks * 1024 + lane * 16);
    const half8 k1 = *reinterpret_cast<const half8*>(kt + (D / 32 + ks) * 1024 + lane * 16);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      s[qb][0] = mfma16x16x32(k0, q[qb][ks], s[qb][0]);
      s[qb][1] = mfma16x16x32(k1, q[qb][ks], s[qb][1]);
    }
  }
}

// Is a page one on which some row of the wave does not see some key?
template <int QB>
__device__ __forceinline__ bool sa_edge(const SaMask<QB>& mk, int key0) {
  return key0 < mk.full_lo || key0 + PAGE - 1 > mk.full_hi;  // (scalars)
}

__device__ __forceinline__ float sa_top(const f32x4 (&x)[2]) {
  return fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
}
// Masks, the references' moves, and P.
template <int D, int QB>
__device__ __forceinline__ void sa_softmax(f32x4 (&s)[QB][2], int key0, const SaMask<QB>& mk, float c, SaState<D, QB>& st,
                                           half8 (&pp)[QB], int lane) {
  const int g = lane >> 4;
  if (sa_edge<QB>(mk, key0)) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int a = key0 + 8 * g + i, b = a + 4;
        s[qb][0][i] = a >= mk.lo[qb] && a <= mk.hi[qb] ? s[qb][0][i] : -INFINITY;
        s[qb][1][i] = b >= mk.lo[qb] && b <= mk.hi[qb] ? s[qb][1][i] : -INFINITY;
      }
  }
  // exponents against the reference as it is; it moves only where one passes TAU (or at a row's first key, from 0)
  bool need = false;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[qb][0][i] = fmaf(s[qb][0][i], c, -st.m[qb]);
      s[qb][1][i] = fmaf(s[qb][1][i], c, -st.m[qb]);
    }
    need = need | (sa_top(s[qb]) > st.thr[qb]);
  }
  if (__builtin_amdgcn_ballot_w64(need) != 0) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float rm = sa_top(s[qb]);
      rm = fmaxf(rm, __shfl_xor(rm, 16));  // the row's four lanes
      rm = fmaxf(rm, __shfl_xor(rm, 32));
      if (rm > st.thr[qb]) {
        const float m = st.m[qb] + (rm - SA_BASE), move = m - st.m[qb];
        const float alpha = st.thr[qb] == SA_TAU ? fast_exp2(-move) : 0.f;
#pragma unroll
        for (int cc = 0; cc < D / 16; ++cc) st.o[qb][cc] *= alpha;
        st.l[qb] *= alpha;
        st.m[qb] = m;
        st.thr[qb] = SA_TAU;
        s[qb][0] -= move;
        s[qb][1] -= move;
      }
    }
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e0 = fast_exp2(s[qb][0][i]), e1 = fast_exp2(s[qb][1][i]);
      st.l[qb] += e0 + e1;
      pp[qb][i] = (_Float16)e0;
      pp[qb][4 + i] = (_Float16)e1;
    }
}
__device__ __forceinline__ float sa_sum(float l) {
  l += __shfl_xor(l, 16);
  return l + __shfl_xor(l, 32);
}

// V's operands of a page in LDS.
template <int D>
__device__ __forceinline__ void sa_v(const char* vt, u32x4 (&v)[D / 16], int lane) {
#pragma unroll
  for (int cc = 0; cc < D / 16; ++cc) v[cc] = *reinterpret_cast<const u32x4*>(vt + cc * 1024 + lane * 16);
}
// O^T += V^T P^T. On an edge page, where some row does not see some key, a value of V that is not finite would spoil
// every row (0 x inf): it counts as zero in the product, and afterwards the rows that do see one get an infinity: a product of
// where it stands with which keys they see, times 2^254.
template <int D, int QB>
__device__ __forceinline__ void sa_values(const char* vt, u32x4 (&v)[D / 16], int key0, const half8 (&pp)[QB], const SaMask<QB>& mk,
                                          SaState<D, QB>& st, int lane) {
  const bool edge = sa_edge<QB>(mk, key0);
  if (edge) {
#pragma unroll
    for (int cc = 0; cc < D / 16; ++cc)
#pragma unroll
      for (int i = 0; i < 4; ++i)  // two halves a word
        v[cc][i] &= ((v[cc][i] & 0x7c00u) == 0x7c00u ? 0u : 0xffffu) | ((v[cc][i] & 0x7c000000u) == 0x7c000000u ? 0u : 0xffff0000u);
  }
#pragma unroll
  for (int cc = 0; cc < D / 16; ++cc)
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) st.o[qb][cc] = mfma16x16x32(as_half8(v[cc]), pp[qb], st.o[qb][cc]);
  if (edge) {
    asm volatile("" ::: "memory");  // (V is read again: nothing of this is worked out for the pages that do not come here)
#pragma unroll
    for (int cc = 0; cc < D / 16; ++cc) {
      u32x4 bad = *reinterpret_cast<const u32x4*>(vt + cc * 1024 + lane * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i)  // 0x3c00 is one
        bad[i] = ((bad[i] & 0x7c00u) == 0x7c00u ? 0x3c00u : 0u) | ((bad[i] & 0x7c000000u) == 0x7c000000u ? 0x3c000000u : 0u);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        half8 sees;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = key0 + 8 * (lane >> 4) + i;
          sees[i] = key >= mk.lo[qb] && key <= mk.hi[qb] ? (_Float16)1 : (_Float16)0;
        }
        const f32x4 n = mfma16x16x32(as_half8(bad), sees, f32x4{0, 0, 0, 0});
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[qb][cc][i] = fmaf(n[i] * 0x1p127f, 0x1p127f, st.o[qb][cc][i]);
      }
      asm volatile("" ::: "memory");  // (one operand at a time: these pages are few, registers are too)
    }
  }
}

// Row and page bookkeeping of a workgroup: pages [pb, pe) of a table (nullptr: the identity) for rows row0 .. of KV head h; rows
// from `rows` on are not there: they read as the last and are not stored.
struct SaWork {
  const int32_t* tab;
  int h, row0, rows, pb, pe, split;
};

// The table's entry of page i, unlooked-at (the load may be in flight), and the page it stands for: -1 absent, or past the range.
__device__ __forceinline__ int sa_entry(const SaWork& w, int i) { return w.tab ? ldc(w.tab + min(i, w.pe - 1)) : i; }
__device__ __forceinline__ int sa_physical(const SharedAttn& p, const SaWork& w, int i, int entry) {
  return i < w.pe && (uint32_t)entry < (uint32_t)p.pages ? entry : -1;
}

// K or V of a page into LDS, 1 KB a load. An absent page (-1) is fetched as page 0, which exists, and not used: every page costs
// the same loads, so that they can be counted. V's operand c of lane (n, g) is row 16 c + n, keys 8 g .. + 8: fetched so that it
// lies at the lane's 16 bytes of the c-th KB, where all 64 lanes read without bank conflicts.
template <int D>
__device__ __forceinline__ void sa_fetch(const SharedAttn& p, bool isv, int pg, int h, char* dst, int lane) {
  const size_t blk = ((size_t)max(pg, 0) * p.KVH + h) * (PAGE * D);
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc((void*)((isv ? p.vp : p.kp) + blk), (short)0, PAGE * D * 2, 0x00020000);
  const uint32_t off = isv ? (lane & 15) * 64 + (lane >> 4) * 16 : lane * 16;
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(dst + i * 1024), 16, off + i * 1024, 0, 0, 0);
}

// The wave's rows from wrow on: q operands, masks (row_mask(row) gives the least and the largest key it sees), empty sums.
template <int D, int QB, typename Mask>
__device__ __forceinline__ void sa_begin(const SharedAttn& p, const SaWork& w, int wrow, half8 (&q)[QB][D / 32], SaMask<QB>& mk,
                                         SaState<D, QB>& st, int lane, Mask row_mask) {
  const int n = lane & 15, g = lane >> 4;
  mk.full_lo = 0;
  mk.full_hi = 0x7fffffff;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int row = min(wrow + 16 * qb + n, w.rows - 1);
    const int t = div_by(row, p.g_div), qh = w.h * p.G + row - t * p.G;
    const _Float16* src = p.q + (size_t)t * p.q_stride + (size_t)qh * D + 8 * g;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) q[qb][s] = as_half8(ldg(reinterpret_cast<const u32x4*>(src + 32 * s)));
    row_mask(row, mk.lo[qb], mk.hi[qb]);
    mk.full_lo = max(mk.full_lo, (int)wave_max_u32((uint32_t)max(mk.lo[qb], 0)));
    mk.full_hi = min(mk.full_hi, 0x7fffffff - (int)wave_max_u32(0x7fffffffu - (uint32_t)max(mk.hi[qb], 0)));
    if (__builtin_amdgcn_ballot_w64(mk.hi[qb] < 0)) mk.full_hi = -1;
    mk.full_lo = __builtin_amdgcn_readfirstlane(mk.full_lo);
    mk.full_hi = __builtin_amdgcn_readfirstlane(mk.full_hi);
#pragma unroll
    for (int cc = 0; cc < D / 16; ++cc) st.o[qb][cc] = f32x4{0, 0, 0, 0};
    st.l[qb] = 0.f;
    st.m[qb] = 0.f;
    st.thr[qb] = -INFINITY;
  }
}

// Many rows: four waves of 16 QB rows each take every page.
template <int D, int QB, typename Mask>
__device__ __forceinline__ void sa_run_rows(const SharedAttn& p, char (&lds0)[sa_slot(D)], char (&lds1)[sa_slot(D)], const SaWork& w, Mask row_mask) {
  constexpr int PAGE_BYTES = PAGE * D * 4;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // a wave's share of a slot: K (even waves) or V of page wave / 2. Table entries are read a step before their pages are fetched.
  const int mine = wave >> 1;
  const bool isv = wave & 1;
  int here[SA_NP], next[SA_NP];
  auto entries = [&](int first, int (&e)[SA_NP]) {
#pragma unroll
    for (int i = 0; i < SA_NP; ++i) e[i] = sa_entry(w, first + i);
  };
  auto issue = [&](int first, const int (&e)[SA_NP], char* slot) {  // (past the range: page 0, into a slot nobody reads)
    sa_fetch<D>(p, isv, sa_physical(p, w, first + mine, mine ? e[1] : e[0]), w.h, slot + mine * PAGE_BYTES + (isv ? PAGE * D * 2 : 0), lane);
  };
  if (w.pb < w.pe) {
    entries(w.pb, here);
    entries(w.pb + SA_NP, next);
    issue(w.pb, here, lds0);
  }
  const int wrow = w.row0 + wave * 16 * QB;
  half8 q[QB][D / 32];
  SaMask<QB> mk;
  SaState<D, QB> st;
  sa_begin<D, QB>(p, w, wrow, q, mk, st, lane, row_mask);
  const bool rows = wrow < w.rows;  // (a wave without any fetches its share alone)
  auto step = [&](int first, const char* cur, char* nxt) {
    ring_barrier<0>();  // this slot is in LDS, every wave is done with the other one
    issue(first + SA_NP, next, nxt);
    int after[SA_NP];
    entries(first + 2 * SA_NP, after);
    if (rows) {
#pragma unroll
      for (int i = 0; i < SA_NP; ++i) {
        if (sa_physical(p, w, first + i, here[i]) < 0) continue;
        const char* kt = cur + i * PAGE_BYTES;
        f32x4 s[QB][2];
        half8 pp[QB];
        u32x4 v[D / 16];
        sa_scores<D, QB>(kt, q, s, lane);
        if (D == 128) sa_v<D>(kt + PAGE * D * 2, v, lane);  // (early where the registers allow it)
        sa_softmax<D, QB>(s, (first + i) * PAGE, mk, p.c, st, pp, lane);
        if (D == 64) sa_v<D>(kt + PAGE * D * 2, v, lane);
        sa_values<D, QB>(kt + PAGE * D * 2, v, (first + i) * PAGE, pp, mk, st, lane);
      }
    }
#pragma unroll
    for (int i = 0; i < SA_NP; ++i) {
      here[i] = next[i];
      next[i] = after[i];
    }
  };
  for (int first = w.pb; first < w.pe; first += 2 * SA_NP) {
    step(first, lds0, lds1);
    if (first + SA_NP >= w.pe) break;
    step(first + SA_NP, lds1, lds0);
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // (the last step's fetch: LDS is not given up before it has arrived)
  const size_t out0 = (size_t)w.h * p.T * p.G;
  const int S = p.Sp + p.So;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int row = wrow + 16 * qb + n;
    const size_t at = (out0 + row) * S + w.split;
    const float l = sa_sum(st.l[qb]);
    if (row >= w.rows) continue;
    if (g == 0) p.part_ml[at] = f32x2{l != 0.f ? st.m[qb] : -INFINITY, l};
    if (l != 0.f) {
      f32x4* dst = reinterpret_cast<f32x4*>(p.part_o + at * D);
#pragma unroll
      for (int cc = 0; cc < D / 16; ++cc) dst[4 * cc + g] = st.o[qb][cc];
    }
  }
}

// Few rows: every wave has all 16 QB of them and a page of its own, wave, wave + 4, ... of the range. Nothing is shared, so there
// are no barriers: K's half of the wave's LDS page is fetched anew while the page's P and products are computed, V's half
// while the next page's scores are.
template <int D, int QB, typename Mask>
__device__ __forceinline__ void sa_run_pages(const SharedAttn& p, char (&lds0)[sa_slot(D)], char (&lds1)[sa_slot(D)], const SaWork& w, Mask row_mask) {
  constexpr int HALF = PAGE * D * 2, LOADS = D / 16;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char* kt = lds0 + wave * HALF;
  char* vt = lds1 + wave * HALF;
  int i = w.pb + wave, pg = -1;
  if (i < w.pe) {
    pg = sa_physical(p, w, i, sa_entry(w, i));
    sa_fetch<D>(p, false, pg, w.h, kt, lane);
    sa_fetch<D>(p, true, pg, w.h, vt, lane);
  }
  half8 q[QB][D / 32];
  SaMask<QB> mk;
  SaState<D, QB> st;
  sa_begin<D, QB>(p, w, w.row0, q, mk, st, lane, row_mask);
  auto loads_but = [](auto left) {  // all but the `left` youngest loads done (and every LDS read), nothing moved across
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(decltype(left)::value) & ~0x0F00);
    asm volatile("" ::: "memory");
  };
  using Zero = std::integral_constant<int, 0>;
  using Half = std::integral_constant<int, LOADS>;
  while (i < w.pe) {
    const int nxt = i + 4;
    const bool more = nxt < w.pe;
    const int entry = sa_entry(w, nxt);
    f32x4 s[QB][2];
    half8 pp[QB];
    int npg = -1;
    loads_but(Half{});
    sa_scores<D, QB>(kt, q, s, lane);
    if (more) {
      loads_but(std::integral_constant<int, 63>{});  // (the reads of K)
      npg = sa_physical(p, w, nxt, entry);
      sa_fetch<D>(p, false, npg, w.h, kt, lane);
    }
    if (pg >= 0) sa_softmax<D, QB>(s, i * PAGE, mk, p.c, st, pp, lane);
    if (more)
      loads_but(Half{});
    else
      loads_but(Zero{});
    if (pg >= 0) {
      u32x4 v[D / 16];
      sa_v<D>(vt, v, lane);
      sa_values<D, QB>(vt, v, i * PAGE, pp, mk, st, lane);
    }
    if (more) {
      loads_but(std::integral_constant<int, 63>{});
      sa_fetch<D>(p, true, npg, w.h, vt, lane);
    }
    i = nxt;
    pg = npg;
  }

  // the four waves' sums through LDS, values in 16-byte pieces at c ^ (row % 16) so that rows lie on different banks
  __shared__ float sm_m[4][16 * QB], sm_l[4][16 * QB];
  lds_barrier();
  auto sums = [&](int v) { return reinterpret_cast<f32x4*>(v < 2 ? lds0 : lds1) + (v & 1) * (16 * QB * D / 4); };  // of wave v
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = 16 * qb + n;
    const float l = sa_sum(st.l[qb]);
    if (g == 0) {
      sm_m[wave][r] = st.thr[qb] == SA_TAU ? st.m[qb] : -1e30f;  // (no key: a reference below all others)
      sm_l[wave][r] = l;
    }
#pragma unroll
    for (int cc = 0; cc < D / 16; ++cc) sums(wave)[r * (D / 4) + ((4 * cc + g) ^ n)] = st.o[qb][cc];
  }
  lds_barrier();
  const size_t out0 = (size_t)w.h * p.T * p.G;
  for (int e = threadIdx.x; e < 16 * QB * (D / 4); e += SA_THREADS) {
    const int r = e / (D / 4), c4 = e % (D / 4);
    if (w.row0 + r >= w.rows) continue;
    const float m = fmaxf(fmaxf(sm_m[0][r], sm_m[1][r]), fmaxf(sm_m[2][r], sm_m[3][r]));
    float l = 0.f;
    f32x4 o = {0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float f = fast_exp2(sm_m[v][r] - m);
      l += f * sm_l[v][r];
      o += sums(v)[r * (D / 4) + (c4 ^ (r & 15))] * f;
    }
    const size_t at = (out0 + w.row0 + r) * (p.Sp + p.So) + w.split;
    if (c4 == 0) p.part_ml[at] = f32x2{l != 0.f ? m : -INFINITY, l};
    if (l != 0.f) reinterpret_cast<f32x4*>(p.part_o + at * D)[c4] = o;
  }
}

// A sequence's rows and own keys, cut to what the arguments allow.
struct SaSeq {
  int t0, m, len;
};
__device__ __forceinline__ SaSeq sa_seq(const SharedAttn& p, int r) {
  SaSeq s;
  const int a = min(max(ldc(p.q_start + r), 0), p.T), b = min(max(ldc(p.q_start + r + 1), 0), p.T);
  s.t0 = a;
  s.m = max(b - a, 0);
  s.len = min(max(ldc(p.own_len + r), 0), p.own_pages * PAGE);
  return s;
}

// ROWS: prefix workgroups of four row waves, else of four page waves.
template <int D, int QB, bool ROWS, int QBO>
__global__ __launch_bounds__(SA_THREADS, sa_waves(D)) void shared_attn_kernel(SharedAttn p) {
  __shared__ __attribute__((aligned(16))) char lds0[sa_slot(D)], lds1[sa_slot(D)];
  constexpr int BLOCK = 16 * QB * (ROWS ? 4 : 1);
  auto go = [&](const SaWork& w, auto mask) {
    if constexpr (ROWS)
      sa_run_rows<D, QB>(p, lds0, lds1, w, mask);
    else
      sa_run_pages<D, QB>(p, lds0, lds1, w, mask);
  };
  const int prefix_groups = (p.KVH * p.Sp + 7) / 8 * 8 * p.RBp;
  int id = blockIdx.x;
  if (id < prefix_groups) {
    // Row blocks of one (head, split) read the same pages: ids 8 apart, so that they run on one XCD and share its L2
    const int within = id % (8 * p.RBp), unit = id / (8 * p.RBp) * 8 + within % 8, rb = within / 8;
    if (unit >= p.KVH * p.Sp) return;
    const int h = unit / p.Sp, split = unit % p.Sp;
    const int row0 = rb * BLOCK, rows = p.T * p.G;
    int pb = split * p.pps;
    const int pe = min(pb + p.pps, (p.prefix + PAGE - 1) / PAGE);
    if (p.window == 0) {
      go(SaWork{p.ptab, h, row0, rows, pb, pe, split}, [&](int, int& lo, int& hi) {
        lo = 0;
        hi = p.prefix - 1;
      });
    } else {
      // the least position any row of the block sees (a token in no sequence: no bound, its sums are not used)
      auto low = [&](int row) {
        const int t = div_by(row, p.g_div);
        int a = 0, b = p.R;  // the last sequence that begins at or before t
        while (b - a > 1) {
          const int mid = (a + b) / 2;
          if (ldg(p.q_start + mid) <= t) a = mid;
          else b = mid;
        }
        const int s0 = ldg(p.q_start + a), s1 = ldg(p.q_start + a + 1);
        if (t < s0 || t >= s1) return p.prefix;
        const int len = min(max(ldg(p.own_len + a), 0), p.own_pages * PAGE);
        const int pos = p.prefix + len - (min(s1, p.T) - t);
        return min(max(pos - p.window + 1, 0), p.prefix);
      };
      __shared__ int least;
      if (threadIdx.x == 0) least = p.prefix;
      __syncthreads();
      for (int r = threadIdx.x; r < BLOCK; r += SA_THREADS)
        if (row0 + r < rows) atomicMin(&least, low(row0 + r));
      __syncthreads();
      pb = max(pb, least / PAGE);
      go(SaWork{p.ptab, h, row0, rows, pb, pe, split}, [&](int row, int& lo, int& hi) {
        lo = low(row);
        hi = p.prefix - 1;
      });
    }
    return;
  }
  id -= prefix_groups;
  const int split = id % p.So;
  id /= p.So;
  const int h = id % p.KVH;
  id /= p.KVH;
  const int rb = id % p.RBo, r = id / p.RBo;
  const SaSeq s = sa_seq(p, r);
  const int m = min(s.m, p.max_tokens);
  if (rb * 16 * QBO >= m * p.G) return;
  const int pages = (s.len + PAGE - 1) / PAGE, per = (pages + p.So - 1) / p.So;
  int pb = split * per;
  const int pe = min(pb + per, pages);
  const int ctx = s.len - s.m;  // own keys before the call's first token
  if (p.window) pb = max(pb, min(max(ctx + div_by(rb * 16 * QBO, p.g_div) - p.window + 1, 0), max(ctx, 0)) / PAGE);
  const SaWork w = {p.own_tab + (size_t)r * p.own_stride, h, s.t0 * p.G + rb * 16 * QBO, (s.t0 + m) * p.G, pb, pe, p.Sp + split};
  sa_run_pages<D, QBO>(p, lds0, lds1, w,
                    [&](int row, int& lo, int& hi) {
                      const int pos = ctx + div_by(row, p.g_div) - s.t0;
                      lo = p.window ? min(max(pos - p.window + 1, 0), max(ctx, 0)) : 0;
                      hi = p.causal ? min(pos, s.len - 1) : s.len - 1;
                    });
}

// A row's partial sums: W waves a row, D / 4 lanes for the values by 256 W / D for the splits, whose sums meet in a fixed order (lanes,
// then waves). Everything a lane loads is asked for before the first of it is used, up to SA_ROUND splits at a time.
constexpr int SA_ROUND = 8;
template <int D, int W>
__global__ __launch_bounds__(SA_THREADS) void shared_merge_kernel(SharedAttn p) {
  constexpr int CH = D / 4, SL = 64 / CH * W;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = (int64_t)blockIdx.x * (4 / W) + wave / W;
  const int qh = (int)(unit % p.QH);
  const int64_t ri = unit / p.QH;
  const int i = (int)(ri % p.max_tokens), r = (int)(ri / p.max_tokens);
  if (r >= p.R) return;  // (W = 4: the whole workgroup)
  const SaSeq s = sa_seq(p, r);
  if (i >= s.m) return;
  const int t = s.t0 + i, h = div_by(qh, p.g_div), S = p.Sp + p.So;
  const size_t row = ((size_t)h * p.T + t) * p.G + (qh - h * p.G);
  const f32x2* ml = p.part_ml + row * S;
  const f32x4* po = reinterpret_cast<const f32x4*>(p.part_o + row * S * D);
  const int c4 = lane % CH, s0 = (wave % W) * (64 / CH) + lane / CH;
  f32x2 x[SA_ROUND];
  f32x4 v[SA_ROUND];
  auto load = [&](int k0) {
#pragma unroll
    for (int j = 0; j < SA_ROUND; ++j) {
      const int k = min(k0 + j * SL, S - 1);
      x[j] = ldg(ml + k);
      v[j] = ldg(po + (size_t)k * CH + c4);
    }
  };
  load(s0);
  float m = -INFINITY;
  for (int k = lane; k < S; k += 64) m = fmaxf(m, ldg(ml + k)[0]);
  m = wave_max(m);
  float l = 0.f;
  f32x4 o = {0, 0, 0, 0};
  for (int k0 = s0; k0 < S; k0 += SA_ROUND * SL) {
    if (k0 != s0) load(k0);
#pragma unroll
    for (int j = 0; j < SA_ROUND; ++j) {
      const bool in = k0 + j * SL < S && x[j][1] != 0.f;  // (a split that saw nothing left no values)
      const float f = in ? fast_exp2(x[j][0] - m) : 0.f;
      l += in ? f * x[j][1] : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += in ? f * v[j][e] : 0.f;
    }
  }
#pragma unroll
  for (int d = CH; d < 64; d *= 2) {
    l += __shfl_xor(l, d);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += __shfl_xor(o[j], d);
  }
  if constexpr (W > 1) {
    __shared__ f32x4 so[W][CH];
    __shared__ float sl[W];
    if (lane < CH) so[wave][lane] = o;
    if (lane == 0) sl[wave] = l;
    __syncthreads();
    if (wave) return;
    l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    o = (so[0][c4] + so[1][c4]) + (so[2][c4] + so[3][c4]);
  }
  if (lane >= CH) return;
  const size_t at = (size_t)t * p.QH + qh;
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : NAN;
  if (p.lse && c4 == 0) p.lse[at] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : l == 0.f ? -INFINITY : NAN;
  o *= inv;
  if (p.gate) o *= 1.f / (1.f + __expf(-ldg(p.gate + at)));
  if (p.out32) reinterpret_cast<f32x4*>(p.out32 + at * D)[c4] = o;
  if (p.out16) {
    half4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (_Float16)o[j];
    reinterpret_cast<half4*>(p.out16 + at * D)[c4] = y;
  }
}

// Shapes of a prefix workgroup: 16-row blocks of a wave, and whether its waves are row waves.
struct SaCfg {
  int qb;
  bool rows;
};
constexpr SaCfg SA_CFG[4] = {{1, false}, {2, false}, {1, true}, {2, true}};

void shared_plan(SharedAttn& p, int D, int splits, int cus) {
  const int64_t rows = (int64_t)p.T * p.G;
  // the least block that holds all rows, else blocks of 128
  p.cfg = rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3;
  const int per = 16 * SA_CFG[p.cfg].qb * (SA_CFG[p.cfg].rows ? 4 : 1), wp = SA_CFG[p.cfg].rows ? 1 : 4;
  p.RBp = (int)((rows + per - 1) / per);
  const int pages = (p.prefix + PAGE - 1) / PAGE;
  p.own_qb = p.max_tokens * p.G <= 16 ? 1 : 2;
  p.RBo = (p.max_tokens * p.G + 16 * p.own_qb - 1) / (16 * p.own_qb);
  // Splits: a start and a share of the merge cost each of them some pages' time, and so does each further page of a split: about as many
  // splits as pages of one, at least half as many workgroups as CUs, at most as many as run at once. (Graph replays, 1024 pages of 8 x 64,
  // 128 rows: 16 splits 43 us, 32 29, 64 32, 128 39; 256 pages of 4 x 128, 320 rows: 8 splits 37, 16 28, 32 32.)
  const int64_t units = (int64_t)p.KVH * p.RBp;
  int64_t sp = pages ? splits ? splits : std::max<int64_t>((int64_t)std::ceil(std::sqrt((double)pages)), cus / (2 * units)) : 0;
  if (!splits) sp = std::min(sp, std::max<int64_t>(1, sa_waves(D) * cus / units));
  sp = std::min<int64_t>(sp, splits ? pages : (pages + 2 * wp - 1) / (2 * wp));
  p.pps = sp ? (int)((pages + sp - 1) / sp) : 0;
  p.Sp = p.pps ? (pages + p.pps - 1) / p.pps : 0;
  const int64_t own = (int64_t)p.R * p.KVH * p.RBo;
  p.So = (int)std::max<int64_t>(1, std::min<int64_t>({sa_waves(D) * cus / own, (p.own_pages + 15) / 16, 64}));
}

size_t shared_workspace(const SharedAttn& p, int D) {
  const size_t rows = (size_t)p.KVH * p.T * p.G * (p.Sp + p.So);
  return rows * D * sizeof(float) + rows * sizeof(f32x2);
}

int shared_launch(SharedAttn& p, int D, hipStream_t s) {
  const size_t rows = (size_t)p.KVH * p.T * p.G * (p.Sp + p.So);
  p.part_ml = reinterpret_cast<f32x2*>(p.part_o + rows * D);
  const dim3 grid((unsigned)((p.KVH * p.Sp + 7) / 8 * 8 * p.RBp + p.R * p.KVH * p.RBo * p.So)), block(SA_THREADS);
#define SA_GO(D, QB, ROWS)                                                                                  \
  do {                                                                                                      \
    if (p.own_qb == 1)                                                                                      \
      hipLaunchKernelGGL((shared_attn_kernel<D, QB, ROWS, 1>), grid, block, 0, s, p);                        \
    else                                                                                                    \
      hipLaunchKernelGGL((shared_attn_kernel<D, QB, ROWS, 2>), grid, block, 0, s, p);                        \
  } while (0)
  if (D == 64) {
    switch (p.cfg) {
      case 0: SA_GO(64, 1, false); break;
      case 1: SA_GO(64, 2, false); break;
      case 2: SA_GO(64, 1, true); break;
      default: SA_GO(64, 2, true); break;
    }
  } else {
    switch (p.cfg) {
      case 0: SA_GO(128, 1, false); break;
      case 1: SA_GO(128, 2, false); break;
      case 2: SA_GO(128, 1, true); break;
      default: SA_GO(128, 2, true); break;
    }
  }
#undef SA_GO
  if (const hipError_t e = hipGetLastError(); e != hipSuccess) return (int)e;
  // four waves for a row whose splits one wave would take in more than two rounds, where a workgroup a row is a launch of under 2^32 threads
  const int64_t units = (int64_t)p.R * p.max_tokens * p.QH;
  const bool four = p.Sp + p.So > 2 * SA_ROUND * 256 / D && units < 1 << 24;
  const dim3 merge((unsigned)(four ? units : (units + 3) / 4));
  if (D == 64 && four)
    hipLaunchKernelGGL((shared_merge_kernel<64, 4>), merge, block, 0, s, p);
  else if (D == 64)
    hipLaunchKernelGGL((shared_merge_kernel<64, 1>), merge, block, 0, s, p);
  else if (four)
    hipLaunchKernelGGL((shared_merge_kernel<128, 4>), merge, block, 0, s, p);
  else
    hipLaunchKernelGGL((shared_merge_kernel<128, 1>), merge, block, 0, s, p);
  return (int)hipGetLastError();
}

}  // namespace dspark
