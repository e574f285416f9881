// extern "C" entry points of the 8-bit block-scaled K/V cache (declared in include/dspark.h). As in capi.cpp, every shape,
// range and alignment a kernel assumes is checked here, on the host, before anything is launched.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>

#include "dspark.h"
#include "dspark_internal.h"
#include "b8.h"

using namespace dspark;

namespace {

constexpr int64_t POS_MAX = ((int64_t)1 << 31) - 2 * DSPARK_PAGE_TOKENS;  // positions and their page ends stay in int32
constexpr int HEADS_MAX = 1024;

hipStream_t S(dspark_stream_t s) { return reinterpret_cast<hipStream_t>(s); }
bool on(const void* p, uintptr_t bytes) { return p && (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
int64_t pages_of(int64_t positions) { return (positions + DSPARK_PAGE_TOKENS - 1) / DSPARK_PAGE_TOKENS; }

bool cache_ok(const dspark_b8_cache* c) {
  if (!c || !on(c->k, 16) || !on(c->v, 16) || !on(c->k_scale, 4) || !on(c->v_scale, 4)) return false;
  if (c->D != 64 && c->D != 128) return false;
  if (c->code != DSPARK_B8_INT8 && c->code != DSPARK_B8_E4M3) return false;
  if (c->KVH < 1 || c->KVH > HEADS_MAX || c->kv_pages < 1 || c->kv_pages >= (int64_t)1 << 31) return false;
  return !c->block_table || on(c->block_table, 4);
}

// Positions 0 .. end - 1 lie in the pool (with a block table: wherever it says).
bool fits(const dspark_b8_cache* c, int64_t end) {
  return end <= POS_MAX && (c->block_table || pages_of(end) <= c->kv_pages);
}

// A launch of a wave per (page, K or V, head), four a workgroup: under 2^32 threads.
bool waves_fit(const dspark_b8_cache* c, int64_t pages) { return pages * 2 * c->KVH <= ((int64_t)1 << 26) - 4; }

B8Pool pool(const dspark_b8_cache* c) {
  B8Pool p;
  p.k = static_cast<uint8_t*>(c->k);
  p.v = static_cast<uint8_t*>(c->v);
  p.ks = c->k_scale;
  p.vs = c->v_scale;
  p.bt = c->block_table;
  p.pages = c->kv_pages;
  p.KVH = c->KVH;
  return p;
}

// Compute units of the current device (queried once per device).
int device_cus() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

bool rows_ok(const dspark_b8_cache* c, const dspark_b8_attn_args* a) {
  if (!cache_ok(c) || !a) return false;
  if (a->M < 1 || a->M > DSPARK_MT_MAX || a->QH < c->KVH || a->QH % c->KVH || (int64_t)a->QH / c->KVH * a->M > 64 * 16) return false;
  if (a->a < 0 || a->start < 0 || a->window < 0 || a->splits < 0) return false;
  return fits(c, (int64_t)a->a + a->M);
}
bool query_ok(const dspark_b8_cache* c, const dspark_b8_attn_args* a) {
  return on(a->q, 16) && a->q_stride >= (int64_t)a->QH * c->D && a->q_stride % 8 == 0;
}

B8Attn attn(const dspark_b8_cache* c, const dspark_b8_attn_args* a) {
  B8Attn p = {};
  p.c = pool(c);
  p.q = static_cast<const _Float16*>(a->q);
  p.q_stride = a->q_stride;
  p.out16 = static_cast<_Float16*>(a->out);
  p.out32 = a->out_f32;
  p.lse = a->lse;
  p.gate = a->gate;
  p.arrivals = a->arrivals;
  p.M = a->M;
  p.QH = a->QH;
  p.G = a->QH / c->KVH;
  p.a = a->a;
  p.start = a->start;
  p.window = a->window;
  p.causal = a->causal ? 1 : 0;
  return p;
}

// Memory that a call reads or writes: `rows` pieces of n bytes, `stride` apart (stride >= n); p NULL or n 0: none.
struct Span {
  const void* p;
  size_t n;
  size_t rows = 1, stride = 0;
};
// A piece of n bytes at `at` and some row of y share a byte: of y's rows the first that ends behind `at` begins before the piece ends.
bool meets(uintptr_t at, size_t n, const Span& y) {
  const uintptr_t b = reinterpret_cast<uintptr_t>(y.p);
  const size_t i = at < b + y.n ? 0 : y.rows > 1 ? (at - b - y.n) / y.stride + 1 : 1;
  return i < y.rows && b + i * y.stride < at + n;
}
bool overlap(const Span& x, const Span& y) {
  if (!x.p || !y.p || !x.n || !y.n) return false;
  const uintptr_t a = reinterpret_cast<uintptr_t>(x.p), b = reinterpret_cast<uintptr_t>(y.p);
  if (a >= b + (y.rows - 1) * y.stride + y.n || b >= a + (x.rows - 1) * x.stride + x.n) return false;
  if (x.rows > y.rows) return overlap(y, x);  // (of two spans here one has at most 1024 rows, heads or tokens)
  for (size_t i = 0; i < x.rows; ++i)
    if (meets(a + i * x.stride, x.n, y)) return true;
  return false;
}
// Nothing that is written shares a byte with what is read, nor with anything else that is written: workgroups read and store in
// no order among each other.
template <size_t NR, size_t NW>
bool apart(const Span (&reads)[NR], const Span (&writes)[NW]) {
  for (size_t i = 0; i < NW; ++i) {
    for (const Span& r : reads)
      if (overlap(r, writes[i])) return false;
    for (size_t j = 0; j < i; ++j)
      if (overlap(writes[j], writes[i])) return false;
  }
  return true;
}
size_t scale_bytes(const dspark_b8_cache* c) { return (size_t)c->kv_pages * c->KVH * sizeof(float); }
size_t code_bytes(const dspark_b8_cache* c) { return (size_t)c->kv_pages * c->KVH * DSPARK_PAGE_TOKENS * c->D; }
Span table(const dspark_b8_cache* c, int64_t positions) { return {c->block_table, (size_t)pages_of(positions) * sizeof(int32_t)}; }
// Rows of KVH D elements, row_stride apart.
Span rows_of(const dspark_b8_cache* c, const void* p, int64_t n, int64_t row_stride, size_t element) {
  return {p, (size_t)c->KVH * c->D * element, (size_t)n, (size_t)row_stride * element};
}
Span query(const dspark_b8_cache* c, const dspark_b8_attn_args* a) {
  return {a->q, (size_t)a->QH * c->D * 2, (size_t)a->M, (size_t)a->q_stride * 2};
}
// Accounts of n positions of every head.
Span accounts(const dspark_b8_cache* c, const float* p, int64_t n, int64_t stride) {
  return {p, (size_t)n * sizeof(float), (size_t)c->KVH, (size_t)stride * sizeof(float)};
}
// Two sets of n such rows share a byte (they may lie in turn in wider rows).
bool rows_meet(const Span& x, const Span& y, int64_t n, size_t row, size_t stride) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(x.p), b = reinterpret_cast<uintptr_t>(y.p);
  const size_t d = a < b ? b - a : a - b, q = d / stride, m = d % stride;
  return (m < row && q < (size_t)n) || (stride - m < row && q + 1 < (size_t)n);
}

}  // namespace

extern "C" {

int dspark_kv_write_b8(const dspark_b8_cache* c, const void* k, const void* v, int64_t row_stride, int32_t pos0, int32_t n,
                       dspark_stream_t stream) {
  if (!cache_ok(c) || pos0 < 0 || n < 0 || !fits(c, (int64_t)pos0 + n)) return DSPARK_EINVAL;
  if (n == 0) return 0;
  if (!on(k, 16) || !on(v, 16) || row_stride < (int64_t)c->KVH * c->D || row_stride % 8) return DSPARK_EINVAL;
  if (!waves_fit(c, pages_of((int64_t)n) + 1)) return DSPARK_EINVAL;
  const Span reads[3] = {rows_of(c, k, n, row_stride, 2), rows_of(c, v, n, row_stride, 2), table(c, (int64_t)pos0 + n)};
  const Span writes[4] = {{c->k, code_bytes(c)}, {c->v, code_bytes(c)}, {c->k_scale, scale_bytes(c)}, {c->v_scale, scale_bytes(c)}};
  if (!apart(reads, writes)) return DSPARK_EINVAL;
  B8Write p;
  p.c = pool(c);
  p.k = static_cast<const _Float16*>(k);
  p.v = static_cast<const _Float16*>(v);
  p.row_stride = row_stride;
  p.pos0 = pos0;
  p.n = n;
  return b8_write_launch(p, c->D, c->code == DSPARK_B8_E4M3, S(stream));
}

int dspark_kv_read_b8(const dspark_b8_cache* c, int32_t pos0, int32_t n, float* k, float* v, int64_t row_stride,
                      dspark_stream_t stream) {
  if (!cache_ok(c) || pos0 < 0 || n < 0 || !fits(c, (int64_t)pos0 + n)) return DSPARK_EINVAL;
  if (n == 0) return 0;
  if (!on(k, 16) || !on(v, 16) || row_stride < (int64_t)c->KVH * c->D || row_stride % 4) return DSPARK_EINVAL;
  if (!waves_fit(c, pages_of((int64_t)n) + 1)) return DSPARK_EINVAL;
  const Span reads[5] = {{c->k, code_bytes(c)}, {c->v, code_bytes(c)}, {c->k_scale, scale_bytes(c)}, {c->v_scale, scale_bytes(c)},
                         table(c, (int64_t)pos0 + n)};
  const Span ks[1] = {rows_of(c, k, n, row_stride, 4)}, vs[1] = {rows_of(c, v, n, row_stride, 4)};
  if (!apart(reads, ks) || !apart(reads, vs)) return DSPARK_EINVAL;
  if (rows_meet(ks[0], vs[0], n, (size_t)c->KVH * c->D * 4, (size_t)row_stride * 4)) return DSPARK_EINVAL;
  B8Read p;
  p.c = pool(c);
  p.k = k;
  p.v = v;
  p.row_stride = row_stride;
  p.pos0 = pos0;
  p.n = n;
  return b8_read_launch(p, c->D, c->code == DSPARK_B8_E4M3, S(stream));
}

size_t dspark_verify_attention_b8_workspace(const dspark_b8_cache* c, const dspark_b8_attn_args* a) {
  if (!rows_ok(c, a)) return 0;
  B8Attn p = attn(c, a);
  b8_attn_plan(p, c->D, a->splits, device_cus());
  return std::max(b8_attn_workspace(p, c->D), (size_t)256);  // (0 says that the arguments are refused)
}

int dspark_verify_attention_b8(const dspark_b8_cache* c, const dspark_b8_attn_args* a, dspark_stream_t stream) {
  if (!rows_ok(c, a) || !query_ok(c, a)) return DSPARK_EINVAL;
  if (!a->out && !a->out_f32) return DSPARK_EINVAL;
  if ((a->arrivals && !on(a->arrivals, 4)) || (a->lse && !on(a->lse, 4)) || (a->gate && !on(a->gate, 4))) return DSPARK_EINVAL;
  if ((a->out && !on(a->out, 16)) || (a->out_f32 && !on(a->out_f32, 16))) return DSPARK_EINVAL;
  B8Attn p = attn(c, a);
  b8_attn_plan(p, c->D, a->splits, device_cus());
  const size_t need = std::max(b8_attn_workspace(p, c->D), (size_t)256), heads = (size_t)a->M * a->QH;
  if (!on(a->workspace, 16) || a->workspace_bytes < need) return DSPARK_ENOSPACE;
  const Span reads[7] = {query(c, a), {a->gate, heads * 4}, {c->k, code_bytes(c)}, {c->v, code_bytes(c)},
                         {c->k_scale, scale_bytes(c)}, {c->v_scale, scale_bytes(c)}, table(c, (int64_t)a->a + a->M)};
  const Span writes[5] = {{a->out, heads * c->D * 2}, {a->out_f32, heads * c->D * 4}, {a->lse, heads * 4}, {a->workspace, need},
                          {a->arrivals, (size_t)c->KVH * DSPARK_B8_ARRIVALS * 4}};
  if (!apart(reads, writes)) return DSPARK_EINVAL;
  p.part_acc = static_cast<float*>(a->workspace);
  p.part_ml = reinterpret_cast<f32x2*>(p.part_acc + (size_t)p.c.KVH * p.R * p.S * c->D);
  return b8_attn_launch(p, c->D, c->code == DSPARK_B8_E4M3, S(stream));
}

int dspark_attention_mass_b8(const dspark_b8_cache* c, const dspark_b8_attn_args* a, const float* lse, const int32_t* rows,
                             const float* mass_in, float* mass_out, int64_t mass_stride, dspark_stream_t stream) {
  if (!rows_ok(c, a) || !query_ok(c, a) || !on(lse, 4) || !on(mass_out, 4) || (rows && !on(rows, 4))) return DSPARK_EINVAL;
  if (mass_stride < (int64_t)a->a + a->M) return DSPARK_EINVAL;
  if (mass_in && !on(mass_in, 4)) return DSPARK_EINVAL;
  const int64_t n = (int64_t)a->a + a->M;
  const Span reads[7] = {accounts(c, mass_in == mass_out ? nullptr : mass_in, n, mass_stride), query(c, a), {lse, (size_t)a->M * a->QH * 4}, {rows, 4},
                         {c->k, code_bytes(c)}, {c->k_scale, scale_bytes(c)}, table(c, (int64_t)a->a + a->M)};
  const Span writes[1] = {accounts(c, mass_out, n, mass_stride)};
  if (!apart(reads, writes)) return DSPARK_EINVAL;
  B8Attn p = attn(c, a);
  p.lse_in = lse;
  p.rows = rows;
  p.mass_in = mass_in;
  p.mass_out = mass_out;
  p.mass_stride = mass_stride;
  return b8_mass_launch(p, c->D, c->code == DSPARK_B8_E4M3, device_cus(), S(stream));
}

size_t dspark_kv_evict_b8_workspace(int32_t KVH, int32_t length) {
  if (KVH < 1 || KVH > HEADS_MAX || length < 0) return 0;
  return b8_evict_workspace(KVH, length);
}

int dspark_kv_evict_b8(const dspark_b8_cache* src, const dspark_b8_cache* dst, int32_t length, int32_t keep, int32_t sinks,
                       int32_t recent, const float* mass, int64_t mass_stride, int32_t* kept, float* mass_out,
                       int64_t mass_out_stride, void* workspace, size_t workspace_bytes, dspark_stream_t stream) {
  if (!cache_ok(src) || !cache_ok(dst) || src->KVH != dst->KVH || src->D != dst->D || src->code != dst->code) return DSPARK_EINVAL;
  if (length < 0 || keep < 0 || keep > length || sinks < 0 || recent < 0 || (int64_t)sinks + recent > keep) return DSPARK_EINVAL;
  if (length > 1 << 30 || !fits(src, length) || !fits(dst, keep) || !waves_fit(dst, pages_of(keep))) return DSPARK_EINVAL;
  if (keep == 0) return 0;
  if (!on(mass, 4) || !on(kept, 4) || !on(mass_out, 4) || mass_stride < length || mass_out_stride < keep) return DSPARK_EINVAL;
  const size_t need = b8_evict_workspace(src->KVH, length);
  if (need && (!on(workspace, 16) || workspace_bytes < need)) return DSPARK_ENOSPACE;
  // a destination page may be written while other rows are still read
  const Span reads[7] = {{src->k, code_bytes(src)}, {src->v, code_bytes(src)}, {src->k_scale, scale_bytes(src)},
                         {src->v_scale, scale_bytes(src)}, accounts(src, mass, length, mass_stride),
                         table(src, length), table(dst, keep)};
  const Span writes[7] = {{dst->k, code_bytes(dst)}, {dst->v, code_bytes(dst)}, {dst->k_scale, scale_bytes(dst)},
                          {dst->v_scale, scale_bytes(dst)}, accounts(src, mass_out, keep, mass_out_stride),
                          {kept, (size_t)src->KVH * keep * 4}, {workspace, need}};
  if (!apart(reads, writes)) return DSPARK_EINVAL;
  B8Evict p;
  p.src = pool(src);
  p.dst = pool(dst);
  p.T = length;
  p.keep = keep;
  p.sinks = sinks;
  p.recent = recent;
  p.mass = mass;
  p.mass_stride = mass_stride;
  p.kept = kept;
  p.mass_out = mass_out;
  p.mass_out_stride = mass_out_stride;
  return b8_evict_launch(p, src->D, src->code == DSPARK_B8_E4M3, workspace, S(stream));
}

}  // extern "C"
