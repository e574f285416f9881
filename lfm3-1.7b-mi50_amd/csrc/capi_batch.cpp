// extern "C" entry points of the operators for a batch of sequences (declared in include/dspark.h). As in capi.cpp, every shape,
// range and alignment a kernel assumes is checked here, on the host, before anything is launched.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "dspark.h"
#include "dspark_internal.h"
#include "batch.h"
#include "spans.h"

using namespace dspark;

namespace {

constexpr int HEADS_MAX = 1024, QUERY_HEADS_MAX = 4096;  // (rows x group < 2^32: div_by)
constexpr int64_t STRIDE_MAX = (int64_t)1 << 30;  // elements between rows: byte offsets of 2^30 rows stay in 64 bits
hipStream_t S(dspark_stream_t s) { return reinterpret_cast<hipStream_t>(s); }
int64_t pages_of(int64_t positions) { return (positions + DSPARK_PAGE_TOKENS - 1) / DSPARK_PAGE_TOKENS; }

size_t pool_bytes(int64_t pages, int KVH, int D) { return (size_t)pages * KVH * DSPARK_PAGE_TOKENS * D * 2; }

// Rows of `heads` heads, `stride` elements apart; nothing if there are no heads.
Span rows_of(const void* p, int64_t n, int heads, int D, int64_t stride, size_t size) {
  return {heads ? p : nullptr, (size_t)heads * D * size, (size_t)n, (size_t)stride * size};
}

SharedAttn shared_params(const dspark_shared_attn_args* a) {
  SharedAttn p = {};
  p.q = static_cast<const _Float16*>(a->q);
  p.q_stride = a->q_stride;
  p.kp = static_cast<const _Float16*>(a->k_pages);
  p.vp = static_cast<const _Float16*>(a->v_pages);
  p.pages = a->kv_pages;
  p.ptab = a->prefix_table;
  p.q_start = a->q_start;
  p.own_len = a->own_len;
  p.own_tab = a->own_table;
  p.own_stride = a->own_stride;
  p.out16 = static_cast<_Float16*>(a->out);
  p.out32 = a->out_f32;
  p.lse = a->lse;
  p.gate = a->gate;
  p.c = (float)(1.4426950408889634074 / std::sqrt((double)a->D));
  p.prefix = a->prefix;
  p.T = a->tokens;
  p.R = a->seqs;
  p.max_tokens = a->max_tokens;
  p.own_pages = a->own_pages;
  p.QH = a->QH;
  p.KVH = a->KVH;
  p.G = a->QH / a->KVH;
  p.g_div = div_magic(p.G);
  // a window of all positions or more is none: the kernels' differences with those that are left (< 3 x 2^29) stay in 32 bits, also
  // from positions below 0 (of sequences with fewer own keys than tokens)
  p.window = a->window < (int64_t)a->prefix + (int64_t)a->own_pages * DSPARK_PAGE_TOKENS ? a->window : 0;
  p.causal = a->causal ? 1 : 0;
  shared_plan(p, a->D, a->splits, device_cus());
  return p;
}

constexpr int SAMPLE_ROWS = 65535, SAMPLE_VOCAB = 1 << 20;

bool shared_ok(const dspark_shared_attn_args* a) {
  if (!a || (a->D != 64 && a->D != 128) || a->KVH < 1 || a->KVH > HEADS_MAX || a->QH < a->KVH || a->QH % a->KVH) return false;
  if (a->QH > QUERY_HEADS_MAX || a->prefix < 0 || a->prefix >= 1 << 30 || a->tokens < 0 || a->seqs < 0 || a->seqs > 1 << 20) return false;
  if (a->max_tokens < 0 || a->max_tokens > a->tokens || (a->tokens && a->max_tokens < 1)) return false;
  if ((int64_t)a->tokens * (a->QH / a->KVH) > 1 << 20) return false;
  if (a->own_pages < 0 || a->own_pages > 1 << 24 || a->own_stride < a->own_pages || a->own_stride >= STRIDE_MAX) return false;
  if (a->kv_pages < 1 || a->kv_pages >= (int64_t)1 << 31 || (!a->prefix_table && pages_of(a->prefix) > a->kv_pages)) return false;
  if (a->window < 0 || a->splits < 0 || a->q_stride < (int64_t)a->QH * a->D || a->q_stride >= STRIDE_MAX) return false;
  if (!a->tokens || !a->seqs) return true;
  // launches of under 2^32 threads
  const SharedAttn p = shared_params(a);
  const int64_t prefix = ((int64_t)p.KVH * p.Sp + 7) / 8 * 8 * p.RBp, own = (int64_t)p.R * p.KVH * p.RBo * p.So;
  return prefix + own < 1 << 24 && (int64_t)p.R * p.max_tokens * p.QH / 4 < 1 << 24;
}

}  // namespace

extern "C" {

int dspark_rope_freqs(int32_t rot, double base, int32_t scaling, double factor, double trained, double low, double high,
                      double* freq, double* scale) {
  if (!freq || rot < 2 || rot % 2 || !(base > 0) || !std::isfinite(base) || !(factor >= 1) || !std::isfinite(factor)) return DSPARK_EINVAL;
  if (scaling < DSPARK_ROPE_PLAIN || scaling > DSPARK_ROPE_RAMP) return DSPARK_EINVAL;
  if (scaling == DSPARK_ROPE_RAMP && !(trained > 0 && low >= 0 && high > low)) return DSPARK_EINVAL;
  // (one pair alone has nothing between the first and the slowest: its frequency is 1 at any base)
  const double b = scaling == DSPARK_ROPE_BASE && rot > 2 ? base * std::pow(factor, rot / (rot - 2.0)) : base;
  for (int i = 0; i < rot / 2; ++i) {
    double f = std::pow(b, -2.0 * i / rot);
    if (scaling == DSPARK_ROPE_LINEAR) f /= factor;
    if (scaling == DSPARK_ROPE_RAMP) {
      const double turns = trained * f / 6.283185307179586476925;
      const double keep = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
      f = f * keep + f / factor * (1 - keep);
    }
    freq[i] = f;
  }
  if (scale) *scale = scaling == DSPARK_ROPE_RAMP ? 0.1 * std::log(factor) + 1 : 1.0;
  return 0;
}

int dspark_rope(const dspark_rope_args* a, dspark_stream_t stream) {
  if (!a || a->n < 0 || a->n >= 1 << 23 || a->QH < 0 || a->KVH < 0 || a->QH > HEADS_MAX || a->KVH > HEADS_MAX || a->QH + a->KVH < 1)
    return DSPARK_EINVAL;
  if (a->D < 2 || a->D > 1024 || a->D % 2 || a->rot < 2 || a->rot > a->D || a->rot % 2) return DSPARK_EINVAL;
  if (a->type != DSPARK_F16 && a->type != DSPARK_BF16 && a->type != DSPARK_F32) return DSPARK_EINVAL;
  const bool append = a->k_pages || a->v_pages;
  // (the strides of what is not there are not looked at)
  if ((a->QH && std::max(a->q_stride, a->q_out_stride) >= STRIDE_MAX) || (a->KVH && a->k_stride >= STRIDE_MAX)) return DSPARK_EINVAL;
  if (a->KVH && (append ? a->v_stride : a->k_out_stride) >= STRIDE_MAX) return DSPARK_EINVAL;
  if (a->n == 0) return 0;
  const size_t size = a->type == DSPARK_F32 ? 4 : 2;
  if (!on(a->positions, 4) || !on(a->freq, 8)) return DSPARK_EINVAL;
  if (a->QH && (!on(a->q, size) || !on(a->q_out, size) || a->q_stride < (int64_t)a->QH * a->D || a->q_out_stride < (int64_t)a->QH * a->D))
    return DSPARK_EINVAL;
  if (a->KVH && (!on(a->k, size) || a->k_stride < (int64_t)a->KVH * a->D)) return DSPARK_EINVAL;
  if (append) {
    if (a->KVH < 1 || a->type != DSPARK_F16 || a->inverse || (a->D != 64 && a->D != 128) || a->k_out) return DSPARK_EINVAL;
    if (!on(a->k_pages, 16) || !on(a->v_pages, 16) || !on(a->v, 2) || a->v_stride < (int64_t)a->KVH * a->D || !on(a->slots, 8)) return DSPARK_EINVAL;
    if (a->kv_pages < 1 || a->kv_pages >= (int64_t)1 << 31 || (int64_t)a->n * a->KVH >= 1 << 27) return DSPARK_EINVAL;
  } else if (a->KVH && (!on(a->k_out, size) || a->k_out_stride < (int64_t)a->KVH * a->D)) {
    return DSPARK_EINVAL;
  }
  // in place: an output that is its input itself
  const bool q_in_place = a->QH && a->q == a->q_out && a->q_stride == a->q_out_stride;
  const bool k_in_place = !append && a->KVH && a->k == a->k_out && a->k_stride == a->k_out_stride;
  const Span q = rows_of(a->q, a->n, a->QH, a->D, a->q_stride, size), k = rows_of(a->k, a->n, a->KVH, a->D, a->k_stride, size);
  const Span v = rows_of(append ? a->v : nullptr, a->n, a->KVH, a->D, a->v_stride, 2);
  const Span pos = {a->positions, (size_t)a->n * 4}, freq = {a->freq, (size_t)a->rot / 2 * 8};
  const Span slots = {append ? a->slots : nullptr, (size_t)a->n * 8};
  const Span q_out[1] = {rows_of(a->q_out, a->n, a->QH, a->D, a->q_out_stride, size)};
  const Span k_out[3] = {rows_of(append ? nullptr : a->k_out, a->n, a->KVH, a->D, a->k_out_stride, size),
                         {append ? a->k_pages : nullptr, pool_bytes(append ? a->kv_pages : 0, a->KVH, a->D)},
                         {append ? a->v_pages : nullptr, pool_bytes(append ? a->kv_pages : 0, a->KVH, a->D)}};
  const Span none = {nullptr, 0};
  const Span q_reads[9] = {q_in_place ? none : q, k, v, pos, freq, slots, k_out[0], k_out[1], k_out[2]};
  const Span k_reads[6] = {q, k_in_place ? none : k, v, pos, freq, slots};
  if (!apart(q_reads, q_out) || !apart(k_reads, k_out)) return DSPARK_EINVAL;
  RopeBatch p = {};
  p.q = {a->q, a->q_out, a->q_stride, a->q_out_stride, a->QH};
  p.k = {a->k, append ? nullptr : a->k_out, a->k_stride, append ? 0 : a->k_out_stride, a->KVH};
  p.v = {append ? a->v : nullptr, nullptr, a->v_stride, 0, append ? a->KVH : 0};
  p.pos = a->positions;
  p.freq = a->freq;
  p.scale = a->scale;
  p.n = a->n;
  p.D = a->D;
  p.rot = a->rot;
  p.inverse = a->inverse ? 1 : 0;
  if (append) {
    p.kp = static_cast<_Float16*>(a->k_pages);
    p.vp = static_cast<_Float16*>(a->v_pages);
    p.slots = a->slots;
    p.n_slots = a->kv_pages * DSPARK_PAGE_TOKENS;
    p.KVH = a->KVH;
  }
  return rope_batch_launch(p, a->type, a->interleaved != 0, S(stream));
}

size_t dspark_verify_attention_shared_workspace(const dspark_shared_attn_args* a) {
  if (!shared_ok(a)) return 0;
  if (a->tokens == 0 || a->seqs == 0) return 256;
  const SharedAttn p = shared_params(a);
  return std::max(shared_workspace(p, a->D), (size_t)256);  // (0 says that the arguments are refused)
}

int dspark_verify_attention_shared(const dspark_shared_attn_args* a, dspark_stream_t stream) {
  if (!shared_ok(a)) return DSPARK_EINVAL;
  if (a->tokens == 0 || a->seqs == 0) return 0;
  if (!on(a->q, 16) || !on(a->k_pages, 16) || !on(a->v_pages, 16) || a->q_stride % 8) return DSPARK_EINVAL;
  if (!on(a->q_start, 4) || !on(a->own_len, 4) || (a->own_pages && !on(a->own_table, 4))) return DSPARK_EINVAL;
  if (!a->out && !a->out_f32) return DSPARK_EINVAL;
  if ((a->out && !on(a->out, 16)) || (a->out_f32 && !on(a->out_f32, 16))) return DSPARK_EINVAL;
  if ((a->lse && !on(a->lse, 4)) || (a->gate && !on(a->gate, 4)) || (a->prefix_table && !on(a->prefix_table, 4))) return DSPARK_EINVAL;
  SharedAttn p = shared_params(a);
  const size_t need = std::max(shared_workspace(p, a->D), (size_t)256), heads = (size_t)a->tokens * a->QH;
  if (!on(a->workspace, 16) || a->workspace_bytes < need) return DSPARK_ENOSPACE;
  const size_t pool = pool_bytes(a->kv_pages, a->KVH, a->D);
  const Span reads[8] = {rows_of(a->q, a->tokens, a->QH, a->D, a->q_stride, 2), {a->gate, heads * 4}, {a->k_pages, pool}, {a->v_pages, pool},
                         {a->prefix_table, (size_t)pages_of(a->prefix) * 4}, {a->q_start, ((size_t)a->seqs + 1) * 4},
                         {a->own_len, (size_t)a->seqs * 4},
                         {a->own_pages ? a->own_table : nullptr, (size_t)a->own_pages * 4, (size_t)a->seqs, (size_t)a->own_stride * 4}};
  const Span writes[4] = {{a->out, heads * a->D * 2}, {a->out_f32, heads * a->D * 4}, {a->lse, heads * 4}, {a->workspace, need}};
  if (!apart(reads, writes)) return DSPARK_EINVAL;
  p.part_o = static_cast<float*>(a->workspace);
  return shared_launch(p, a->D, S(stream));
}

size_t dspark_verify_sample_workspace(int32_t n, int32_t V) {
  if (n < 0 || n > SAMPLE_ROWS || V < 1 || V > SAMPLE_VOCAB) return 0;
  SampleParams p = {};
  p.n = std::max(n, 1);
  p.V = V;
  sample_plan(p);
  return sample_workspace(p, nullptr);
}

int dspark_verify_sample(const dspark_sample_args* a, dspark_stream_t stream) {
  if (!a || a->n < 0 || a->n > SAMPLE_ROWS || a->V < 1 || a->V > SAMPLE_VOCAB) return DSPARK_EINVAL;
  if (a->type != DSPARK_F16 && a->type != DSPARK_BF16 && a->type != DSPARK_F32) return DSPARK_EINVAL;
  if (a->n == 0) return 0;
  const size_t size = a->type == DSPARK_F32 ? 4 : 2, n = a->n;
  if (!on(a->logits, size) || a->row_stride < a->V || a->row_stride >= STRIDE_MAX || !on(a->u, 4)) return DSPARK_EINVAL;
  if (!a->tokens && !a->keys) return DSPARK_EINVAL;
  for (const void* x : {(const void*)a->temperature, (const void*)a->top_k, (const void*)a->top_p, (const void*)a->min_p,
                        (const void*)a->tokens, (const void*)a->kept, (const void*)a->logprob})
    if (x && !on(x, 4)) return DSPARK_EINVAL;
  if (a->keys && !on(a->keys, 8)) return DSPARK_EINVAL;
  SampleParams p = {};
  p.logits = a->logits;
  p.stride = a->row_stride;
  p.u = a->u;
  p.temperature = a->temperature;
  p.top_k = a->top_k;
  p.top_p = a->top_p;
  p.min_p = a->min_p;
  p.temperature_all = a->temperature_all;
  p.top_p_all = a->top_p_all;
  p.min_p_all = a->min_p_all;
  p.top_k_all = a->top_k_all;
  p.tokens = a->tokens;
  p.keys = a->keys;
  p.kept = a->kept;
  p.logprob = a->logprob;
  p.n = a->n;
  p.V = a->V;
  p.wide = on(a->logits, 16) && (a->n == 1 || (size_t)a->row_stride * size % 16 == 0);
  sample_plan(p);
  const size_t need = sample_workspace(p, a->workspace);
  if (!on(a->workspace, 16) || a->workspace_bytes < need) return DSPARK_ENOSPACE;
  const Span reads[6] = {{a->logits, (size_t)a->V * size, n, (size_t)a->row_stride * size}, {a->u, n * 4}, {a->temperature, n * 4},
                         {a->top_k, n * 4}, {a->top_p, n * 4}, {a->min_p, n * 4}};
  const Span writes[5] = {{a->tokens, n * 4}, {a->keys, n * 8}, {a->kept, n * 4}, {a->logprob, n * 4}, {a->workspace, need}};
  if (!apart(reads, writes)) return DSPARK_EINVAL;
  return sample_launch(p, a->type, S(stream));
}

}  // extern "C"
