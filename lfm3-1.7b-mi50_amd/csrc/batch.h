// Launch descriptors of the operators for a batch of sequences: rotary positions with K/V by slot (rope.hip), attention
// behind a shared prefix (attn_shared.hip) and sampling (sample.hip).
#pragma once
#include "common.h"

namespace dspark {

struct RopeTensor {
  const void* x;
  void* y;             // (append: nullptr for K and V, whose rows go into the pages)
  int64_t x_stride, y_stride;
  int heads;
};
struct RopeBatch {
  RopeTensor q, k, v;  // v: append only
  const int32_t* pos;
  const double* freq;
  double scale;
  int n, D, rot, inverse;
  _Float16* kp;        // append: the page pools, or nullptr
  _Float16* vp;
  const int64_t* slots;
  int64_t n_slots;
  int KVH;
  // rope_batch_launch sets: units of a head and of a token, their divisors, tokens of a workgroup
  int uph, upt, tok;
  int fill, v_wide;    // append: workgroups that fill pages; V in pieces of 16 bytes
  uint32_t uph_div, upt_div;
};
int rope_batch_launch(RopeBatch& p, int type, bool interleaved, hipStream_t s);

// Attention of `R` sequences behind a shared prefix. Rows of a KV head: r = token G + query head of the group. A row's partial
// sums lie at (head rows + r) S + s: s < Sp the prefix's splits, then So of its sequence's own keys.
struct SharedAttn {
  const _Float16* q;
  int64_t q_stride;
  const _Float16* kp;
  const _Float16* vp;
  int64_t pages;
  const int32_t* ptab;
  const int32_t* q_start;
  const int32_t* own_len;
  const int32_t* own_tab;
  int64_t own_stride;
  _Float16* out16;
  float* out32;
  float* lse;
  const float* gate;
  float* part_o;       // [KVH][T G][S][D], unnormalised
  f32x2* part_ml;      // [KVH][T G][S]: reference (log2 units), sum
  float c;             // log2(e) / sqrt(D)
  int prefix, T, R, max_tokens, own_pages, QH, KVH, G, window, causal;
  uint32_t g_div;
  // shared_plan
  int cfg;             // prefix workgroups' shape
  int Sp, pps;         // splits of the prefix, pages of each
  int So;              // splits of a sequence's own pages
  int RBp, RBo;        // row blocks of the prefix (all rows) and of a sequence
  int own_qb;          // 16-row blocks of an own workgroup: 1 or 2
};
void shared_plan(SharedAttn& p, int D, int splits, int cus);
size_t shared_workspace(const SharedAttn& p, int D);
int shared_launch(SharedAttn& p, int D, hipStream_t s);

// Sampling (sample.hip).
// A row's settings, and what is known of it between the launches.
struct SampleLocals {
  double inv_t, inv_t2;  // 1 / T, log2(e) / T
  double low;            // min-p's bound of (z - m) / T
  float m;               // the row's maximum
  uint32_t first;        // where it is first
  float p;               // top-p (1: none)
  int k;                 // top-k (0: none)
  bool greedy, empty, cut_low, inf;  // inf: the maximum is +inf, differences to it are no numbers
};
struct SampleBegun {
  SampleLocals s;        // without what needs the maximum
};
struct SampleRow {
  SampleLocals s;
  uint32_t mode, bin;     // bin in which the cut lies
  uint32_t by_mass;       // the cut is top-p's (else top-k's)
  float u;                // (set by the third launch)
  uint64_t above, limit;  // weight (else tokens) in the bins above it, and of what is kept, before min-p
};
struct SampleParams {
  const void* logits;
  int64_t stride;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int32_t* tokens;
  uint64_t* keys;
  int32_t* kept;
  float* logprob;
  int n, V, wide;         // rows on 16-byte boundaries
  int P, ps;              // parts of a row in the first launch and their tokens (a multiple of a workgroup's step),
  int P2, ps2, P3, ps3;   // in the second and the third
  int chunks;             // of a row: as many tokens as a wave takes at a time
  // workspace
  uint64_t* part_key;     // [n][P] the part's largest key
  uint64_t* chunk_sum;    // [n][chunks] weight that is kept whatever the cut in the bin
  uint64_t* hist_mass;    // [n][bins]
  uint64_t* whole;        // [n] the row's weight
  SampleBegun* rows;      // [n] after the first launch
  SampleRow* result;      // [n] after the second
  float* part_sum;        // [n][P] about the part's weight, in units of its largest
  uint32_t* hist_count;   // [n][bins]
  uint64_t* list;         // [n][list] tokens: argmax keys
  uint64_t* taken;        // [n] tokens listed, and above bit 32 tokens kept above the bin
  uint32_t* marks;        // [n][2] arrivals of the second and the third launch
};
void sample_plan(SampleParams& p);
size_t sample_workspace(SampleParams& p, void* ws);
int sample_launch(const SampleParams& p, int type, hipStream_t s);

}  // namespace dspark
