// kv_attention.cuh -- what the attention kernels over the paged 8-bit cache share.
//
// Arithmetic (both kernels).  With codes kc, vc and block exponents ek, ev:
//   s   = (q . kc) 2^ek scale log2(e)               score, in powers of two
//   w   = 2^(s + ev - m)                             weight with V's scale folded in
//   out = sum(w vc) / sum(w 2^-ev)
// V's scale rides in the exponent, so P.V needs no factor per block: w is
// rounded once to f16 beside the exact f16 widening of vc, and the denominator
// takes the unrounded w times 2^-ev in 32 bits.  Scales are at least 2^-64, so
// that denominator stays below 2^80 times the token count.
// m is a running reference, not the maximum: it moves to max(s + ev) - 10 only
// when a value passes m + 15.  Rescaling is then rare, w stays below 2^15, and
// f16 keeps its 11 bits for weights down to 2^-24 of the largest.
// q is divided by a power of two per row that brings its largest value to
// [1, 2): exact in f16 except below 2^-24 of that.
#pragma once

#include "kv.cuh"

namespace qg {

struct KvAttnArgs {
  const uint8_t *k, *v, *ks, *vs;
  const uint16_t* q;
  int64_t q_stride, q_head_stride;
  const int32_t *starts, *lens, *table;
  int width, block_log2;  // table width, log2 of tokens per block
  int64_t blocks;
  int requests, tokens, heads, group;  // group: query heads per KV head
  int max_new;
  float scale_log2;  // scale * log2(e)
  int window, causal;
  uint16_t* out;
  float* lse;
  unsigned* tickets;  // zero between calls
  float* partials;
};

constexpr float kKvTop = 10.0f;   // log2 of the largest weight after m moves
constexpr float kKvGrow = 15.0f;  // and the one that makes it move

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Tokens row i of n sees: [lo, hi).
__device__ __forceinline__ int row_hi(const KvAttnArgs& a, int len, int n, int i) {
  return a.causal ? min(max(len - n + i + 1, 0), len) : len;
}
__device__ __forceinline__ int row_lo(const KvAttnArgs& a, int len, int n, int i) {
  return a.window > 0 ? (int)max((long long)len - n + i - a.window + 1, 0ll) : 0;
}

// A request's rows and length as the kernels take them (rows past max_new or
// past the row count are not computed, lengths end with the table).
struct KvRequest {
  int start, n, len, n_all;
};
__device__ __forceinline__ KvRequest kv_request(const KvAttnArgs& a, int r) {
  KvRequest q;
  q.start = a.starts[r];
  q.n_all = a.starts[r + 1] - q.start;
  q.n = min(min(q.n_all, a.max_new), a.tokens - q.start);
  if (q.start < 0 || q.n < 0) q.n = 0;
  q.len = (int)min((long long)max(a.lens[r], 0), (long long)a.width << a.block_log2);
  return q;
}

}  // namespace qg
