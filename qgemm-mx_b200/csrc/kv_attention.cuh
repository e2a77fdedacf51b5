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

constexpr int kKvMaxRequests = 1024;  // per launch: they are kept in shared memory

struct KvAttnArgs {
  const uint8_t *k, *v, *ks, *vs;
  const uint16_t* q;
  int64_t q_stride, q_head_stride;
  const int32_t *starts, *lens, *table;
  int width, block_log2;  // table width, log2 of tokens per block
  int64_t blocks;
  int requests, tokens, heads, group;  // group: query heads per KV head
  int max_new;
  int rows_min, rows_max;  // rows per KV head of the requests this launch takes
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

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

__device__ __forceinline__ float kv_lse(float m, float l) {
  return l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Tokens row i of n sees: [lo, hi).
__device__ __forceinline__ int row_hi(const KvAttnArgs& a, int len, int n, int i) {
  return a.causal ? min(max(len - n + i + 1, 0), len) : len;
}
__device__ __forceinline__ int row_lo(const KvAttnArgs& a, int len, int n, int i) {
  return a.window > 0 ? (int)max((long long)len - n + i - a.window + 1, 0ll) : 0;
}

// A request's rows and length as the kernels take them: rows past max_new or
// past the row count are not computed, lengths end with the table, and a
// request whose rows per KV head are not in (rows_min, rows_max] belongs to
// the other kernel and has none here.
struct KvRequest {
  int start, n, len, n_all;
};
__device__ __forceinline__ KvRequest kv_request(const KvAttnArgs& a, int start, int end, int len) {
  KvRequest q;
  q.start = start;
  q.n_all = end - start;
  q.n = min(min(q.n_all, a.max_new), a.tokens - start);
  const long long rows = (long long)q.n * a.group;
  if (start < 0 || q.n < 0 || rows <= a.rows_min || rows > a.rows_max) q.n = 0;
  q.len = (int)min((long long)max(len, 0), (long long)a.width << a.block_log2);
  return q;
}
// A launch's requests in shared memory: prefix sums of their places on the
// line (below), row starts and lengths.
struct KvBatch {
  int prefix[kKvMaxRequests + 1], start[kKvMaxRequests + 1], len[kKvMaxRequests];
  __device__ __forceinline__ KvRequest at(const KvAttnArgs& a, int r) const {
    return kv_request(a, start[r], start[r + 1], len[r]);
  }
};

// ---- the line: all pairs' tiles, one after another ---------------------------
// A pair is (request, KV head, group of RG rows); its tokens are tiles of
// T = 2^TL.  The line gives group g of a request S(g + 1) - S(g) places,
//   S(g) = floor(sum over k < g of (h0 + (k + 1) slope) / T + 1),
// where h0 + (g + 1) slope bounds the tokens the group sees: slope is RG / group
// tokens for causal rows, 0 otherwise.  floor(a + x) - floor(a) >= floor(x), so
// the places suffice for the group's tiles; the spare one stands for the cost
// of starting a pair.  A closed form keeps causal prompts balanced (their
// groups see from few to all tokens) without a list of groups.
template <int RG, int TL>
struct KvLine {
  long long c0, den;  // S(g) = (c0 g + RG g (g + 1)) / den, or c0 g / T without a slope
  int groups;
  __device__ __forceinline__ KvLine(const KvAttnArgs& a, const KvRequest& q) {
    long long h0 = q.len;
    den = 0;
    const int span = min(q.n, (RG + a.group - 2) / a.group + 1);  // tokens of one group
    const long long near = (long long)a.window + span - 1 + (1 << TL);
    if (a.window > 0 && a.causal && near < q.len) {
      h0 = near;
    } else if (a.causal && q.n > 1) {
      h0 = max(q.len - q.n_all, 0) + 1;
      den = (2ll * a.group) << TL;
    }
    c0 = h0 + (1 << TL);
    if (den) c0 *= 2 * a.group;
    groups = (q.n * a.group + RG - 1) / RG;
  }
  __device__ __forceinline__ int upto(int g) const {
    return den ? (int)((c0 * g + (long long)RG * g * (g + 1ll)) / den) : (int)((c0 * g) >> TL);
  }
};

// One stretch of one pair's tiles.
struct KvSeg {
  int pair_v, pair_end;  // the pair's range on the line
  int r, h, row0, rows;  // rows: the request's n * group
  int start, n, n_all, len;
  int tile, tile_end;    // absolute tiles to visit
};

template <int RG, int TL>
__device__ __forceinline__ void kv_seg(const KvAttnArgs& a, const KvBatch& b, int& r, int v, int v_end, KvSeg& s) {
  while (b.prefix[r + 1] <= v) ++r;
  const KvRequest q = b.at(a, r);
  const KvLine<RG, TL> line(a, q);
  const int per_head = line.upto(line.groups);
  s.r = r;
  s.h = (v - b.prefix[r]) / per_head;
  const int head_v = b.prefix[r] + s.h * per_head;
  int g = 0;
  for (int hi = line.groups; hi - g > 1;) {
    const int mid = (g + hi) >> 1;
    if (head_v + line.upto(mid) <= v) g = mid; else hi = mid;
  }
  s.row0 = g * RG;
  s.rows = q.n * a.group;
  s.start = q.start; s.n = q.n; s.n_all = q.n_all; s.len = q.len;
  s.pair_v = head_v + line.upto(g);
  s.pair_end = head_v + line.upto(g + 1);
  const int i0 = s.row0 / a.group, i1 = (min(s.row0 + RG, s.rows) - 1) / a.group;
  const int lo = row_lo(a, q.len, q.n_all, i0) >> TL;
  const int hi = (int)(((long long)row_hi(a, q.len, q.n_all, i1) + (1 << TL) - 1) >> TL);
  s.tile = lo + (v - s.pair_v);
  s.tile_end = min(hi, lo + min(s.pair_end, v_end) - s.pair_v);
}

// Most places one request can take on the line (host).
inline long long kv_line_most(const KvAttnArgs& a, int rg, int tl) {
  const long long rows = (long long)a.max_new * a.group < a.rows_max ? (long long)a.max_new * a.group : a.rows_max;
  const long long groups = (rows + rg - 1) / rg;
  const long long tokens = ((long long)a.width << a.block_log2) + a.max_new + rg + (2ll << tl);
  const long long per_head = groups * ((tokens >> tl) + 2);
  return per_head > (1ll << 40) ? per_head : per_head * a.heads;
}

// The request whose pairs hold line position v (empty ones hold none).
__device__ __forceinline__ int kv_find(const KvBatch& b, int requests, int v) {
  int lo = 0, hi = requests;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.prefix[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}

// Fills the batch and returns the line's length.  The first WARPS warps do the
// work; all threads must call it.
template <int RG, int TL, int WARPS>
__device__ __forceinline__ int kv_line(const KvAttnArgs& a, KvBatch& b, int* scan) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int base = 0;
  for (int r0 = 0; r0 < a.requests; r0 += WARPS * 32) {
    const int r = r0 + tid;
    const bool on = tid < WARPS * 32 && r < a.requests;
    int c = 0;
    if (on) {
      const int start = a.starts[r], end = a.starts[r + 1], len = a.lens[r];
      b.start[r] = start;
      b.len[r] = len;
      if (r == a.requests - 1) b.start[r + 1] = end;
      const KvRequest q = kv_request(a, start, end, len);
      if (q.n > 0) {
        const KvLine<RG, TL> line(a, q);
        c = a.heads * line.upto(line.groups);
      }
    }
    int v = c;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
      if (lane >= d) v += u;
    }
    if (lane == 31 && warp < WARPS) scan[warp] = v;
    __syncthreads();
    int before = base, total = base;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w == warp) before = total;
      total += scan[w];
    }
    if (on) b.prefix[r] = before + v - c;
    base = total;
    __syncthreads();
  }
  if (tid == 0) b.prefix[a.requests] = base;
  __syncthreads();
  return base;
}

// The last CTA of a pair that crosses CTAs joins their partials, in CTA order:
// values 4 e4 .. 4 e4 + 3 of the group's RG x HD.  BATCH partials' loads are
// in flight before the first is used; one at a time this was a chain of L2
// trips as long as the contributors.
struct KvJoined {
  float4 acc;
  float M, L;
};
template <int RG, int HD, int BATCH>
__device__ __forceinline__ KvJoined kv_join(const float* partials, size_t slot, int c_first, int c_last, int e4) {
  const int qr = e4 * 4 / HD;
  KvJoined j{make_float4(0.0f, 0.0f, 0.0f, 0.0f), -INFINITY, 0.0f};
  for (int c0 = c_first; c0 <= c_last; c0 += BATCH) {
    float mx[BATCH], lx[BATCH];
    float4 ov[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      lx[i] = 0.0f;
      if (c0 + i <= c_last) {
        const float* p = partials + (size_t)((c0 + i) * 2 + (c0 + i == c_first ? 1 : 0)) * slot;
        mx[i] = __ldcg(p + RG * HD + qr);
        lx[i] = __ldcg(p + RG * HD + RG + qr);
        ov[i] = __ldcg(reinterpret_cast<const float4*>(p) + e4);
      }
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (lx[i] == 0.0f) continue;
      const float mn = fmaxf(j.M, mx[i]), f0 = j.M == -INFINITY ? 0.0f : ex2(j.M - mn), f1 = ex2(mx[i] - mn);
      j.acc.x = fmaf(ov[i].x, f1, j.acc.x * f0); j.acc.y = fmaf(ov[i].y, f1, j.acc.y * f0);
      j.acc.z = fmaf(ov[i].z, f1, j.acc.z * f0); j.acc.w = fmaf(ov[i].w, f1, j.acc.w * f0);
      j.L = fmaf(lx[i], f1, j.L * f0);
      j.M = mn;
    }
  }
  if (j.L == 0.0f) j.M = 0.0f;
  return j;
}
// Stores values 4 e4 .. of a finished group (and its rows' lse).
template <int HD>
__device__ __forceinline__ void kv_store(const KvAttnArgs& a, const KvSeg& s, int e4, const KvJoined& j) {
  const int row = s.row0 + e4 * 4 / HD, d = e4 * 4 % HD;
  if (row >= s.rows) return;
  const int i = row / a.group, gh = row - i * a.group;
  const int64_t at = (int64_t)(s.start + i) * a.heads * a.group + s.h * a.group + gh;
  const float f = j.L == 0.0f ? 0.0f : 1.0f / j.L;
  *reinterpret_cast<uint2*>(a.out + at * HD + d) =
      make_uint2(pack_bf16(j.acc.x * f, j.acc.y * f), pack_bf16(j.acc.z * f, j.acc.w * f));
  if (a.lse && d == 0) a.lse[at] = kv_lse(j.M, j.L);
}

}  // namespace qg
