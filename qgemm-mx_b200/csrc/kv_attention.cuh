// kv_attention.cuh -- what the attention kernels over the paged 8-bit cache share.
//
// Arithmetic (both kernels).  With codes kc, vc and block exponents ek, ev:
//   s   = (q . kc) 2^ek scale log2(e)               score, in powers of two
//   w   = 2^(s + ev - m)                             weight with V's scale folded in
//   out = sum(w vc) / sum(w 2^-ev)
// V's scale rides in the exponent, so P.V needs no factor per block: w is
// rounded once to f16 beside the exact f16 widening of vc (off by 2^-11 of a weight at
// most, where the result's own rounding to bf16 may be off by 2^-8; the tensor cores
// take f16 beside f16 only), and the denominator takes the unrounded w times 2^-ev in 32 bits.  Scales
// are 2^-64 .. 2^122, as the append writes them (the cache's description requires
// it), so that denominator stays below 2^80 times the token count.
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
  int rows_min, rows_max;  // rows per KV head of the requests this launch takes
  float scale_log2;  // scale * log2(e)
  int window, causal;
  uint16_t* out;
  float* lse;
  int beside;  // the launch before is this call's other kernel, whose results are not needed
  unsigned* ready;  // set once what came before the call is done, cleared by the join kernel; or null
  unsigned* tickets;  // the decode kernel's: zero between calls
  float* partials;
};

constexpr float kKvTop = 10.0f;   // log2 of the largest weight after m moves
constexpr float kKvGrow = 15.0f;  // and the one that makes it move

// The approximate exp2 and reciprocal are off by some 2^-22 of the value, the roundings
// of the weights and of the result by up to 2^-11 and 2^-8.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// 1 / l, 0 for a row that saw no token (l is 2^-112 or more otherwise, or NaN)
__device__ __forceinline__ float kv_inv(float l) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(l));
  return l == 0.0f ? 0.0f : y;
}
__device__ __forceinline__ float kv_lse(float m, float l) {
  return l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
}

// A kernel that starts beside the one before it reads the call's inputs, which earlier
// kernels wrote, without a griddepcontrol.wait of its own.  What orders those reads: a
// kernel that has waited says so (release) before its dependents may start, and they
// look (acquire).  A block that does not see it waits for the whole kernel instead.
// All threads must call kv_look.
__device__ __forceinline__ void kv_tell(const KvAttnArgs& a) {
  if (a.ready && blockIdx.x == 0 && threadIdx.x == 0)
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(a.ready), "r"(1u) : "memory");
}
__device__ __forceinline__ void kv_look(const KvAttnArgs& a) {
  unsigned seen = 0;
  if (threadIdx.x == 0) asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(a.ready) : "memory");
  if (!__syncthreads_or((int)seen)) pdl_wait();
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
template <int MOST>
struct KvBatch {
  int prefix[MOST + 1], start[MOST + 1], len[MOST];
  __device__ __forceinline__ KvRequest at(const KvAttnArgs& a, int r) const {
    return kv_request(a, start[r], start[r + 1], len[r]);
  }
};

// ---- the line: all pairs' tiles, one after another ---------------------------
// A pair is (request, KV head, group of RG rows); its tokens are tiles of
// T = 2^TL.  The line gives group g of a request S(g + 1) - S(g) places,
//   S(g) = floor(sum over k < g of (h0 + (k + 1) slope) / T + kStart),
// where h0 + (g + 1) slope bounds the tokens the group sees: slope is RG / group
// tokens, rounded up, for causal rows and 0 otherwise.  floor(a + x) - floor(a)
// >= floor(x), so kStart = 1 suffices for the group's tiles; the places beyond
// stand for the cost of starting a pair.  A closed form keeps causal prompts
// balanced (their groups see from few to all tokens) without a list of groups.
template <int RG, int TL>
struct KvLine {
  // Tiles of 16 go by in a quarter of the time that a pair's queries, search and
  // store take: 64 requests of 129 to 8192 tokens 97 us, 200 in a window of 128
  // 18.5 us, against 101 and 19.9 with 2, 97 and 19.2 with 8, 104 and 29.4 with 1.
  // Of the prefill kernel's 128 tokens a start weighs three: 13 decoding requests and 3
  // prompt chunks of up to 512 tokens 120 us, 132 with 1, 122 with 5.  (All of them
  // calls behind one another in a CUDA graph, in one run.)
  static constexpr int kStart = TL == 4 ? 4 : 3;
  int h0, slope, groups;
  __host__ __device__ __forceinline__ KvLine(const KvAttnArgs& a, const KvRequest& q) {
    h0 = q.len;
    slope = 0;
    const int per = (RG + a.group - 1) / a.group;
    const long long near = (long long)a.window + min(q.n, per + 1) - 1 + (1 << TL);  // a group spans per + 1 tokens at most
    if (a.window > 0 && a.causal && near < q.len) {
      h0 = (int)near;
    } else if (a.causal && q.n > 1) {
      h0 = max(q.len - q.n_all, 0) + 1;
      slope = per;
    }
    groups = (int)(((unsigned)q.n * (unsigned)a.group + RG - 1u) / RG);
  }
  __device__ __forceinline__ int upto(int g) const {
    return (int)(((long long)g * h0 + (long long)slope * ((long long)g * (g + 1) / 2)) >> TL) + g * kStart;
  }
};

// One stretch of one pair's tiles.
struct KvSeg {
  int pair_v, pair_end;  // the pair's range on the line
  int r, h, row0, rows;  // rows: the request's n * group
  int start, n, n_all, len;
  int tile, tile_end;    // absolute tiles to visit
};

// The stretch that begins at place v of the line and ends with its pair or at
// v_end; r: a request at or before v's, moved to it.  Its loops are not
// unrolled: code that runs once a stretch costs its instruction fetches.
template <int RG, int TL, int MOST>
__device__ __forceinline__ void kv_seg(const KvAttnArgs& a, const KvBatch<MOST>& b, int& r, int v, int v_end, KvSeg& s) {
#pragma unroll 1
  while (b.prefix[r + 1] <= v) ++r;
  const KvRequest q = b.at(a, r);
  const KvLine<RG, TL> line(a, q);
  const int per_head = line.upto(line.groups);
  s.r = r;
  s.h = (int)((unsigned)(v - b.prefix[r]) / (unsigned)per_head);
  const int head_v = b.prefix[r] + s.h * per_head;
  int g = 0;
#pragma unroll 1
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

// Most places one request can take on the line (host): no group is given more tokens
// than its request holds and one more, and the slope of all groups.
inline long long kv_line_most(const KvAttnArgs& a, int rg, int tl) {
  const long long rows = (long long)a.max_new * a.group < a.rows_max ? (long long)a.max_new * a.group : a.rows_max;
  const long long groups = (rows + rg - 1) / rg;
  const long long tokens = ((long long)a.width << a.block_log2) + 1 + groups * ((rg + a.group - 1) / a.group);
  const long long per_head = groups * ((tokens >> tl) + 5);
  return per_head > (1ll << 40) ? per_head : per_head * a.heads;
}

// The line cut into E shares of V / E or one more places.
struct KvCuts {
  unsigned size, longer;  // the first `longer` shares have size + 1 places
  __device__ __forceinline__ KvCuts(int V, int E) : size((unsigned)V / (unsigned)E), longer((unsigned)V % (unsigned)E) {}
  __device__ __forceinline__ int at(int k) const { return (int)(k * size + min((unsigned)k, longer)); }
  __device__ __forceinline__ int share_of(int v) const {
    const unsigned u = (unsigned)v, edge = longer * (size + 1);
    return (int)(u < edge ? u / (size + 1) : longer + (u - edge) / size);
  }
};

// The request whose pairs hold line position v (empty ones hold none).
template <int MOST>
__device__ __forceinline__ int kv_find(const KvBatch<MOST>& b, int requests, int v) {
  int lo = 0, hi = requests;
#pragma unroll 1
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.prefix[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}

// Fills the batch and returns the line's length; LONGEST: and the most places a pair
// has, at most 2^15, in `longest`.  The first WARPS warps do the work; all threads must
// call it.  scan: WARPS words, 2 WARPS with LONGEST.
template <int RG, int TL, int WARPS, bool LONGEST, int MOST>
__device__ __forceinline__ int kv_line_any(const KvAttnArgs& a, KvBatch<MOST>& b, int* scan, int& longest) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int base = 0;
  longest = 0;
#pragma unroll 1
  for (int r0 = 0; r0 < a.requests; r0 += WARPS * 32) {
    const int r = r0 + tid;
    const bool on = tid < WARPS * 32 && r < a.requests;
    int c = 0, most = 0;
    if (on) {
      const int start = a.starts[r], end = a.starts[r + 1], len = a.lens[r];
      b.start[r] = start;
      b.len[r] = len;
      if (r == a.requests - 1) b.start[r + 1] = end;
      const KvRequest q = kv_request(a, start, end, len);
      if (q.n > 0) {
        const KvLine<RG, TL> line(a, q);
        c = a.heads * line.upto(line.groups);
        // the last group's is the largest
        if (LONGEST) most = min(line.upto(line.groups) - line.upto(line.groups - 1), 1 << 15);
      }
    }
    int v = c;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
      if (lane >= d) v += u;
    }
    if (LONGEST) most = __reduce_max_sync(0xFFFFFFFFu, most);
    if (lane == 31 && warp < WARPS) {
      scan[warp] = v;
      if (LONGEST) scan[WARPS + warp] = most;
    }
    __syncthreads();
    int before = base, total = base;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w == warp) before = total;
      total += scan[w];
      if (LONGEST) longest = max(longest, scan[WARPS + w]);
    }
    if (on) b.prefix[r] = before + v - c;
    base = total;
    __syncthreads();
  }
  if (tid == 0) b.prefix[a.requests] = base;
  __syncthreads();
  return base;
}
template <int RG, int TL, int WARPS, int MOST>
__device__ __forceinline__ int kv_line(const KvAttnArgs& a, KvBatch<MOST>& b, int* scan) {
  int longest;
  return kv_line_any<RG, TL, WARPS, false>(a, b, scan, longest);
}
template <int RG, int TL, int WARPS, int MOST>
__device__ __forceinline__ int kv_line(const KvAttnArgs& a, KvBatch<MOST>& b, int* scan, int& longest) {
  return kv_line_any<RG, TL, WARPS, true>(a, b, scan, longest);
}

// One row (of RG) of a pair that crosses CTAs, joined by a warp from the CTAs'
// partials in CTA order: lane i takes dims 4 i .. 4 i + 3 (HD = 128), or 2 i,
// 2 i + 1.  Lanes first take a contributor's (m, l) each, so that the chain of
// L2 trips is short: one for every 16 contributors' values.
template <int RG, int HD>
struct KvJoined {
  float acc[HD / 32], M, L;
};
template <int RG, int HD>
__device__ __forceinline__ KvJoined<RG, HD> kv_join(const float* partials, int slot, int c_first, int c_last, int row) {
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31;
  KvJoined<RG, HD> j;
  j.M = -INFINITY;
  j.L = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) j.acc[i] = 0.0f;
#pragma unroll 1
  for (int c0 = c_first; c0 <= c_last; c0 += 32) {
    constexpr int Y = 16;
    const int n = min(c_last - c0 + 1, 32);
    const float* const p0 = partials + 2 * (size_t)c0 * slot;  // contributor c's at 2 c slot, the first one's one slot on
    const int begun = c0 == c_first ? slot : 0;
    float m = -INFINITY, l = 0.0f, f = 0.0f;
    if (lane < n) {
      const float* p = p0 + 2 * lane * slot + (lane == 0 ? begun : 0) + RG * HD + row;
      m = __ldcg(p);
      l = __ldcg(p + RG);
    }
    const float* p = p0 + row * HD + lane * N;
#pragma unroll 1
    for (int c = 0; c < n; c += Y, p += 2 * Y * slot) {
      float x[Y][N];
#pragma unroll
      for (int y = 0; y < Y; ++y) {
        const float* q = p + 2 * y * slot;
        if (y == 0 && c == 0) q += begun;
#pragma unroll
        for (int i = 0; i < N; ++i) x[y][i] = 0.0f;
        if (c + y < n) {
          if (N == 4) {
            const float4 o = __ldcg(reinterpret_cast<const float4*>(q));
            x[y][0] = o.x; x[y][1] = o.y; x[y][N - 2] = o.z; x[y][N - 1] = o.w;
          } else {
            const float2 o = __ldcg(reinterpret_cast<const float2*>(q));
            x[y][0] = o.x; x[y][1] = o.y;
          }
        }
      }
      if (c == 0) {  // here, so that the loads above are under way meanwhile
        if (l == 0.0f) m = -INFINITY;  // a share that saw no token
        float top = m;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        top = fmaxf(top, j.M);
        const float mu = top == -INFINITY ? 0.0f : top;
        const float f0 = ex2(j.M - mu);
        f = l != 0.0f ? ex2(m - mu) : 0.0f;
        float sum = l * f;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        j.L = fmaf(j.L, f0, sum);
        j.M = top;
#pragma unroll
        for (int i = 0; i < N; ++i) j.acc[i] *= f0;
      }
#pragma unroll
      for (int y = 0; y < Y; ++y) {
        const float w = __shfl_sync(0xFFFFFFFFu, f, c + y);  // lanes from n on hold 0
        if (w != 0.0f) {
#pragma unroll
          for (int i = 0; i < N; ++i) j.acc[i] = fmaf(x[y][i], w, j.acc[i]);
        }
      }
    }
  }
  if (j.L == 0.0f) j.M = 0.0f;
  return j;
}
// Stores that row: query row `token` (of the batch), query head `head`.
template <int RG, int HD>
__device__ __forceinline__ void kv_store(const KvAttnArgs& a, int token, int head, const KvJoined<RG, HD>& j) {
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)token * (a.heads * a.group) + head;
  const float f = kv_inv(j.L);
  uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + at * HD) + lane * (HD / 64);
#pragma unroll
  for (int i = 0; i < HD / 64; ++i) dst[i] = pack_bf16(j.acc[2 * i] * f, j.acc[2 * i + 1] * f);
  if (a.lse && lane == 0) a.lse[at] = kv_lse(j.M, j.L);
}

}  // namespace qg
