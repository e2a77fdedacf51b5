// kv_plan.cu -- block tables and slot maps of a paged KV cache, built on the
// GPU from the requests' lengths (no counterpart in titoatwork/qgemm-mx, which
// stops at the GEMMs).
//
// With P tokens per block, request r holding len_r tokens and bringing n_r:
//   starts = exclusive prefix sum of n
//   need_r = ceil((len_r + n_r) / P) - ceil(len_r / P)   new blocks
//   upto_r = inclusive prefix sum of need
// and r's j-th new block is free_list[count - 1 - (upto_r - need_r + j)]: the
// free list is a stack, taken from its end in request order.
//
// What bounds it: latency.  A step's lengths are a few KB and its slot map 12
// bytes a token; the dependent chain is lengths -> scan -> block id -> slot.
// So it is one launch: every CTA scans all requests itself (chunks of 1024
// from L2) instead of waiting for another CTA's prefix, and then fills its own
// range of 256-token rows, finding each token's request by binary search in
// shared memory.
#include "kv.cuh"

namespace qg {

constexpr int kPlanThreads = 256;
constexpr int kPlanItems = 4;                          // requests per thread and chunk
constexpr int kPlanChunk = kPlanThreads * kPlanItems;

struct PlanArgs {
  const int32_t *lens, *news;
  int32_t* table;
  const int32_t *free_list, *free_count;
  int32_t free_len;  // entries of the free list
  int32_t requests, width, block_log2, tokens, max_runs;
  int32_t *lens_out, *starts;
  int64_t* slots;
  int32_t *positions, *runs, *counts;
};

// One request's sizes.
struct PlanSize {
  int len, n, have, need, touched;
  bool fits;  // its tokens fit its row of the table
};
// Sums that stop at 2^30; the terms are at most that each, so 32 bits unsigned hold them.
__device__ __forceinline__ int sat_add(int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)kKvMaxTokens); }
// Blocks that n tokens after the first len touch.
__device__ __forceinline__ int runs_of(int len, int n, int lg) {
  return n > 0 ? (int)(((long long)len + n - 1) >> lg) - (len >> lg) + 1 : 0;
}
__device__ __forceinline__ PlanSize plan_size(int len, int n, int width, int lg) {
  PlanSize s;
  const int P1 = (1 << lg) - 1;
  s.len = max(len, 0);
  s.n = max(n, 0);
  s.have = (int)(((long long)s.len + P1) >> lg);
  const long long last = ((long long)s.len + s.n + P1) >> lg;
  s.fits = last <= width && len >= 0;
  s.need = s.fits ? (int)last - s.have : 0;
  s.touched = runs_of(s.len, s.n, lg);
  return s;
}

__global__ void __launch_bounds__(kPlanThreads) k_kv_plan(const PlanArgs a) {
  __shared__ int s_start[kPlanChunk + 1], s_upto[kPlanChunk], s_run[kPlanChunk], s_len[kPlanChunk];
  __shared__ int s_warp[3][kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int lg = a.block_log2;
  pdl_begin();
  const int count = a.free_list ? min(max(*a.free_count, 0), a.free_len) : 0;
  // this CTA's rows
  const int t0 = (int)((long long)blockIdx.x * a.tokens / gridDim.x);
  const int t1 = (int)((long long)(blockIdx.x + 1) * a.tokens / gridDim.x);
  long long base_tok = 0;
  int base_need = 0, base_run = 0;  // needs stop mattering past `count`, so they saturate below
  int used = 0, refused = 0, leads = 0;
  for (int r0 = 0; r0 < a.requests; r0 += kPlanChunk) {
    PlanSize z[kPlanItems];
    long long tok = 0;
    int need = 0, run = 0;
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i) {
      const int r = r0 + tid * kPlanItems + i;
      z[i] = r < a.requests ? plan_size(a.lens[r], a.news[r], a.width, lg) : PlanSize{0, 0, 0, 0, 0, true};
      tok += z[i].n; need += z[i].need; run += z[i].touched;
    }
    // Sums stop at 2^30: rows past `tokens` are never written, and no request is granted
    // blocks where their count has stopped.
    int sums[3] = {(int)min(tok, (long long)kKvMaxTokens), min(need, kKvMaxTokens), min(run, kKvMaxTokens)};
    int incl[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int v = sums[k];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
        if (lane >= d) v = sat_add(v, u);
      }
      incl[k] = v;
      if (lane == 31) s_warp[k][warp] = v;
    }
    __syncthreads();
    int before[3], total[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int b = 0, t = 0;
#pragma unroll
      for (int w = 0; w < kPlanThreads / 32; ++w) {
        if (w == warp) b = t;
        t = sat_add(t, s_warp[k][w]);
      }
      const int up = __shfl_up_sync(0xFFFFFFFFu, incl[k], 1);
      before[k] = sat_add(b, lane ? up : 0);
      total[k] = t;
    }
    long long at = base_tok + before[0];
    int upto = sat_add(base_need, before[1]), runs = sat_add(base_run, before[2]);
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i) {
      const int j = tid * kPlanItems + i, r = r0 + j;
      upto = sat_add(upto, z[i].need);
      const bool granted = z[i].fits && at + z[i].n <= a.tokens && (z[i].need == 0 || (upto <= count && upto < kKvMaxTokens));
      s_start[j] = (int)min(at, (long long)kKvMaxTokens);
      s_upto[j] = granted ? upto - z[i].need : -1;
      s_run[j] = runs;
      s_len[j] = z[i].len;
      if (r < a.requests) {
        leads += runs_of(z[i].len, (int)min((long long)z[i].n, max(a.tokens - at, 0ll)), lg);  // of rows that exist
        if (granted) used = max(used, upto);
        else ++refused;
        if (blockIdx.x == 0) {
          a.starts[r] = s_start[j];
          a.lens_out[r] = granted ? z[i].len + z[i].n : a.lens[r];
        }
      }
      at = min(at + z[i].n, (long long)kKvMaxTokens);
      runs = sat_add(runs, z[i].touched);
    }
    base_tok = min(base_tok + total[0], (long long)kKvMaxTokens);
    if (tid == kPlanThreads - 1) s_start[kPlanChunk] = (int)base_tok;
    base_need = sat_add(base_need, total[1]);
    base_run = sat_add(base_run, total[2]);
    __syncthreads();
    // tokens of this chunk in this CTA's range
    const int lo = max(t0, s_start[0]), hi = min(t1, s_start[kPlanChunk]);
    for (int t = lo + tid; t < hi; t += kPlanThreads) {
      int b = 0;  // the last request with start <= t: empty requests share a start with the next
#pragma unroll
      for (int step = kPlanChunk / 2; step; step >>= 1)
        if (s_start[b + step] <= t) b += step;
      const int r = r0 + b, len = s_len[b];
      // 64 bits: a request that is refused may hold close to 2^31 tokens
      const long long at_t = (long long)len + (t - s_start[b]);
      const int blk = (int)(at_t >> lg), off = (int)at_t & ((1 << lg) - 1);
      const int taken = s_upto[b];
      int64_t slot = -1;
      if (taken >= 0) {
        const int have = (len + (1 << lg) - 1) >> lg;
        int id;
        if (blk < have) {
          id = a.table[(size_t)r * a.width + blk];
        } else {
          id = a.free_list[count - 1 - (taken + blk - have)];
          if (off == 0) a.table[(size_t)r * a.width + blk] = id;  // a new block starts with a new token
        }
        slot = ((int64_t)id << lg) + off;
      }
      a.slots[t] = slot;
      a.positions[t] = taken >= 0 ? (int)at_t : -1;
      if (t == s_start[b] || off == 0) {
        const int k = s_run[b] + blk - (len >> lg);
        if (k < a.max_runs) a.runs[k] = t;
      }
    }
    __syncthreads();
  }
  // rows no request covers, the runs' end marks, and the totals
  const int total = (int)min(base_tok, (long long)a.tokens);
  for (int t = max(t0, total) + tid; t < t1; t += kPlanThreads) {
    a.slots[t] = -1;
    a.positions[t] = -1;
  }
  if (blockIdx.x != 0) return;
  __shared__ int s_used, s_refused, s_leads;
  if (tid == 0) { s_used = 0; s_refused = 0; s_leads = 0; }
  __syncthreads();
  if (used) atomicMax(&s_used, used);
  if (refused) atomicAdd(&s_refused, refused);
  if (leads) atomicAdd(&s_leads, leads);
  __syncthreads();
  for (int k = s_leads + tid; k <= a.max_runs; k += kPlanThreads) a.runs[k] = total;
  if (tid == 0) {
    a.starts[a.requests] = (int)base_tok;
    a.counts[0] = count - s_used;
    a.counts[1] = s_leads;
    a.counts[2] = total;
    a.counts[3] = s_refused;
  }
}

// Two of the call's buffers that share a byte, one of them an output: CTAs read the inputs
// while others write the outputs.
struct PlanSpan {
  const char* name;
  const void* at;
  long long bytes;
};
static bool plan_overlap(const PlanArgs& a, const char** x, const char** y) {
  const long long R = a.requests, T = a.tokens;
  const PlanSpan spans[] = {
      {"lens_out", a.lens_out, 4 * R}, {"starts", a.starts, 4 * R + 4}, {"slots", a.slots, 8 * T},
      {"positions", a.positions, 4 * T}, {"runs", a.runs, 4 * (a.max_runs + 1ll)}, {"counts", a.counts, 16},
      {"lens", a.lens, 4 * R}, {"news", a.news, 4 * R}, {"table", a.table, 4 * R * a.width},
      {"free_list", a.free_list, !a.free_list ? 0 : a.free_len == INT32_MAX ? 4 : 4ll * a.free_len}, {"free_count", a.free_count, 4}};
  constexpr int outputs = 6, all = sizeof(spans) / sizeof(spans[0]);
  auto meet = [&](int i, int j) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(spans[i].at), q = reinterpret_cast<uintptr_t>(spans[j].at);
    const uintptr_t n = (uintptr_t)spans[i].bytes, m = (uintptr_t)spans[j].bytes;
    return (n > 0) & (m > 0) & (p < q + m) & (q < p + n);
  };
  int any = 0;  // no branches while there is nothing to report
  for (int i = 0; i < outputs; ++i)
    for (int j = i + 1; j < all; ++j) any |= meet(i, j);
  for (int i = 0; any && i < outputs; ++i)
    for (int j = i + 1; j < all; ++j)
      if (meet(i, j)) {
        *x = spans[i].name;
        *y = spans[j].name;
        return true;
      }
  return false;
}

}  // namespace qg

using namespace qg;

extern "C" {

int32_t qgemm_kv_max_runs(int32_t requests, int32_t tokens, int32_t block) {
  if (requests < 0 || tokens < 0 || !kv_block_ok(block)) return -1;
  const long long b = 2ll * requests + tokens / block;
  return (int32_t)(b < tokens ? b : tokens);
}

qgemm_status_t qgemm_kv_plan_bounded(int32_t block, int32_t requests, const int32_t* lens, const int32_t* news,
                                     int32_t* table, int32_t table_width, const int32_t* free_list, int32_t free_len,
                                     const int32_t* free_count, int32_t tokens, int32_t* lens_out, int32_t* starts,
                                     int64_t* slots, int32_t* positions, int32_t* runs, int32_t* counts,
                                     void* stream) {
  if (!kv_block_ok(block)) return fail(QGEMM_ERR_INVALID_ARG, "kv_plan: block must be 16, 32, 64 or 128 tokens");
  if (requests < 0 || tokens < 0 || table_width < 0 || free_len < 0)
    return fail(QGEMM_ERR_INVALID_ARG, "kv_plan: negative size");
  if (tokens >= kKvMaxTokens) return fail(QGEMM_ERR_INVALID_ARG, "kv_plan: at most 2^30 - 1 rows");
  if ((long long)table_width * block > INT32_MAX)  // lengths and positions have 32 bits
    return fail(QGEMM_ERR_UNSUPPORTED_SHAPE, "kv_plan: table rows of more than 2^31 - 1 tokens");
  if (!free_count || !starts || !runs || !counts || (requests && (!lens || !news || !lens_out)) ||
      (requests && table_width && !table) || (tokens && (!slots || !positions)))
    return fail(QGEMM_ERR_INVALID_ARG, "kv_plan: null pointer");
  PlanArgs a;
  a.lens = lens; a.news = news; a.table = table; a.free_list = free_list; a.free_count = free_count;
  a.free_len = free_len;
  a.requests = requests; a.width = table_width; a.tokens = tokens;
  a.block_log2 = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7;
  a.max_runs = qgemm_kv_max_runs(requests, tokens, block);
  a.lens_out = lens_out; a.starts = starts; a.slots = slots; a.positions = positions; a.runs = runs;
  a.counts = counts;
  const char *x = nullptr, *y = nullptr;
  if (plan_overlap(a, &x, &y))
    return fail(QGEMM_ERR_INVALID_ARG, "kv_plan: %s and %s overlap: CTAs read inputs while others write outputs", x, y);
  DevProps dp;
  qgemm_status_t st = device_props(&dp);
  if (st != QGEMM_OK) return st;
  int grid = (tokens + kPlanThreads - 1) / kPlanThreads;
  grid = grid < 1 ? 1 : grid > dp.sm_count ? dp.sm_count : grid;
  QG_CUDA_RET(pdl_launch(k_kv_plan, dim3((unsigned)grid), dim3(kPlanThreads), 0, as_stream(stream), a));
  return QGEMM_OK;
}

qgemm_status_t qgemm_kv_plan(int32_t block, int32_t requests, const int32_t* lens, const int32_t* news,
                             int32_t* table, int32_t table_width, const int32_t* free_list,
                             const int32_t* free_count, int32_t tokens, int32_t* lens_out, int32_t* starts,
                             int64_t* slots, int32_t* positions, int32_t* runs, int32_t* counts, void* stream) {
  return qgemm_kv_plan_bounded(block, requests, lens, news, table, table_width, free_list, INT32_MAX, free_count, tokens,
                               lens_out, starts, slots, positions, runs, counts, stream);
}

}  // extern "C"
