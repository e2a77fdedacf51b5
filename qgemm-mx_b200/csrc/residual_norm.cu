// residual_norm.cu -- the norms before and after a decoder block in one pass:
//   r' = r + alpha * gate * N(y; post)      h = N(r'; pre)
// (no counterpart in titoatwork/qgemm-mx).  N is RMSNorm, or LayerNorm as
// mean, then mean square of the centred values.
//
// What bounds it: HBM for many rows, latency for few.  A row lives in
// registers from its one read to its one write: threads load all of y, the
// residual and the gate before the first reduction, so a row costs one trip
// to memory and one barrier per norm.  All sums are 32-bit floats; r' is
// rounded once, for its store, and h is the norm of the unrounded r'.
//
// With many rows the instructions count as well as the bytes (some 45 for each
// value's 14 bytes): values are worked on in pairs, and the warps' sums are
// joined by as many lanes as the row has warps.  Measured: 6000 rows of 2880,
// LayerNorm, gate, FP32 residual (242 MB): 49.5 us, 4.9 TB/s, 54.1 us with
// single values and the warps' sums added up one by one; one row of 8192,
// RMS: 2.9 us in a CUDA graph of such calls (host time sets 4.7 outside of one).
#include <cuda_bf16.h>

#include "common.cuh"

namespace qg {

struct NormArgs {
  const uint16_t* y;
  const void* residual;
  const uint16_t *post, *post_bias, *gate;
  int64_t gate_stride;
  const uint16_t *pre, *pre_bias;
  float alpha, eps;
  void* residual_out;
  uint16_t* h;
  int tokens, width;
  int nv;  // vectors of 8 in a row
  float inv_width;
  int row_warps;  // warps per row
  int row_half;   // half the power of two that spans them, 0 for one warp
};

// Two values in one 64-bit register: the FP32 pipe takes such pairs at twice
// the values per instruction.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ float2 split(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ void unpack8(const uint4& w, Pair (&f)[4]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = pair(u2f(u[i] << 16), u2f(u[i] & 0xFFFF0000u));
}
__device__ __forceinline__ uint4 pack8(const Pair (&f)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __float22bfloat162_rn(split(f[i]));
    u[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ uint4 vec_at(const uint16_t* p, int v) { return ld16(reinterpret_cast<const uint4*>(p) + v); }

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
  return x;
}

// A thread's place in its row: its first vector, the first warp of the row and
// how many values the own warp holds.
struct Place {
  int v0, first;
  float held;
};

// Sum of x over `2 * half` neighbouring lanes.
__device__ __forceinline__ float lanes_sum(float x, int half) {
  for (int d = half; d; d >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
  return x;
}

// x <- N(x) in place.  V vectors of 8 values per thread; those past the row are
// zero.  LayerNorm centres each warp's values on the warp's own mean m_w and
// joins the warps by M2 = sum_w (M2_w + n_w (m_w - mean)^2): as sound as a
// second pass over the centred row, at one barrier instead of two.  (The warp's mean may
// be off by the approximate division's 2^-22 of it, as by its sum's own rounding.)  `buf`: one
// entry per warp of the CTA, another one for each norm of a row.
template <int V, bool LAYER>
__device__ __forceinline__ void normalise(Pair (&x)[V][4], const uint16_t* weight, const uint16_t* bias, const Place& t,
                                          const NormArgs& a, float4* buf) {
  float shift = 0.0f;  // what LayerNorm still has to subtract
  float own_mean = 0.0f;
  if (LAYER) {
    Pair s = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) s = add2(s, x[j][i]);
    const float2 f = split(s);
    own_mean = __fdividef(warp_sum(f.x + f.y), t.held);
    const Pair m = pair(-own_mean, -own_mean);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (t.v0 + j * 32 * a.row_warps < a.nv) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[j][i] = add2(x[j][i], m);
      }
  }
  Pair q = 0;
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) q = fma2(x[j][i], x[j][i], q);
  const float2 f = split(q);
  float ss = warp_sum(f.x + f.y);
  if (a.row_warps > 1) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) buf[threadIdx.x >> 5] = make_float4(ss, own_mean, t.held, 0.0f);
    __syncthreads();
    const int peer = lane & (2 * a.row_half - 1);
    float4 e = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (peer < a.row_warps) e = buf[t.first + peer];
    if (LAYER) {
      const float mean = lanes_sum(e.y * e.z, a.row_half) * a.inv_width;
      const float d = e.y - mean;
      ss = lanes_sum(e.x + e.z * d * d, a.row_half);
      shift = own_mean - mean;
    } else {
      ss = lanes_sum(e.x, a.row_half);
    }
  }
  const float rs = rsqrtf(ss * a.inv_width + a.eps);
  const Pair rs2 = pair(rs, rs), off = pair(shift * rs, shift * rs);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int v = t.v0 + j * 32 * a.row_warps;
    if (v < a.nv) {
      Pair w[4];
      unpack8(vec_at(weight, v), w);
      if (LAYER) {
        Pair b[4] = {0, 0, 0, 0};
        if (bias) unpack8(vec_at(bias, v), b);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[j][i] = fma2(fma2(x[j][i], rs2, off), w[i], b[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[j][i] = mul2(mul2(x[j][i], rs2), w[i]);
      }
    }
  }
}

template <int V, bool LAYER, bool F32>
__global__ void __launch_bounds__(1024) k_residual_norm(const NormArgs a) {
  __shared__ float4 s_buf[2][32];
  const int row_threads = a.row_warps * 32;
  const int rows = blockDim.x / row_threads;  // rows per CTA
  const int mine = threadIdx.x / row_threads;
  const int row_raw = blockIdx.x * rows + mine;
  const bool live = row_raw < a.tokens;
  const int64_t row = live ? row_raw : a.tokens - 1;  // spare rows recompute the last one and store nothing
  Place t;
  t.v0 = threadIdx.x - mine * row_threads;
  t.first = mine * a.row_warps;
  // a warp's vectors: 32 from each 32 * warp + j * row_threads that the row has.
  // The first of them is never past the row, so no warp holds nothing.
  int held = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) held += min(max(a.nv - ((t.v0 & ~31) + j * row_threads), 0), 32);
  t.held = 8.0f * (float)held;
  pdl_begin();
  Pair r[V][4], x[V][4];
  uint4 g[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int v = t.v0 + j * row_threads;
    const bool on = v < a.nv;
    if (F32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.residual) + row * a.width) + 2 * v;
      const float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const float4 lo = on ? p[0] : z, hi = on ? p[1] : z;
      r[j][0] = pair(lo.x, lo.y); r[j][1] = pair(lo.z, lo.w);
      r[j][2] = pair(hi.x, hi.y); r[j][3] = pair(hi.z, hi.w);
    } else {
      const uint4 w = on ? reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.residual) + row * a.width)[v]
                         : make_uint4(0, 0, 0, 0);
      unpack8(w, r[j]);
    }
    const uint4 w = on && a.y ? reinterpret_cast<const uint4*>(a.y + row * a.width)[v] : make_uint4(0, 0, 0, 0);
    unpack8(w, x[j]);
    g[j] = on && a.gate ? vec_at(a.gate + row * a.gate_stride, v) : make_uint4(0, 0, 0, 0);
  }
  if (a.y) {
    if (a.post) normalise<V, LAYER>(x, a.post, a.post_bias, t, a, s_buf[0]);
    const Pair alpha = pair(a.alpha, a.alpha);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int v = t.v0 + j * row_threads;
      if (a.gate) {
        Pair f[4];
        unpack8(g[j], f);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[j][i] = mul2(x[j][i], f[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) r[j][i] = fma2(alpha, x[j][i], r[j][i]);
      if (live && v < a.nv) {
        if (F32) {
          float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.residual_out) + row * a.width) + 2 * v;
          const float2 f0 = split(r[j][0]), f1 = split(r[j][1]), f2 = split(r[j][2]), f3 = split(r[j][3]);
          p[0] = make_float4(f0.x, f0.y, f1.x, f1.y);
          p[1] = make_float4(f2.x, f2.y, f3.x, f3.y);
        } else {
          reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.residual_out) + row * a.width)[v] = pack8(r[j]);
        }
      }
    }
  }
  if (a.pre) {
    normalise<V, LAYER>(r, a.pre, a.pre_bias, t, a, s_buf[1]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int v = t.v0 + j * row_threads;
      if (live && v < a.nv) reinterpret_cast<uint4*>(a.h + row * a.width)[v] = pack8(r[j]);
    }
  }
}

template <int V, bool LAYER>
static cudaError_t launch_norm(const NormArgs& a, bool f32, unsigned grid, unsigned threads, cudaStream_t s) {
  return pdl_launch(f32 ? k_residual_norm<V, LAYER, true> : k_residual_norm<V, LAYER, false>, dim3(grid), dim3(threads), 0,
                    s, a);
}

// Whether an output shares a byte with the other output, or with an input whose elements
// there are not the same ones: a thread reads its own elements of a row before it writes
// them, but neither another thread's nor another row's.
static bool norm_overlap(const qgemm_residual_norm_t* p) {
  struct Span {
    const void* at;
    long long bytes, cell, stride;  // cell: bytes of an element; stride: bytes from row to row, 0 for all rows' one
  };
  const long long w = p->width, rows = p->tokens, own = p->residual_f32 ? 4 : 2;
  const Span outs[2] = {{p->y ? p->residual_out : nullptr, rows * w * own, own, w * own},
                        {p->pre ? p->h : nullptr, rows * w * 2, 2, w * 2}};
  const Span ins[7] = {{p->y, rows * w * 2, 2, w * 2},
                       {p->residual, rows * w * own, own, w * own},
                       {p->gate, ((p->gate_stride ? rows - 1 : 0) * p->gate_stride + w) * 2, 2,
                        rows == 1 ? w * 2 : p->gate_stride * 2},
                       {p->post, w * 2, 2, 0},
                       {p->post_bias, w * 2, 2, 0},
                       {p->pre, w * 2, 2, 0},
                       {p->pre_bias, w * 2, 2, 0}};
  auto meet = [](const Span& a, const Span& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    return x && y && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
  };
  if (meet(outs[0], outs[1])) return true;
  for (const Span& o : outs)
    for (const Span& i : ins)
      if (meet(o, i) && !(o.at == i.at && o.cell == i.cell && o.stride == i.stride)) return true;
  return false;
}

}  // namespace qg

using namespace qg;

extern "C" {

qgemm_status_t qgemm_residual_norm(const qgemm_residual_norm_t* p, void* stream) {
  if (!p) return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: null arguments");
  if (p->kind != QGEMM_NORM_RMS && p->kind != QGEMM_NORM_LAYER)
    return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: unknown kind %d", (int)p->kind);
  if (p->tokens < 0) return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: negative token count");
  if (p->width < 8 || p->width % 8 || p->width > 16384)
    return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: width must be a multiple of 8 in 8 .. 16384");
  if (!(p->eps >= 0.0f)) return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: eps must not be negative");
  if (!p->y && (p->post || p->gate)) return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: post or gate without y");
  if (!p->y && !p->pre) return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: neither y nor pre: nothing to do");
  if ((p->post_bias && !p->post) || (p->pre_bias && !p->pre))
    return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: a bias without its weight");
  if (p->kind == QGEMM_NORM_RMS && (p->post_bias || p->pre_bias))
    return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: the RMS norm has no bias");
  if (p->gate && (p->gate_stride < 0 || p->gate_stride % 8))
    return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: gate_stride must be a multiple of 8");
  if (p->tokens == 0) return QGEMM_OK;
  if (!p->residual || (p->y && !p->residual_out) || (p->pre && !p->h))
    return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: null pointer");
  const uintptr_t all = reinterpret_cast<uintptr_t>(p->y) | reinterpret_cast<uintptr_t>(p->residual) |
                        reinterpret_cast<uintptr_t>(p->post) | reinterpret_cast<uintptr_t>(p->post_bias) |
                        reinterpret_cast<uintptr_t>(p->gate) | reinterpret_cast<uintptr_t>(p->pre) |
                        reinterpret_cast<uintptr_t>(p->pre_bias) | reinterpret_cast<uintptr_t>(p->residual_out) |
                        reinterpret_cast<uintptr_t>(p->h);
  if (all & 15u) return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: arrays must be 16-byte aligned");
  if (norm_overlap(p))
    return fail(QGEMM_ERR_INVALID_ARG, "residual_norm: outputs overlap each other, or an input at other places or of another type");
  NormArgs a;
  a.y = p->y; a.residual = p->residual; a.post = p->post; a.post_bias = p->post_bias; a.gate = p->gate;
  a.gate_stride = p->gate_stride; a.pre = p->pre; a.pre_bias = p->pre_bias; a.alpha = p->alpha; a.eps = p->eps;
  a.residual_out = p->residual_out; a.h = p->h; a.tokens = p->tokens; a.width = p->width;
  a.inv_width = 1.0f / (float)p->width;
  const int nv = p->width / 8;
  a.nv = nv;
  // Two vectors a thread: 49 us at 6000 x 2880 against 57 us with one, whose
  // reductions and addresses are paid twice as often.  Four (rows beyond 8192 in
  // 512 threads) would need 118 registers: 94 us at 1500 x 16384 against 91.
  const int V = nv <= 32 ? 1 : 2;
  a.row_warps = (nv + 32 * V - 1) / (32 * V);
  a.row_half = 0;
  while (2 * a.row_half < a.row_warps && a.row_warps > 1) a.row_half = a.row_half ? 2 * a.row_half : 1;
  const unsigned row_threads = 32u * a.row_warps;
  const unsigned rows = row_threads >= 256 ? 1 : 256 / row_threads;
  const unsigned grid = ((unsigned)p->tokens + rows - 1) / rows;
  cudaStream_t s = as_stream(stream);
  const bool layer = p->kind == QGEMM_NORM_LAYER, f32 = p->residual_f32 != 0;
  cudaError_t e = cudaSuccess;
#define QG_NORM(V_)                                                       \
  case V_:                                                                \
    e = layer ? launch_norm<V_, true>(a, f32, grid, rows * row_threads, s)  \
              : launch_norm<V_, false>(a, f32, grid, rows * row_threads, s); \
    break;
  switch (V) { QG_NORM(1) QG_NORM(2) }
#undef QG_NORM
  QG_CUDA_RET(e);
  return QGEMM_OK;
}

}  // extern "C"
