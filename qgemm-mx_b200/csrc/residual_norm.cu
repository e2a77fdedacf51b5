// residual_norm.cu -- the norms before and after a decoder block in one pass:
//   r' = r + alpha * gate * N(y; post)      h = N(r'; pre)
// (no counterpart in titoatwork/qgemm-mx).  N is RMSNorm, or LayerNorm as
// mean, then mean square of the centred values.
//
// What bounds it: HBM for many rows, latency for few.  A row lives in
// registers from its one read to its one write: threads load all of y, the
// residual and the gate before the first reduction, so a row costs one trip
// to memory and two (RMS) or four (LayerNorm) reductions in shared memory.
// All sums are 32-bit floats; r' is rounded once, for its store, and h is the
// norm of the unrounded r'.
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
  int row_warps;  // warps per row
};

__device__ __forceinline__ void unpack8(const uint4& w, float (&f)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = u2f(u[i] << 16);
    f[2 * i + 1] = u2f(u[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    u[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ uint4 vec_at(const uint16_t* p, int v) { return __ldg(reinterpret_cast<const uint4*>(p) + v); }

// Sum over the row's warps; every thread of the row gets it.  buf: one float
// per warp of the CTA, a fresh one for each reduction of a row.
__device__ __forceinline__ float row_sum(float x, float* buf, int row_warps) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
  if (row_warps == 1) return x;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) buf[warp] = x;
  __syncthreads();
  const int first = warp / row_warps * row_warps;
  x = 0.0f;
  for (int w = 0; w < row_warps; ++w) x += buf[first + w];
  return x;
}

// x <- N(x) in place.  V vectors of 8 values per thread, `live` ones real.
template <int V, bool LAYER>
__device__ __forceinline__ void normalise(float (&x)[V][8], const uint16_t* weight, const uint16_t* bias, int v0,
                                          int step, int nv, float inv_width, float eps, float* buf, int row_warps) {
  if (LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += x[j][i];
    const float mean = row_sum(s, buf, row_warps) * inv_width;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (v0 + j * step < nv) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] -= mean;
      }
  }
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[j][i] * x[j][i];
  const float rs = rsqrtf(row_sum(ss, buf + 32, row_warps) * inv_width + eps);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int v = v0 + j * step;
    if (v < nv) {
      float w[8];
      unpack8(vec_at(weight, v), w);
      if (LAYER && bias) {
        float b[8];
        unpack8(vec_at(bias, v), b);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = x[j][i] * rs * w[i] + b[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = x[j][i] * rs * w[i];
      }
    }
  }
}

template <int V, bool LAYER, bool F32>
__global__ void __launch_bounds__(512) k_residual_norm(const NormArgs a) {
  __shared__ float s_buf[128];
  const int row_threads = a.row_warps * 32;
  const int rows = blockDim.x / row_threads;  // rows per CTA
  const int v0 = threadIdx.x % row_threads, nv = a.width / 8;
  const int row_raw = blockIdx.x * rows + threadIdx.x / row_threads;
  const bool live = row_raw < a.tokens;
  const int64_t row = live ? row_raw : a.tokens - 1;  // spare rows recompute the last one and store nothing
  const float inv_width = 1.0f / (float)a.width;
  pdl_begin();
  float r[V][8], x[V][8];
  uint4 g[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int v = v0 + j * row_threads;
    const bool on = v < nv;
    if (F32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.residual) + row * a.width) + 2 * v;
      const float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const float4 lo = on ? p[0] : z, hi = on ? p[1] : z;
      r[j][0] = lo.x; r[j][1] = lo.y; r[j][2] = lo.z; r[j][3] = lo.w;
      r[j][4] = hi.x; r[j][5] = hi.y; r[j][6] = hi.z; r[j][7] = hi.w;
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
    if (a.post)
      normalise<V, LAYER>(x, a.post, a.post_bias, v0, row_threads, nv, inv_width, a.eps, s_buf, a.row_warps);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int v = v0 + j * row_threads;
      if (a.gate) {
        float f[8];
        unpack8(g[j], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] *= f[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) r[j][i] += a.alpha * x[j][i];
      if (live && v < nv) {
        if (F32) {
          float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.residual_out) + row * a.width) + 2 * v;
          p[0] = make_float4(r[j][0], r[j][1], r[j][2], r[j][3]);
          p[1] = make_float4(r[j][4], r[j][5], r[j][6], r[j][7]);
        } else {
          reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.residual_out) + row * a.width)[v] = pack8(r[j]);
        }
      }
    }
  }
  if (a.pre) {
    normalise<V, LAYER>(r, a.pre, a.pre_bias, v0, row_threads, nv, inv_width, a.eps, s_buf + 64, a.row_warps);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int v = v0 + j * row_threads;
      if (live && v < nv) reinterpret_cast<uint4*>(a.h + row * a.width)[v] = pack8(r[j]);
    }
  }
}

template <int V, bool LAYER>
static cudaError_t launch_norm(const NormArgs& a, bool f32, unsigned grid, unsigned threads, cudaStream_t s) {
  return pdl_launch(f32 ? k_residual_norm<V, LAYER, true> : k_residual_norm<V, LAYER, false>, dim3(grid), dim3(threads), 0,
                    s, a);
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
  NormArgs a;
  a.y = p->y; a.residual = p->residual; a.post = p->post; a.post_bias = p->post_bias; a.gate = p->gate;
  a.gate_stride = p->gate_stride; a.pre = p->pre; a.pre_bias = p->pre_bias; a.alpha = p->alpha; a.eps = p->eps;
  a.residual_out = p->residual_out; a.h = p->h; a.tokens = p->tokens; a.width = p->width;
  const int nv = p->width / 8;
  const int V = nv <= 32 ? 1 : nv <= 1024 ? 2 : 4;
  a.row_warps = (nv + 32 * V - 1) / (32 * V);
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
  switch (V) { QG_NORM(1) QG_NORM(2) QG_NORM(4) }
#undef QG_NORM
  QG_CUDA_RET(e);
  return QGEMM_OK;
}

}  // extern "C"
