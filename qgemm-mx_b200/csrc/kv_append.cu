// kv_append.cu -- quantises a step's K and V rows into their slots of the
// paged 8-bit cache (no counterpart in titoatwork/qgemm-mx).
//
// An item is one run of rows that share a block, for one head, of K or V.
// With off tokens already in the block and e_old its scale's exponent:
//   e = max(e_old if off > 0, min { e : max|x| <= qmax 2^e })
//   old codes:  rne(c 2^(e_old - e)), only when e > e_old
//   new codes:  rne(x 2^-e)
// so one pass: a thread group loads its rows once into registers, reduces the
// maximum, and writes the codes; 2 bytes read and 1 written per value.
//
// What bounds it: HBM for prompts, latency for a decode step (runs -> slot ->
// rows and scale -> codes).  A group is one warp where runs are short (a
// decode step's run is one row, 256 B of K) and 256 threads where a run fills
// a block.
#include "kv.cuh"

namespace qg {

constexpr int kAppendThreads = 256;
struct AppendArgs {
  uint8_t *k, *v, *ks, *vs;
  const uint16_t *xk, *xv;
  int64_t k_stride, k_head_stride, v_stride, v_head_stride;
  const int64_t* slots;
  const int32_t* runs;
  int64_t blocks;
  int heads, block_log2, tokens;
  unsigned items;
};

// |x| of bf16 pairs as bits: the larger of each half.
__device__ __forceinline__ uint32_t amax2(uint32_t w, uint32_t m) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(w & 0x7FFF7FFFu), "r"(m));
  return d;
}
// Largest finite |x| of two bf16 values, where infinities or NaN occur.
__device__ __forceinline__ uint32_t amax_finite(uint32_t w, uint32_t m) {
  const uint32_t lo = w & 0x7FFFu, hi = (w >> 16) & 0x7FFFu;
  if (lo < 0x7F80u) m = max(m, lo);
  if (hi < 0x7F80u) m = max(m, hi);
  return m;
}
// Four bf16 values times f to codes.  FINITE: none is infinite or NaN, and the scale
// keeps them in range, so only rounding is left.
template <int TYPE, bool FINITE>
__device__ __forceinline__ uint32_t encode4(uint32_t w0, uint32_t w1, float f) {
  const float x0 = u2f(w0 << 16) * f, x1 = u2f(w0 & 0xFFFF0000u) * f;
  const float x2 = u2f(w1 << 16) * f, x3 = u2f(w1 & 0xFFFF0000u) * f;
  if (!FINITE)
    return kv_encode<TYPE>(x0) | (kv_encode<TYPE>(x1) << 8) | (kv_encode<TYPE>(x2) << 16) | (kv_encode<TYPE>(x3) << 24);
  if (TYPE == QGEMM_KV_E4M3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x1), "f"(x0));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x3), "f"(x2));
    return (uint32_t)lo | ((uint32_t)hi << 16);
  }
  uint32_t d;  // bytes 0, 1 of the second packing, then 2, 3
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(__float2int_rn(x3)), "r"(__float2int_rn(x2)), "r"(0));
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(__float2int_rn(x1)), "r"(__float2int_rn(x0)), "r"(d));
  return d;
}

// HELD: 16-byte vectors a thread keeps in registers.
template <int TYPE, int HD, int GT, int HELD>
__global__ void __launch_bounds__(kAppendThreads) k_kv_append(const AppendArgs a) {
  constexpr int VPR = HD / 8;  // 16-byte vectors in a row
  __shared__ uint32_t s_max[kAppendThreads / 32];
  const int gl = threadIdx.x % GT;  // place in the group
  const unsigned item = blockIdx.x * (kAppendThreads / GT) + threadIdx.x / GT;
  pdl_begin();
  if (item >= a.items) return;  // whole groups
  const unsigned run = item / (2u * a.heads), rest = item - run * 2u * a.heads;
  const int which = rest >= (unsigned)a.heads, h = (int)rest - (which ? a.heads : 0);
  const int P = 1 << a.block_log2;
  const int t0 = a.runs[run], tend = a.runs[run + 1];
  if (t0 < 0 || t0 >= a.tokens || tend <= t0) return;
  const int64_t slot = a.slots[t0];
  const int64_t blk = slot >> a.block_log2;
  if (slot < 0 || blk >= a.blocks) return;
  const int off = (int)(slot & (P - 1));
  const int n = min(min(tend, a.tokens) - t0, P - off);
  const int nv = n * VPR;
  const int64_t stride = which ? a.v_stride : a.k_stride;
  const uint16_t* x = (which ? a.xv : a.xk) + (int64_t)t0 * stride + (int64_t)h * (which ? a.v_head_stride : a.k_head_stride);
  auto src = [&](int v) { return reinterpret_cast<const uint4*>(x + (int64_t)(v / VPR) * stride + (v % VPR) * 8); };
  const size_t cell = (size_t)blk * a.heads + h;
  uint8_t* codes = (which ? a.v : a.k) + cell * (size_t)(P * HD);
  uint8_t* scale = (which ? a.vs : a.ks) + cell;
  const int e_old = off > 0 ? (int)*scale - 127 : kKvLowestExp;

  uint4 held[HELD];
  uint32_t m2 = 0;
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    const int v = gl + j * GT;
    held[j] = v < nv ? ld16(src(v)) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < HELD; ++j)
    m2 = amax2(held[j].x, amax2(held[j].y, amax2(held[j].z, amax2(held[j].w, m2))));
#pragma unroll 1
  for (int v = gl + HELD * GT; v < nv; v += GT) {  // only a warp's long runs; read again below
    const uint4 w = ld16(src(v));
    m2 = amax2(w.x, amax2(w.y, amax2(w.z, amax2(w.w, m2))));
  }
  auto group_max = [&](uint32_t m) {
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if constexpr (GT > 32) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < GT / 32; ++w) m = max(m, s_max[w]);
    }
    return m;
  };
  uint32_t m = group_max(max(m2 & 0xFFFFu, m2 >> 16));
  const bool finite = m < 0x7F80u;  // of the whole group
  if (!finite) {
    m = 0;
#pragma unroll 1
    for (int v = gl; v < nv; v += GT) {
      const uint4 w = ld16(src(v));
      m = amax_finite(w.x, amax_finite(w.y, amax_finite(w.z, amax_finite(w.w, m))));
    }
    m = group_max(m);
  }
  const int e = max(e_old, kv_exp_for<TYPE>(u2f(m << 16)));
  if (off > 0 && e > e_old) {  // the block's scale grows: rescale the codes it holds
    const float f = pow2f(max(e_old - e, -126));
    uint32_t* old = reinterpret_cast<uint32_t*>(codes);
    for (int i = gl; i < off * HD / 4; i += GT) {
      const uint32_t w = old[i];
      uint32_t r = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) r |= kv_encode<TYPE>(kv_decode<TYPE>((w >> (8 * b)) & 0xFFu) * f) << (8 * b);
      old[i] = r;
    }
  }
  const float f = pow2f(-e);
  uint8_t* dst = codes + off * HD;
  if (finite) {
    auto put = [&](int v, const uint4& w) {
      *reinterpret_cast<uint2*>(dst + v * 8) =
          make_uint2(encode4<TYPE, true>(w.x, w.y, f), encode4<TYPE, true>(w.z, w.w, f));
    };
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const int v = gl + j * GT;
      if (v < nv) put(v, held[j]);
    }
#pragma unroll 1
    for (int v = gl + HELD * GT; v < nv; v += GT) put(v, ld16(src(v)));
  } else {
#pragma unroll 1
    for (int v = gl; v < nv; v += GT) {
      const uint4 w = ld16(src(v));
      *reinterpret_cast<uint2*>(dst + v * 8) =
          make_uint2(encode4<TYPE, false>(w.x, w.y, f), encode4<TYPE, false>(w.z, w.w, f));
    }
  }
  if (gl == 0) *scale = (uint8_t)(e + 127);
}

template <int TYPE, int HD>
static cudaError_t launch_append(const AppendArgs& a, int vectors, cudaStream_t s) {
  const bool wide = vectors > 8 * 32;
  const unsigned per = wide ? 1 : kAppendThreads / 32;
  const unsigned grid = (a.items + per - 1) / per;
  auto kernel = !wide ? (vectors > 2 * 32 ? k_kv_append<TYPE, HD, 32, 8> : k_kv_append<TYPE, HD, 32, 2>)
                      : (vectors > 4 * kAppendThreads ? k_kv_append<TYPE, HD, kAppendThreads, 8>
                                                      : k_kv_append<TYPE, HD, kAppendThreads, 4>);
  return pdl_launch(kernel, dim3(grid), dim3(kAppendThreads), 0, s, a);
}

}  // namespace qg

using namespace qg;

extern "C" {

qgemm_status_t qgemm_kv_append(const qgemm_kv_cache_t* c, const uint16_t* k, const uint16_t* v, int64_t k_stride,
                               int64_t k_head_stride, int64_t v_stride, int64_t v_head_stride, int32_t tokens,
                               const int64_t* slots, const int32_t* runs, int32_t max_runs, void* stream) {
  if (const char* e = kv_cache_error(c)) return fail(QGEMM_ERR_INVALID_ARG, "kv_append: %s", e);
  if (tokens < 0 || tokens >= kKvMaxTokens || max_runs < 0)
    return fail(QGEMM_ERR_INVALID_ARG, "kv_append: bad row or run count");
  if (tokens == 0 || max_runs == 0) return QGEMM_OK;
  if (!k || !v || !slots || !runs) return fail(QGEMM_ERR_INVALID_ARG, "kv_append: null pointer");
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u)
    return fail(QGEMM_ERR_INVALID_ARG, "kv_append: k and v must be 16-byte aligned");
  if (k_stride % 8 || v_stride % 8 || k_head_stride % 8 || v_head_stride % 8)
    return fail(QGEMM_ERR_INVALID_ARG, "kv_append: strides must be multiples of 8");
  const long long items = 2ll * c->heads * max_runs;
  if (items > INT32_MAX) return fail(QGEMM_ERR_UNSUPPORTED_SHAPE, "kv_append: more than 2^31 - 1 items");
  AppendArgs a;
  a.k = c->k; a.v = c->v; a.ks = c->k_scales; a.vs = c->v_scales;
  a.xk = k; a.xv = v; a.k_stride = k_stride; a.v_stride = v_stride;
  a.k_head_stride = k_head_stride; a.v_head_stride = v_head_stride;
  a.slots = slots; a.runs = runs; a.blocks = c->blocks; a.heads = c->heads; a.tokens = tokens;
  a.block_log2 = c->block == 16 ? 4 : c->block == 32 ? 5 : c->block == 64 ? 6 : 7;
  a.items = (unsigned)items;
  // 16-byte vectors of the usual run: they choose the threads of an item and what
  // each keeps in registers, so that a run is read once
  const int rows = (tokens + max_runs - 1) / max_runs;
  const int wide = (rows < c->block ? rows : c->block) * c->head_dim / 8;
  cudaStream_t s = as_stream(stream);
  const bool d64 = c->head_dim == 64;
  QG_CUDA_RET(c->type == QGEMM_KV_E4M3
                  ? (d64 ? launch_append<QGEMM_KV_E4M3, 64>(a, wide, s) : launch_append<QGEMM_KV_E4M3, 128>(a, wide, s))
                  : (d64 ? launch_append<QGEMM_KV_INT8, 64>(a, wide, s) : launch_append<QGEMM_KV_INT8, 128>(a, wide, s)));
  return QGEMM_OK;
}

}  // extern "C"
