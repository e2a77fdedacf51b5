// kv.cuh -- the paged 8-bit KV cache: argument checks, code conversions and
// exponent helpers shared by the plan, append and attention kernels.
//
// A block holds `block` consecutive tokens of one request for every KV head:
// codes [blocks][heads][block][head_dim] (E4M3 or INT8) and one E8M0 scale
// byte per (block, head), 2^(byte - 127).  Scales are powers of two so that a
// block whose scale grows when tokens arrive rescales its older codes exactly
// (E4M3, down to its subnormals) or with a total error below one step (INT8),
// and so that a scale is an exponent the attention kernels add, not multiply.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace qg {

constexpr int kKvLowestExp = -64;  // smallest scale written: 2^-64
constexpr int kKvMaxTokens = 1 << 30;

inline bool kv_block_ok(int32_t block) { return block == 16 || block == 32 || block == 64 || block == 128; }

// Null if the cache description can be used, else a message.
inline const char* kv_cache_error(const qgemm_kv_cache_t* c) {
  if (!c) return "null cache";
  if (c->type != QGEMM_KV_E4M3 && c->type != QGEMM_KV_INT8) return "unknown cache type";
  if (!kv_block_ok(c->block)) return "block must be 16, 32, 64 or 128 tokens";
  if (c->head_dim != 64 && c->head_dim != 128) return "head_dim must be 64 or 128";
  if (c->heads < 1 || c->heads > 65535) return "heads must be 1 .. 65535";
  if (c->blocks < 1 || c->blocks > INT32_MAX) return "blocks must be 1 .. 2^31 - 1";
  if (!c->k || !c->v || !c->k_scales || !c->v_scales) return "null cache pointer";
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15u)
    return "cache codes must be 16-byte aligned";
  return nullptr;
}

// 2^e as a float for -126 <= e <= 127.
__device__ __forceinline__ float pow2f(int e) { return u2f((uint32_t)(e + 127) << 23); }

// Two E4M3 codes (low 16 bits) -> f16x2, exact (NaN code -> NaN).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v) {
  uint32_t d;
  asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.rn.f16x2.e4m3x2 %0, lo; }" : "=r"(d) : "r"(v));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t v) {
  uint32_t d;
  asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.rn.f16x2.e4m3x2 %0, hi; }" : "=r"(d) : "r"(v));
  return d;
}
// Four codes of one type -> f16x2 pairs (c0, c1), (c2, c3), exact.  INT8: the
// byte c + 128 in the mantissa of f16 1024 is 1024 + 128 + c.
template <int TYPE>
__device__ __forceinline__ void codes4_to_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  if constexpr (TYPE == QGEMM_KV_E4M3) {
    lo = e4m3x2_to_f16x2(v);
    hi = e4m3x2_hi_to_f16x2(v);
  } else {
    const uint32_t u = v ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
  }
}

// x (already divided by the scale) to a code: nearest, ties to even,
// saturating at the largest code; NaN becomes 0, so the cache holds finite
// numbers only and a masked token can never reach a row it is masked from.
template <int TYPE>
__device__ __forceinline__ uint32_t kv_encode(float x) {
  if (x != x) x = 0.0f;
  if constexpr (TYPE == QGEMM_KV_E4M3) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(0.0f), "f"(x));
    return d & 0xFFu;
  } else {
    return (uint32_t)(__float2int_rn(fminf(fmaxf(x, -127.0f), 127.0f)) & 0xFF);
  }
}
template <int TYPE>
__device__ __forceinline__ float kv_decode(uint32_t code) {
  if constexpr (TYPE == QGEMM_KV_E4M3) return e4m3_decode(code);
  return (float)(int8_t)(code & 0xFFu);
}
// The smallest e with amax <= largest code * 2^e, at least kKvLowestExp.
// amax = 1.f * 2^x: E4M3's largest code is 1.75 * 2^8, INT8's 1.984375 * 2^6.
template <int TYPE>
__device__ __forceinline__ int kv_exp_for(float amax) {
  const uint32_t u = f2u(amax), frac = u & 0x7FFFFFu;
  const int x = (int)(u >> 23) - 127;  // subnormals and zero fall to the lowest exponent
  const int e = TYPE == QGEMM_KV_E4M3 ? x - 8 + (frac > 0x600000u) : x - 6 + (frac > 0x7E0000u);
  return e < kKvLowestExp ? kKvLowestExp : e;
}

}  // namespace qg
