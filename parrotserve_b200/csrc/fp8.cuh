// Conversions of the 8-bit cache: e4m3 codes with a power-of-two (or any other) fp32 scale per (block, head).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace pb {
namespace fp8 {

// The tensor-core kernels hold sums of 2^-lv with lv = log2 of the value scales, so these have bounds: below 2^kMinLv they count as 0 (the
// values are below 4e-28, the type's 2^-126 is out of reach of the sums), and from 2^100 on small weights are lost from the sums. (A unit
// chosen by an item's first blocks would lift both; its one vote among the listing warp's lanes cost the prefix kernel 3 %.)
constexpr float kMinLv = -100.f, kMinValueScale = 7.888609052210118e-31f;

// The shapes whose single queries go to the tcgen05 kernel (decode_fp8_tc.cu); the others go to single_query_fp8.cuh.
constexpr bool decode_on_tc(bool half_queries, int head_size, int block_size) {
  return half_queries && block_size == 16 && (head_size == 64 || head_size == 96 || head_size == 128);
}

// Two codes (the low 16 bits of `w`) as fp16, exactly: every e4m3 value, subnormals included, is a normal fp16 value.
__device__ __forceinline__ uint32_t to_half2(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
  return (uint32_t)h.x | ((uint32_t)h.y << 16);
}
__device__ __forceinline__ uint32_t to_half2_high(uint32_t w) { return to_half2(w >> 16); }
__device__ __forceinline__ float2 to_float2(uint32_t w) {
  const uint32_t h = to_half2(w);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// x * inv rounded to e4m3, to nearest even, saturating; NaN and infinities give NaN (e4m3 has no infinity).
__device__ __forceinline__ float scaled(float x, float inv) { return fabsf(x) <= 3.402823466e38f ? __fmul_rn(x, inv) : __int_as_float(0x7fc00000); }
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t pack2(__half2 v) {
  return (uint32_t)__nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(v), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) { return pack2(a, b) | (pack2(c, d) << 16); }

// The smallest power of two s with top <= 448 * s (448 = 1.75 * 2^8), from 2^-126 on; 0 for 0. top is finite, >= 0.
__device__ __forceinline__ float scale_for(float top) {
  if (!(top > 0.f)) return 0.f;
  const uint32_t bits = __float_as_uint(top);
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)(e < 1 ? 1 : e) << 23);
}

// The maximum m that a partial carries. Maxima drop NaN; a partial whose logits are all NaN would go to the merge with -inf, like one without
// tokens, and be left out. One whose sum l is NaN (a logit was) carries 0 then, and its NaN enters the sums whatever the others' maxima are.
__device__ __forceinline__ float told_max(float m, float l) { return l == l ? m : 0.f; }

__device__ __forceinline__ float pow2(float e) { return __uint_as_float((uint32_t)((int)e + 127) << 23); }  // whole e in [-126, 127]

// Maximum over a warp (NaN counts as nothing, like fmaxf).
__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

}  // namespace fp8
}  // namespace pb
