// The 8-bit key / value cache: e4m3 codes [B, Hkv, capacity, D] and one int8 exponent per head and block of tokens
// [B, Hkv, capacity / block]; a value is code * 2^exponent.  Power-of-two scales lose nothing with floating codes (the relative
// step of e4m3 does not depend on the scale), make every stored value exact in bf16 and let a block that has to grow its
// exponent re-encode the codes it holds.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace b200 {

// 448 * 2^119 is the largest value below the end of bf16; a block of tiny values keeps steps of 2^-49 at worst
constexpr int KV8_EMIN = -40, KV8_EMAX = 119;

__device__ __forceinline__ float pow2i(int e) { return __int_as_float((max(e, -126) + 127) << 23); }   // e <= 127

// The least exponent that brings `amax` (finite, > 0) to at most 448 = 0.875 * 2^9; as far as it is stored.
__device__ __forceinline__ int kv8_exponent_any(float amax) {
  const int bits = __float_as_int(amax);
  return (bits >> 23) - 126 - 9 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0);
}
__device__ __forceinline__ int kv8_exponent(float amax) {
  return amax > 0.f ? min(max(kv8_exponent_any(amax), KV8_EMIN), KV8_EMAX) : KV8_EMIN;
}
// Magnitude that counts for a block's exponent: infinities (stored as the largest code) and NaN (stored as NaN) do not.
__device__ __forceinline__ float kv8_mag(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}
// Four values -> four codes, to nearest, at most the largest code; `inv` = 2^-exponent.
__device__ __forceinline__ uint32_t kv8_encode4(float a, float b, float c, float d, float inv) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * inv, d * inv), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// Two codes -> f16x2 (exact); `hi`: the upper two of the word.
__device__ __forceinline__ uint32_t kv8_half2(uint32_t w, bool hi) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<unsigned short>(hi ? w >> 16 : w)));
  return h;
}
__device__ __forceinline__ float2 kv8_float2(uint32_t w, bool hi) {
  const uint32_t h = kv8_half2(w, hi);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Codes of four values under another exponent; `f` = 2^(old - new).
__device__ __forceinline__ uint32_t kv8_recode4(uint32_t w, float f) {
  const float2 a = kv8_float2(w, false), b = kv8_float2(w, true);
  return kv8_encode4(a.x, a.y, b.x, b.y, f);
}

}  // namespace b200
