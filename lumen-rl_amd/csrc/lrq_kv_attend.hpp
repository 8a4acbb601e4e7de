// What the attention kernels on an FP8 KV cache share (lrq_kv_attend.hip has the formulas).
#pragma once

#include "lrq_kv.hpp"

namespace lrq {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kUnit = 64;         // keys that are taken at a time
constexpr float kLow = -3.0e38f;  // a maximum before the first key
constexpr float kLn2 = 0.69314718056f;
constexpr float kLift = 10.0f;    // log2 of what p is multiplied with

// Two e4m3 codes of a word, exactly, in the type of the queries (bf16 or fp16).
template <int DT, bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
  if constexpr (DT == kBF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}
template <int DT>
__device__ __forceinline__ v4u widen8(uint32_t a, uint32_t b) {
  return v4u{widen2<DT, false>(a), widen2<DT, true>(a), widen2<DT, false>(b), widen2<DT, true>(b)};
}
__device__ __forceinline__ uint32_t f16_pair(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
}

// Bytes of `w` that are NaN codes, as 0x80 in each.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
// The first `n` bytes of a word (n any number).
__device__ __forceinline__ uint32_t low_bytes(int n) { return n <= 0 ? 0u : n >= 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u; }

// Four results, rounded to their type.
template <int DT>
__device__ __forceinline__ void store4(void* out, int64_t at, f32x4 v) {
  uint16_t* const p = static_cast<uint16_t*>(out) + at;
  v2u w;
  if constexpr (DT == kBF16) {
    w = v2u{bf16x2_bits(v.x, v.y), bf16x2_bits(v.z, v.w)};
  } else {
    w = v2u{f16_pair(v.x, v.y), f16_pair(v.z, v.w)};
  }
  gst<v2u>(p, w);
}

}  // namespace lrq
