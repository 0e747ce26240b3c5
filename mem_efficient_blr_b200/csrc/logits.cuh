// Rows of logits: their values, and the order that they are in.
#pragma once
#include "q8.cuh"

namespace blr {

// Whole numbers in the order of the values; 0 is below all of them, and 0xffffffff, with which a search begins, above: a NaN, which comes first, is one less.
static constexpr uint32_t kOrderOfNan = 0xfffffffeu;
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? kOrderOfNan : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o == kOrderOfNan ? 0x7fffffffu : o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// The largest number below the one of order o.  (0x7fffffff is the order of none: it lies between 0 and the number below it, and would be -0, which equals 0.)
__device__ __forceinline__ float value_below(uint32_t o) { return value_of(o == 0x80000000u ? 0x7ffffffeu : o - 1); }

// 16 bytes of logits: kPer values.
template <int KIND>
struct Vec {
  static constexpr int kPer = KIND == 2 ? 4 : 8;
  // their running maximum (16-bit values: of the odd and the even ones), a NaN before anything else
  __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (KIND == 0) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else if constexpr (KIND == 1) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ static uint32_t largest(const uint4& w) { return larger(larger(w.x, w.y), larger(w.z, w.w)); }
  static constexpr uint32_t kLowest = KIND == 0 ? 0xfc00fc00u : KIND == 1 ? 0xff80ff80u : 0xff800000u;  // -inf
  __device__ __forceinline__ static float most(uint32_t m) {
    if constexpr (KIND == 2) return __uint_as_float(m);
    else return [](float2 v) { return v.x != v.x || v.x > v.y ? v.x : v.y; }(q8_up2<KIND == 1>(m));
  }
  __device__ __forceinline__ static float value(const uint4& w, int i) {
    const uint32_t u = i < kPer / 2 ? i < kPer / 4 ? w.x : w.y : i < 3 * kPer / 4 ? w.z : w.w;
    if constexpr (KIND == 2) return __uint_as_float(u);
    else return [&](float2 v) { return i & 1 ? v.y : v.x; }(q8_up2<KIND == 1>(u));
  }
  __device__ __forceinline__ static void floats(const uint4& w, float (&f)[kPer]) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (KIND == 2) {
        f[i] = __uint_as_float(ws[i]);
      } else {
        const float2 v = q8_up2<KIND == 1>(ws[i]);
        f[2 * i] = v.x, f[2 * i + 1] = v.y;
      }
    }
  }
};
template <int KIND>
__device__ __forceinline__ float logit(const void* row, long long i) {
  if constexpr (KIND == 0) return __half2float(static_cast<const __half*>(row)[i]);
  else if constexpr (KIND == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]);
  else return static_cast<const float*>(row)[i];
}

}  // namespace blr
