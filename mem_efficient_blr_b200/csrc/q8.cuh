// What the kernels around an 8-bit key / value cache share: its layout, and its codes as 16- and 32-bit floats.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/blr_b200.h"
#include "ptx.cuh"
#include "tmap.h"

namespace blr {

// Codes (n_seq, kv_heads, slots, hd), one fp32 scale per `block` slots of a head: value = code * scale.
struct Q8View {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  int kv_heads, slots, block_log2, n_blocks;
};

// Codes are int8 in [-127, 127], or e4m3 in [-448, 448].
template <bool E4M3>
__device__ __forceinline__ float q8_top() { return E4M3 ? 448.f : 127.f; }

// Two codes in the low (high) half of a word -> the same numbers as a pair of halves.  Exact for both kinds.
template <bool E4M3>
__device__ __forceinline__ uint32_t q8_half2(uint32_t w, bool high) {
  if constexpr (E4M3) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, %2;\n\t}" : "=r"(r) : "r"(w), "h"((uint16_t)(high ? w >> 16 : w)));
    return r;
  } else {
    return cvt_u8pair<false>(w, high);  // (w biased by 128: q8_bias)
  }
}
template <bool E4M3>
__device__ __forceinline__ uint32_t q8_bias(uint32_t w) { return E4M3 ? w : w ^ 0x80808080u; }

// Four codes of a word as floats.
template <bool E4M3>
__device__ __forceinline__ void q8_floats(uint32_t w, float (&f)[4]) {
  const uint32_t b = q8_bias<E4M3>(w), lo = q8_half2<E4M3>(b, false), hi = q8_half2<E4M3>(b, true);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo)), y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  f[0] = x.x, f[1] = x.y, f[2] = y.x, f[3] = y.y;
}
// Four numbers in a code's range (or beyond it by less than half a step) as codes, to nearest even.
template <bool E4M3>
__device__ __forceinline__ uint32_t q8_codes(const float (&f)[4]) {
  if constexpr (E4M3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(f[0]), "f"(f[1]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(f[2]), "f"(f[3]));
    return (uint32_t)lo | (uint32_t)hi << 16;
  } else {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // 1.5 * 2^23 + x is rounded to a whole number, whose last byte is x's
      b[i] = __float_as_uint(__fadd_rn(f[i], 12582912.f));
    return prmt(prmt(b[0], b[1], 0x0040u), prmt(b[2], b[3], 0x0040u), 0x5410u);
  }
}

template <bool BF16>
__device__ __forceinline__ float2 q8_up2(uint32_t w) {
  if constexpr (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t q8_down2(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two floats of one 64-bit register: one instruction for both.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// ---- host side
// A launch that may begin while the kernel ahead of it ends (every kernel here waits before it looks at anything).
template <typename K, typename... A>
static int q8_launch(K kernel, dim3 grid, int threads, int smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  BLR_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, args...));
  return BLR_OK;
}
int q8_view(const blr_q8_cache* cache, Q8View* out);  // checks the cache's description

}  // namespace blr
