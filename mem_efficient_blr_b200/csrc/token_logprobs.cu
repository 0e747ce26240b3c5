// Log probabilities of given tokens, entropy and likeliest tokens of rows of logits.
//   M = max x,  S = sum e^(x - M),  log p(i) = (x_i - M) - log S,  H = log S - (sum e^(x - M) (x - M)) / S
// Sums are fp32.  Order of the likeliest: falling value (NaN above everything, -0 equal to 0), ties by rising id.
#include <math_constants.h>

#include "../../include/blr_b200.h"
#include "q8.cuh"
#include "tmap.h"

namespace blr {

static constexpr int kLpThreads = 256, kLpMaxTop = 64;

template <int KIND>
__device__ __forceinline__ float logit(const void* row, long long i) {
  if constexpr (KIND == 0) return __half2float(static_cast<const __half*>(row)[i]);
  else if constexpr (KIND == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]);
  else return static_cast<const float*>(row)[i];
}
// Whole numbers in the order of the values; 0 is below all of them.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o == 0xffffffffu ? 0x7fffffffu : o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

template <int KIND>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const void* logits, long long ld, int vocab, const long long* ids, int top,
                                                                    float* logprob, float* entropy, float* top_lp, long long* top_ids) {
  __shared__ unsigned long long red[kLpThreads / 32];
  __shared__ float sums[2][kLpThreads / 32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long r = blockIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const void* row = static_cast<const char*>(logits) + r * ld * (KIND == 2 ? 4 : 2);
  // the largest of 64-bit numbers (order, ~id)
  auto most = [&](unsigned long long v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < kLpThreads / 32; ++w) v = max(v, red[w]);
    return v;
  };
  uint32_t best = 0;
  for (int i = tid; i < vocab; i += kLpThreads) best = max(best, order_of(logit<KIND>(row, i)));
  const float M = value_of((uint32_t)most(best));
  const bool finite = M <= 3.402823466e38f && M >= -3.402823466e38f;
  float S = 0.f, D = 0.f;
  for (int i = tid; finite && i < vocab; i += kLpThreads) {
    const float d = logit<KIND>(row, i) - M, e = __expf(d);
    S += e;
    if (e > 0.f) D = fmaf(e, d, D);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) S += __shfl_xor_sync(0xffffffffu, S, d), D += __shfl_xor_sync(0xffffffffu, D, d);
  if (lane == 0) sums[0][warp] = S, sums[1][warp] = D;
  __syncthreads();
  S = D = 0.f;
  for (int w = 0; w < kLpThreads / 32; ++w) S += sums[0][w], D += sums[1][w];
  const float log_s = logf(S);
  // (a row of -inf alone: every log probability -inf, entropy 0; a NaN or +inf: NaN)
  const bool empty = M == -CUDART_INF_F;
  auto lp = [&](float x) { return finite ? (x - M) - log_s : empty ? -CUDART_INF_F : CUDART_NAN_F; };
  if (tid == 0) {
    const long long id = ids[r];
    logprob[r] = id < 0 ? 0.f : id >= vocab ? CUDART_NAN_F : lp(logit<KIND>(row, id));
    entropy[r] = finite ? log_s - D / S : empty ? 0.f : CUDART_NAN_F;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long v = 0;
    for (int i = tid; i < vocab; i += kLpThreads) {
      const unsigned long long c = (unsigned long long)order_of(logit<KIND>(row, i)) << 32 | (0xffffffffu - (uint32_t)i);
      if (c < last) v = max(v, c);
    }
    last = most(v);
    if (tid == 0) top_lp[r * top + k] = lp(value_of((uint32_t)(last >> 32))), top_ids[r * top + k] = 0xffffffffu - (uint32_t)last;
  }
}

template <typename K, typename... A>
static int launch(K kern, dim3 grid, dim3 block, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  BLR_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, args...));
  return BLR_OK;
}

}  // namespace blr

using namespace blr;

extern "C" {

int blr_token_logprobs(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int kind, const int64_t* ids, int top, float* logprob,
                       float* entropy, float* top_logprob, int64_t* top_ids, void* stream) {
  BLR_REQUIRE(kind >= 0 && kind <= 2, BLR_ERR_ARG, "unknown kind of logits %d", kind);
  BLR_REQUIRE(rows >= 0 && rows < (1ll << 31) && vocab > 0 && vocab < (1ll << 31) && (rows <= 1 || ld >= vocab), BLR_ERR_ARG,
              "token_logprobs: %lld rows of %lld", (long long)rows, (long long)vocab);
  BLR_REQUIRE(top >= 0 && top <= kLpMaxTop && top <= vocab, BLR_ERR_ARG, "token_logprobs gives 0 to %d tokens (and no more than there are), not %d", kLpMaxTop, top);
  if (rows == 0) return BLR_OK;
  BLR_REQUIRE(logits && ids && logprob && entropy && (top == 0 || (top_logprob && top_ids)), BLR_ERR_ARG, "null pointer");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel) {
    return launch(kernel, dim3((unsigned)rows), dim3(kLpThreads), st, logits, (long long)ld, (int)vocab, reinterpret_cast<const long long*>(ids), top, logprob,
                  entropy, top_logprob, reinterpret_cast<long long*>(top_ids));
  };
  return kind == 0 ? go(token_logprobs_kernel<0>) : kind == 1 ? go(token_logprobs_kernel<1>) : go(token_logprobs_kernel<2>);
}

}  // extern "C"
