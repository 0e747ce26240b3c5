// Attention over an 8-bit cache: what its kernels share.  q8_attention.cu has the one for few rows and the entry point, q8_prompt.cu the one for many.
#pragma once
#include "q8.cuh"

namespace blr {

struct Q8AttnParams {
  Q8View c;
  const uint16_t* q;
  uint16_t* out;
  long long ldq, ldo;
  const long long *start, *n_new;
  float* part;       // ns > 1: of each (sequence, kv head, row, split) hd sums, the maximum that they are taken against, the sum of the weights, 2 free
  uint8_t* wide;     // NULL, or room for the codes as fp16: of each (sequence, kv head, 128 slots) a tile of keys and one of values
  unsigned* status;  // NULL, or where a wait that gave up is noted
  float scale_log2;
  int T, H, G, rows, q_tiles, ns, bf16, n_bh, n_seq;
  int room, wide_tiles;  // CTAs that the SMs hold; tiles of a head
};

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Slots that a row of token t sees.
__device__ __forceinline__ int q8_seen(long long start, long long count, long long t, int slots) {
  if (t >= count) return 0;
  const long long n = start + t + 1;
  return n <= 0 ? 0 : n > slots ? slots : (int)n;
}
// The slots that the last of rows [r0, r1) of a kv head sees: 0 where none of them is a token.
__device__ __forceinline__ int q8_seen_by(const Q8AttnParams& p, long long start, long long count, int r0, int r1) {
  r1 = min(r1, p.rows);
  if (r0 >= r1 || r0 / p.G >= count) return 0;
  return q8_seen(start, count, min((long long)((r1 - 1) / p.G), count - 1), p.c.slots);
}
// The power of two that brings a bf16 row whose largest value has these bits to 2^14, in fp16's range, as an exponent (127: 1); fp16 rows stay as they are.
__device__ __forceinline__ int q8_row_up(uint32_t most, int bf16) {
  const int ex = (int)(most >> 23);
  return bf16 && ex != 0 && ex != 255 ? min(268 - ex, 253) : 127;
}


// A row's weights are taken against two references of its own: p = 2^(s - m), and P = p vs D, rounded to fp16, for the product with the codes, so that O = D sum p v.
// m is a whole number, the largest score rounded up when it was last moved; D = 2^-d brings the largest p vs to between 2^2 and 2^4 when it is moved.  Both are moved
// where the row's own keys ask for it, so that what it does not see has no part in any of its bits, and both by powers of two, so that nothing but P is rounded:
// a weight loses 2^-11 of itself, or 2^-27 of the row's heaviest where it is next to nothing beside that one.
static constexpr float kQ8Lift = 4.f;
// A whole number above log2 of a block's scale; -inf where it is 0 (or next to it) or no number: such a block moves nothing.
__device__ __forceinline__ float q8_above(float scale) {
  const uint32_t e = (__float_as_uint(scale) >> 23) & 0xff;
  return e == 0 || e == 255 ? -INFINITY : (float)e - 126.f;
}
__device__ __forceinline__ float q8_exponent(float D) { return 127.f - (float)(int)(__float_as_uint(D) >> 23); }  // d
__device__ __forceinline__ float q8_unit(float D) { return __uint_as_float((254u << 23) - __float_as_uint(D)); }                  // 2^d
// To m = `to`, the heaviest of the new keys at 2^heavy against it.  l is to be multiplied with `down`, O with `corr`.
__device__ __forceinline__ void q8_move(float to, float heavy, float& m, float& D, float& down, float& corr) {
  const float keep = q8_exponent(D) + (m - to), next = fmaxf(fmaxf(keep, heavy - kQ8Lift), -126.f);
  down = ex2(m - to), corr = ex2(keep - next);
  m = to;
  D = __uint_as_float((uint32_t)(127 - (int)next) << 23);
}

int q8_launch_prompt(const Q8AttnParams& p, int head_dim, int code, cudaStream_t stream);
static constexpr int kQ8PromptRows = 256;  // rows of a CTA

}  // namespace blr
