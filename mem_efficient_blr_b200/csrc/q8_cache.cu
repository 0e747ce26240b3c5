// An 8-bit key / value cache: written as the rotary embedding makes the keys, and read back.
//
// A block of 16 to 128 slots of a head has one fp32 scale for its keys and one for its values.  Writing tokens into a block takes
//   s = max(s_before, max|x| (1 / top))  (top = 127 for int8, 448 for e4m3; s_before = 0 where the block begins with this call)
// and codes round(x (1 / s)); where s has grown, the codes that were there become round(code (s_before (1 / s))).  So a block's scale only ever grows while the
// block fills, a value is off by half a step of its block's final scale, and by half a step more for each time that the scale grew over it.  Nothing
// else of the cache is touched: codes behind a call's last token stay, although their block's scale may change, since a call ends its sequence there.
// All of it is fp32 with every product and sum rounded by itself (no fused multiply-add), so that the codes are a matter of the formula alone.
#include "../../include/blr_b200.h"
#include "q8.cuh"
#include "tmap.h"

namespace blr {

int q8_view(const blr_q8_cache* c, Q8View* out) {
  BLR_REQUIRE(c != nullptr, BLR_ERR_ARG, "null cache");
  BLR_REQUIRE(c->code == BLR_Q8_INT8 || c->code == BLR_Q8_E4M3, BLR_ERR_ARG, "unknown kind of codes %d", c->code);
  BLR_REQUIRE(c->n_seq >= 0 && c->kv_heads > 0 && c->slots > 0, BLR_ERR_ARG, "an 8-bit cache needs kv_heads and slots");
  BLR_REQUIRE(c->head_dim == 64 || c->head_dim == 128, BLR_ERR_UNSUPPORTED, "8-bit caches have heads of 64 or 128 values, got %d", c->head_dim);
  BLR_REQUIRE(c->block == 16 || c->block == 32 || c->block == 64 || c->block == 128, BLR_ERR_UNSUPPORTED,
              "an 8-bit cache has blocks of 16, 32, 64 or 128 slots, got %d", c->block);
  BLR_REQUIRE(c->n_seq * c->kv_heads < (1ll << 31), BLR_ERR_SHAPE, "too many sequences");
  if (c->n_seq > 0) {
    BLR_REQUIRE(c->k && c->v && c->k_scale && c->v_scale, BLR_ERR_ARG, "null pointer");
    BLR_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) == 0 &&
                    ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3) == 0,
                BLR_ERR_ARG, "an 8-bit cache needs 16-byte aligned codes and 4-byte aligned scales");
  }
  out->k = static_cast<uint8_t*>(c->k), out->v = static_cast<uint8_t*>(c->v);
  out->k_scale = c->k_scale, out->v_scale = c->v_scale;
  out->kv_heads = c->kv_heads, out->slots = c->slots;
  out->block_log2 = c->block == 16 ? 4 : c->block == 32 ? 5 : c->block == 64 ? 6 : 7;
  out->n_blocks = (c->slots + c->block - 1) >> out->block_log2;
  return BLR_OK;
}

struct AppendParams {
  Q8View c;
  const uint16_t *q, *k, *v;
  uint16_t* q_out;
  long long ldq, ldk, ldv, ldo;
  const float *cos_t, *sin_t;
  const long long *start, *n_new;
  uint32_t rows, units;  // units: blocks to look at, over sequences, heads, keys and values
  int T, H, blocks_per, q_heads, q_parts;
  unsigned unit_ctas;
};

// 8 lanes share a row of a head: lane e holds E = hd / 16 neighbouring values of each half, the pairs that the rotation turns.
template <bool BF16, int E>
__device__ __forceinline__ void load_row(const uint16_t* row, int e, float (&a)[E], float (&b)[E]) {
  uint32_t x[E / 2], y[E / 2];
  if constexpr (E == 8) {
    const uint4 p = *reinterpret_cast<const uint4*>(row + e * E), r = *reinterpret_cast<const uint4*>(row + 8 * E + e * E);
    x[0] = p.x, x[1] = p.y, x[2] = p.z, x[3] = p.w, y[0] = r.x, y[1] = r.y, y[2] = r.z, y[3] = r.w;
  } else {
    const uint2 p = *reinterpret_cast<const uint2*>(row + e * E), r = *reinterpret_cast<const uint2*>(row + 8 * E + e * E);
    x[0] = p.x, x[1] = p.y, y[0] = r.x, y[1] = r.y;
  }
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const float2 f = q8_up2<BF16>(x[i]), g = q8_up2<BF16>(y[i]);
    a[2 * i] = f.x, a[2 * i + 1] = f.y, b[2 * i] = g.x, b[2 * i + 1] = g.y;
  }
}
template <int E>
__device__ __forceinline__ void load_angles(const float* t, int e, float (&c)[E]) {
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    const float4 f = *reinterpret_cast<const float4*>(t + e * E + 4 * i);
    c[4 * i] = f.x, c[4 * i + 1] = f.y, c[4 * i + 2] = f.z, c[4 * i + 3] = f.w;
  }
}
template <int E>
__device__ __forceinline__ void rotate(float (&a)[E], float (&b)[E], const float (&c)[E], const float (&s)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float x = a[i], y = b[i];
    a[i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i]));
    b[i] = __fadd_rn(__fmul_rn(y, c[i]), __fmul_rn(x, s[i]));
  }
}
template <bool E4M3, int E>
__device__ __forceinline__ void store_codes(uint8_t* row, int e, const float (&a)[E], const float (&b)[E]) {
  uint32_t w[2][E / 4];
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    const float p[4] = {a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3]}, r[4] = {b[4 * i], b[4 * i + 1], b[4 * i + 2], b[4 * i + 3]};
    w[0][i] = q8_codes<E4M3>(p), w[1][i] = q8_codes<E4M3>(r);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (E == 8) *reinterpret_cast<uint2*>(row + h * 8 * E + e * E) = make_uint2(w[h][0], w[h][1]);
    else *reinterpret_cast<uint32_t*>(row + h * 8 * E + e * E) = w[h][0];
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// CTAs [0, unit_ctas): a warp has 8 slots of a block of one head's keys or values, a block's warps meet over its maximum; heads run fastest, so that the
// warps of a CTA share their tokens' angles and read neighbouring parts of a row.  The rest: a warp rotates q_heads heads of a row of q.
// Bound by HBM; a value is read once and held in registers between the maximum and its code.  (16 slots a warp: 110 registers, half the warps: a prompt of
// 2048 tokens x 32 heads of 128 took 31.7 us, with 8 26.7; 64-bit index divisions and clamps were 3.3 of those.  Now 23.7, 3.6 TB/s.)
static constexpr int kAppendWarps = 16, kAppendThreads = 32 * kAppendWarps, kSlotsLog2 = 3, kSteps = 2;  // kSteps: of 4 slots

template <bool BF16, bool E4M3, int E>
__global__ void __launch_bounds__(kAppendThreads, 2) rope_append_q8_kernel(const __grid_constant__ AppendParams p) {
  __shared__ uint32_t most[kAppendWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int hd = 16 * E;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane >> 3, e = lane & 7;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x >= p.unit_ctas) {
    // (32 bits: the divisions of 64 took a quarter of the instructions)
    const uint32_t item = (blockIdx.x - p.unit_ctas) * kAppendWarps + warp, row = item / (uint32_t)p.q_parts, b = row / (uint32_t)p.T, t = row - b * p.T;
    const int h0 = (int)(item - row * p.q_parts) * p.q_heads;
    if (row >= p.rows) return;
    const long long r = row, slot = p.start[b] + t;
    const bool live = (p.n_new == nullptr || t < p.n_new[b]) && slot >= 0 && slot < p.c.slots;
    float c[E] = {}, s[E] = {};
    if (live) {
      load_angles<E>(p.cos_t + slot * (hd / 2), e, c);
      load_angles<E>(p.sin_t + slot * (hd / 2), e, s);
    }
    for (int h = h0 + sub; h < min(h0 + p.q_heads, p.H); h += 4) {
      float x[E] = {}, y[E] = {};
      if (live) {
        load_row<BF16, E>(p.q + r * p.ldq + (long long)h * hd, e, x, y);
        rotate<E>(x, y, c, s);
      }
      uint32_t o[2][E / 2];
#pragma unroll
      for (int i = 0; i < E / 2; ++i) o[0][i] = q8_down2<BF16>(x[2 * i], x[2 * i + 1]), o[1][i] = q8_down2<BF16>(y[2 * i], y[2 * i + 1]);
      uint16_t* to = p.q_out + r * p.ldo + (long long)h * hd + e * E;
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        if constexpr (E == 8) *reinterpret_cast<uint4*>(to + z * 8 * E) = make_uint4(o[z][0], o[z][1], o[z][2], o[z][3]);
        else *reinterpret_cast<uint2*>(to + z * 8 * E) = make_uint2(o[z][0], o[z][1]);
      }
    }
    return;
  }
  // ---- 8 slots of a block
  const int wl = p.c.block_log2 - kSlotsLog2, per_cta = kAppendWarps >> wl, w = warp & ((1 << wl) - 1);
  const uint32_t unit = blockIdx.x * per_cta + (warp >> wl);
  const bool mine = unit < p.units;
  uint32_t u = mine ? unit : 0, v = u / (uint32_t)p.c.kv_heads;
  const int h = (int)(u - v * p.c.kv_heads);
  const bool is_v = v & 1;
  v >>= 1;
  const long long b = v / (uint32_t)p.blocks_per;
  const int j = (int)(v - (uint32_t)b * p.blocks_per);
  const long long start = p.start[b], count = p.n_new == nullptr ? p.T : max(0ll, min((long long)p.T, p.n_new[b]));
  const long long first = max(start, 0ll), end = min(start + count, (long long)p.c.slots);  // the new slots
  const long long block = (first >> p.c.block_log2) + j, s0 = (block << p.c.block_log2) + (w << kSlotsLog2);
  const bool touched = mine && first < end && (block << p.c.block_log2) < end;  // (the same for all warps of a block)
  float x[kSteps][E], y[kSteps][E];
  float big = 0.f;  // (max.NaN: a block with a NaN has it for its maximum, and reads back as NaN throughout)
  const long long head = b * p.c.kv_heads + h;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const long long slot = s0 + 4 * i + sub;
    if (touched && slot >= first && slot < end) {
      const long long r = b * p.T + (slot - start);
      if (is_v) {
        load_row<BF16, E>(p.v + r * p.ldv + (long long)h * hd, e, x[i], y[i]);
      } else {
        float c[E], s[E];
        load_row<BF16, E>(p.k + r * p.ldk + (long long)h * hd, e, x[i], y[i]);
        load_angles<E>(p.cos_t + slot * (hd / 2), e, c);
        load_angles<E>(p.sin_t + slot * (hd / 2), e, s);
        rotate<E>(x[i], y[i], c, s);
      }
#pragma unroll
      for (int z = 0; z < E; ++z) big = max_nan(big, fabsf(x[i][z])), big = max_nan(big, fabsf(y[i][z]));
    }
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(big) & 0x7fffffffu);
  if (lane == 0) most[warp] = top;
  __syncthreads();
  if (!touched) return;
  for (int i = 0; i < (1 << wl); ++i) top = max(top, most[(warp & ~((1 << wl) - 1)) + i]);
  float* const scale = (is_v ? p.c.v_scale : p.c.k_scale) + head * p.c.n_blocks + block;
  uint8_t* const codes = (is_v ? p.c.v : p.c.k) + (head * p.c.slots + s0) * hd;
  const float before = (block << p.c.block_log2) >= first ? 0.f : *scale;
  float asked = __fmul_rn(__uint_as_float(top), 1.f / q8_top<E4M3>());
  if (asked < 1.17549435e-38f) asked = 0.f;  // (its inverse would be infinite)
  const float after = __uint_as_float(max(__float_as_uint(before), __float_as_uint(asked)));
  const float inverse = after > 0.f ? __fdiv_rn(1.f, after) : 0.f;  // (an infinite or NaN scale: codes 0, which read back as NaN)
  const bool grown = __float_as_uint(after) > __float_as_uint(before);
  const float ratio = __fmul_rn(before, inverse);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const long long slot = s0 + 4 * i + sub;
    uint8_t* const row = codes + (4 * i + sub) * hd;
    if (slot >= first && slot < end) {
#pragma unroll
      for (int z = 0; z < E; ++z) x[i][z] = __fmul_rn(x[i][z], inverse), y[i][z] = __fmul_rn(y[i][z], inverse);
      if (inverse == 0.f) {  // (what is no number has code 0)
#pragma unroll
        for (int z = 0; z < E; ++z) x[i][z] = y[i][z] = 0.f;
      }
      store_codes<E4M3, E>(row, e, x[i], y[i]);
    } else if (grown && slot < first) {
#pragma unroll
      for (int z = 0; z < 2; ++z) {
#pragma unroll
        for (int m = 0; m < E / 4; ++m) {
          uint32_t* const at = reinterpret_cast<uint32_t*>(row + z * 8 * E + e * E + 4 * m);
          float f[4];
          q8_floats<E4M3>(*at, f);
#pragma unroll
          for (int n = 0; n < 4; ++n) f[n] = __fmul_rn(f[n], ratio);
          *at = q8_codes<E4M3>(f);
        }
      }
    }
  }
  // (every warp of the block has read the old scale by now only if they meet again)
  asm volatile("bar.sync %0, %1;" ::"r"(1 + (warp >> wl)), "r"(32 << wl) : "memory");
  if (w == 0 && lane == 0) *scale = after;
}

// value = code * scale, the product in fp32 and then rounded to 16 bits; 16 codes a thread; zeros behind a sequence's length.  Bound by HBM, 1 byte in, 2 out: 16 x 8 x 4099 slots of 64, 186 MB, 34 us,
// 5.4 TB/s.
template <bool BF16, bool E4M3>
__global__ void __launch_bounds__(256) cache_read_q8_kernel(Q8View c, int hd_log2, const long long* lengths, long long pieces, uint16_t* k_out, uint16_t* v_out) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= pieces) return;
  const bool is_v = blockIdx.y;
  const long long row = i >> (hd_log2 - 4), head = row / c.slots, slot = row - head * c.slots;
  uint4 o[2] = {};
  if (lengths == nullptr || slot < lengths[head / c.kv_heads]) {
    const uint4 w = *reinterpret_cast<const uint4*>((is_v ? c.v : c.k) + i * 16);
    const float s = (is_v ? c.v_scale : c.k_scale)[head * c.n_blocks + (slot >> c.block_log2)];
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    uint32_t r[8];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float f[4];
      q8_floats<E4M3>(ws[n], f);
      r[2 * n] = q8_down2<BF16>(f[0] * s, f[1] * s), r[2 * n + 1] = q8_down2<BF16>(f[2] * s, f[3] * s);
    }
    o[0] = make_uint4(r[0], r[1], r[2], r[3]), o[1] = make_uint4(r[4], r[5], r[6], r[7]);
  }
  uint4* const to = reinterpret_cast<uint4*>((is_v ? v_out : k_out) + i * 16);
  to[0] = o[0], to[1] = o[1];
}

}  // namespace blr

using namespace blr;

extern "C" {

int blr_rope_append_q8(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const float* cos_table,
                       const float* sin_table, const int64_t* start, const int64_t* n_new, int64_t n_tok, int heads, int dtype,
                       const blr_q8_cache* cache, void* q_out, int64_t ldo, void* stream) {
  AppendParams p = {};
  int rc;
  if ((rc = q8_view(cache, &p.c))) return rc;
  BLR_REQUIRE(dtype == BLR_DTYPE_F16 || dtype == BLR_DTYPE_BF16, BLR_ERR_ARG, "unknown dtype %d", dtype);
  BLR_REQUIRE(n_tok >= 0 && n_tok < (1ll << 31) && heads > 0, BLR_ERR_ARG, "rope_append_q8: n_tok = %lld, heads = %d", (long long)n_tok, heads);
  BLR_REQUIRE((ldq | ldk | ldv | ldo) % 8 == 0, BLR_ERR_ARG, "rope_append_q8: row strides must be multiples of 8");
  if (cache->n_seq == 0 || n_tok == 0) return BLR_OK;
  BLR_REQUIRE(q && k && v && cos_table && sin_table && start && q_out, BLR_ERR_ARG, "null pointer");
  BLR_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(q_out) |
                reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) & 15) == 0, BLR_ERR_ARG,
              "rope_append_q8 needs 16-byte aligned pointers");
  p.q = static_cast<const uint16_t*>(q), p.k = static_cast<const uint16_t*>(k), p.v = static_cast<const uint16_t*>(v);
  p.q_out = static_cast<uint16_t*>(q_out);
  p.ldq = ldq, p.ldk = ldk, p.ldv = ldv, p.ldo = ldo;
  p.cos_t = cos_table, p.sin_t = sin_table;
  p.start = reinterpret_cast<const long long*>(start), p.n_new = reinterpret_cast<const long long*>(n_new);
  p.T = (int)n_tok, p.H = heads;
  // T neighbouring slots lie in at most this many blocks
  p.blocks_per = (int)(((n_tok + cache->block - 2) >> p.c.block_log2) + 1);
  const long long units = cache->n_seq * p.blocks_per * 2 * p.c.kv_heads, rows = cache->n_seq * n_tok;
  const int per_cta = kAppendWarps >> (p.c.block_log2 - kSlotsLog2);
  const long long unit_ctas = (units + per_cta - 1) / per_cta;
  // a row's heads by as few warps as leave every SM its sixteen
  p.q_heads = 4;
  while (p.q_heads < 16 && rows * ((heads + 2 * p.q_heads - 1) / (2 * p.q_heads)) >= 16ll * sm_count()) p.q_heads *= 2;
  p.q_parts = (heads + p.q_heads - 1) / p.q_heads;
  const long long ctas = unit_ctas + (rows * p.q_parts + kAppendWarps - 1) / kAppendWarps;
  BLR_REQUIRE(ctas < (1ll << 31) / kAppendWarps && units < (1ll << 31) && rows * p.q_parts < (1ll << 31) - kAppendWarps, BLR_ERR_SHAPE, "too many tokens");
  p.units = (uint32_t)units, p.rows = (uint32_t)rows;
  p.unit_ctas = (unsigned)unit_ctas;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == BLR_DTYPE_BF16, e4 = cache->code == BLR_Q8_E4M3;
  auto go = [&](auto kernel) { return q8_launch(kernel, dim3((unsigned)ctas), kAppendThreads, 0, st, p); };
  if (cache->head_dim == 128)
    return bf ? (e4 ? go(rope_append_q8_kernel<true, true, 8>) : go(rope_append_q8_kernel<true, false, 8>))
              : (e4 ? go(rope_append_q8_kernel<false, true, 8>) : go(rope_append_q8_kernel<false, false, 8>));
  return bf ? (e4 ? go(rope_append_q8_kernel<true, true, 4>) : go(rope_append_q8_kernel<true, false, 4>))
            : (e4 ? go(rope_append_q8_kernel<false, true, 4>) : go(rope_append_q8_kernel<false, false, 4>));
}

int blr_cache_read_q8(const blr_q8_cache* cache, const int64_t* lengths, int dtype, void* k_out, void* v_out, void* stream) {
  Q8View c;
  int rc;
  if ((rc = q8_view(cache, &c))) return rc;
  BLR_REQUIRE(dtype == BLR_DTYPE_F16 || dtype == BLR_DTYPE_BF16, BLR_ERR_ARG, "unknown dtype %d", dtype);
  if (cache->n_seq == 0) return BLR_OK;
  BLR_REQUIRE(k_out && v_out, BLR_ERR_ARG, "null pointer");
  BLR_REQUIRE(((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) == 0, BLR_ERR_ARG,
              "cache_read_q8 needs 16-byte aligned outputs");
  const int hd_log2 = cache->head_dim == 128 ? 7 : 6;
  const long long pieces = cache->n_seq * c.kv_heads * c.slots << (hd_log2 - 4), ctas = (pieces + 255) / 256;
  BLR_REQUIRE(ctas < (1ll << 31), BLR_ERR_SHAPE, "too many slots");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == BLR_DTYPE_BF16, e4 = cache->code == BLR_Q8_E4M3;
  auto go = [&](auto kernel) {
    return q8_launch(kernel, dim3((unsigned)ctas, 2), 256, 0, st, c, hd_log2, reinterpret_cast<const long long*>(lengths), pieces,
                  static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out));
  };
  return bf ? (e4 ? go(cache_read_q8_kernel<true, true>) : go(cache_read_q8_kernel<true, false>))
            : (e4 ? go(cache_read_q8_kernel<false, true>) : go(cache_read_q8_kernel<false, false>));
}

}  // extern "C"
