// Causal attention of a sequence's newest tokens over an 8-bit cache (q8.cuh), a few rows at a time (sm_100a).
//
// A kv head's rows are its T tokens x (heads / kv_heads) query heads, token by token.  For 16 keys a warp computes S^T = K Q^T and O^T += V^T P^T with
// mma.sync (keys, then dimensions, as the 16 rows, 8 query rows as the columns), so that one query row costs what eight do and no operand is transposed in
// memory: the sum of the first product may run over the dimensions in any order, so a thread takes 16 neighbouring bytes of a key, and the second over the keys in
// any order, so it takes 16 neighbouring dimensions of four keys; P^T comes out of S^T by movmatrix.
//   s_j = ks_j c (q . k_j),  p_j = 2^(s_j - m),  l = sum p_j,  o = sum (p_j vs_j / R) v_j  with codes k_j, v_j and the scales ks_j, vs_j of their blocks:
// codes are exact in fp16, q is too (bf16 rows are brought into its range by a power of two), so the only roundings to 16 bits are q's own and p's; sums are fp32.
// m follows the maximum only where it is more than 2^8 behind, R the largest value scale where it is more than 2^4 behind: p stays below 2^12, and what is lost of
// a small p is 2^-25 of the largest.
// Bound by HBM on the codes (a key and its value are 2 hd bytes).  The keys of a row are shared out over the warps of a CTA and over up to kMaxSplits CTAs.
#include "../../include/blr_b200.h"
#include "q8_attention.h"
#include "tmap.h"

namespace blr {

static constexpr int kQ8Warps = 8, kMaxSplits = 64;

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <int HD>
struct Q8Keys {  // 16 keys of a warp: rows g and g + 8 of K, keys 2t, 2t + 1, 2t + 8, 2t + 9 of V
  uint32_t k[2][HD / 16], v[4][HD / 32];
  float ks, vs;
};
template <int HD>
__device__ __forceinline__ void q8_load(Q8Keys<HD>& x, const Q8View& c, const uint8_t* kh, const uint8_t* vh, const float* ksh, const float* vsh, int j0, int g, int t) {
  const int last = c.slots - 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* row = kh + (long long)min(j0 + 8 * i + g, last) * HD + 16 * t;
#pragma unroll
    for (int m = 0; m < HD / 64; ++m) {
      const uint4 w = *reinterpret_cast<const uint4*>(row + 64 * m);
      x.k[i][4 * m] = w.x, x.k[i][4 * m + 1] = w.y, x.k[i][4 * m + 2] = w.z, x.k[i][4 * m + 3] = w.w;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint8_t* row = vh + (long long)min(j0 + 2 * t + (i & 1) + 8 * (i >> 1), last) * HD + (HD / 8) * g;
    if constexpr (HD == 128) {
      const uint4 w = *reinterpret_cast<const uint4*>(row);
      x.v[i][0] = w.x, x.v[i][1] = w.y, x.v[i][2] = w.z, x.v[i][3] = w.w;
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(row);
      x.v[i][0] = w.x, x.v[i][1] = w.y;
    }
  }
  x.ks = ksh[j0 >> c.block_log2], x.vs = vsh[j0 >> c.block_log2];
}

template <bool E4M3, int HD, int NT>
__global__ void __launch_bounds__(32 * kQ8Warps) q8_attention_kernel(const __grid_constant__ Q8AttnParams p) {
  constexpr int kSteps = HD / 16, kRows = 8 * NT, kPitch = HD + 4;
  __shared__ float os[kQ8Warps][8][kPitch];
  __shared__ float wm[kQ8Warps][kRows], wl[kQ8Warps][kRows];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % p.ns, tile = blockIdx.x / p.ns, qt = tile % p.q_tiles, bh = tile / p.q_tiles;
  const int b = bh / p.c.kv_heads, h = bh - b * p.c.kv_heads, r0 = qt * kRows;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long start = p.start[b], count = p.n_new == nullptr ? p.T : min((long long)p.T, p.n_new[b]);
  const int keys = q8_seen_by(p, start, count, r0, r0 + kRows);
  const int share = ((keys + p.ns - 1) / p.ns + 63) & ~63, k0 = min(keys, split * share), k1 = min(keys, k0 + share);

  // ---- the query rows as fp16 fragments, and what their dot products are to be multiplied with
  uint32_t qf[NT][kSteps][2];
  float factor[NT][2];
  int lim[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + 8 * n + g;
    float f[HD / 4];
    uint32_t most = 0;
    if (r < p.rows && r / p.G < count) {
      const int tok = r / p.G;
      const uint16_t* row = p.q + ((long long)b * p.T + tok) * p.ldq + (long long)(h * p.G + r - tok * p.G) * HD + 16 * t;
#pragma unroll
      for (int m = 0; m < HD / 64; ++m) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint4 x = *reinterpret_cast<const uint4*>(row + 64 * m + 8 * w);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = p.bf16 ? q8_up2<true>(xs[i]) : q8_up2<false>(xs[i]);
            f[16 * m + 8 * w + 2 * i] = v.x, f[16 * m + 8 * w + 2 * i + 1] = v.y;
            most = max(most, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < HD / 4; ++i) f[i] = 0.f;
    }
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int up = q8_row_up(most, p.bf16);
    const float mul = __uint_as_float((uint32_t)up << 23), back = __uint_as_float((uint32_t)(254 - up) << 23);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      qf[n][s][0] = pack_half2(f[4 * s] * mul, f[4 * s + 1] * mul);
      qf[n][s][1] = pack_half2(f[4 * s + 2] * mul, f[4 * s + 3] * mul);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      factor[n][i] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * i) * p.scale_log2;
      const int rc = r0 + 8 * n + 2 * t + i;
      lim[n][i] = rc < p.rows ? q8_seen(start, count, rc / p.G, p.c.slots) : 0;
    }
  }

  const long long base = (long long)bh * p.c.slots * HD;
  const uint8_t *kh = p.c.k + base, *vh = p.c.v + base;
  const float *ksh = p.c.k_scale + (long long)bh * p.c.n_blocks, *vsh = p.c.v_scale + (long long)bh * p.c.n_blocks;
  float o[NT][kSteps][4] = {}, m[NT][2], mu[NT][2], l[NT][2] = {}, R = 0.f, inv_R = 0.f;
#pragma unroll
  for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, mu[n][0] = mu[n][1] = 0.f;

  Q8Keys<HD> next;
  int j0 = k0 + 16 * warp;
  if (j0 < k1) q8_load<HD>(next, p.c, kh, vh, ksh, vsh, j0, g, t);
#pragma unroll 1
  for (; j0 < k1; j0 += 16 * kQ8Warps) {
    Q8Keys<HD> x = next;
    if (j0 + 16 * kQ8Warps < k1) q8_load<HD>(next, p.c, kh, vh, ksh, vsh, j0 + 16 * kQ8Warps, g, t);
    // ---- S^T
    float s[NT][4] = {};
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const uint32_t w0 = q8_bias<E4M3>(x.k[0][st]), w1 = q8_bias<E4M3>(x.k[1][st]);
      const uint32_t a0 = q8_half2<E4M3>(w0, false), a1 = q8_half2<E4M3>(w1, false), a2 = q8_half2<E4M3>(w0, true), a3 = q8_half2<E4M3>(w1, true);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_16816<false>(s[n], a0, a1, a2, a3, qf[n][st][0], qf[n][st][1]);
    }
    // ---- p
    bool behind = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[n][i] = j0 + g + 8 * (i >> 1) < lim[n][i & 1] ? s[n][i] * (factor[n][i & 1] * x.ks) : -INFINITY;
        behind |= s[n][i] > m[n][i & 1] + 8.f;
      }
    if (__any_sync(0xffffffffu, behind)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = fmaxf(s[n][i], s[n][i + 2]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          mx = fmaxf(mx, m[n][i]);
          const float corr = mx == -INFINITY ? 1.f : ex2(m[n][i] - mx);
          m[n][i] = mx, mu[n][i] = mx == -INFINITY ? 0.f : mx;
          l[n][i] *= corr;
#pragma unroll
          for (int d = 0; d < kSteps; ++d) o[n][d][i] *= corr, o[n][d][i + 2] *= corr;
        }
    }
    if (x.vs > 16.f * R && x.vs <= 3.4e38f) {
      const float corr = R / x.vs;
      R = x.vs, inv_R = 1.f / R;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int d = 0; d < kSteps; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][d][i] *= corr;
    }
    const float f = x.vs * inv_R;
    uint32_t pt[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = j0 + g + 8 * (i >> 1) < lim[n][i & 1];  // (a masked place of a block that holds a NaN stays 0)
        const float v = ex2(s[n][i] - mu[n][i & 1]);
        l[n][i & 1] += v;
        e[i] = in ? v * f : 0.f;
      }
      pt[n][0] = transpose8x8(pack_half2(e[0], e[1])), pt[n][1] = transpose8x8(pack_half2(e[2], e[3]));
    }
    if (j0 + 16 > keys) {  // (slots that nobody wrote may hold anything)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j0 + 2 * t + (i & 1) + 8 * (i >> 1) >= keys)
#pragma unroll
          for (int w = 0; w < HD / 32; ++w) x.v[i][w] = 0;
    }
    // ---- O^T
#pragma unroll
    for (int w = 0; w < HD / 32; ++w) {
      uint32_t pr[2][2];  // [keys][bytes 0, 1 | 2, 3], interleaved by key
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        pr[i][0] = q8_bias<E4M3>(prmt(x.v[2 * i][w], x.v[2 * i + 1][w], 0x5140u));
        pr[i][1] = q8_bias<E4M3>(prmt(x.v[2 * i][w], x.v[2 * i + 1][w], 0x7362u));
      }
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const uint32_t a0 = q8_half2<E4M3>(pr[0][z], false), a1 = q8_half2<E4M3>(pr[0][z], true);
        const uint32_t a2 = q8_half2<E4M3>(pr[1][z], false), a3 = q8_half2<E4M3>(pr[1][z], true);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_16816<false>(o[n][2 * w + z], a0, a1, a2, a3, pt[n][0], pt[n][1]);
      }
    }
  }

  // ---- the warps' results meet
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], d);
      if (g == 0) wm[warp][8 * n + 2 * t + i] = m[n][i], wl[warp][8 * n + 2 * t + i] = l[n][i];
    }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float M[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      M[i] = -INFINITY;
      for (int w = 0; w < kQ8Warps; ++w) M[i] = fmaxf(M[i], wm[w][8 * n + 2 * t + i]);
      const float weight = m[n][i] == -INFINITY ? 0.f : ex2(m[n][i] - M[i]) * R;
#pragma unroll
      for (int d = 0; d < kSteps; ++d)  // dimensions HD / 8 g + 2 d, + 1
        *reinterpret_cast<float2*>(&os[warp][2 * t + i][(HD / 8) * g + 2 * d]) =
            m[n][i] == -INFINITY ? make_float2(0.f, 0.f) : make_float2(o[n][d][i] * weight, o[n][d][i + 2] * weight);
    }
    __syncthreads();
    constexpr int kPer = 8 * HD / (32 * kQ8Warps);  // values of a thread: 4 or 2 neighbours
    const int row = threadIdx.x / (HD / kPer), d0 = (threadIdx.x - row * (HD / kPer)) * kPer, r = r0 + 8 * n + row;
    float Mr = -INFINITY, Lr = 0.f, sum[kPer] = {};
    for (int w = 0; w < kQ8Warps; ++w) Mr = fmaxf(Mr, wm[w][8 * n + row]);
    for (int w = 0; w < kQ8Warps; ++w) {
      if (wm[w][8 * n + row] != -INFINITY || wl[w][8 * n + row] != 0.f) Lr += wl[w][8 * n + row] * (Mr == -INFINITY ? 1.f : ex2(wm[w][8 * n + row] - Mr));
#pragma unroll
      for (int i = 0; i < kPer; ++i) sum[i] += os[w][row][d0 + i];
    }
    if (r < p.rows) {
      const int tok = r / p.G;
      if (p.ns == 1) {
        const float inv = Lr == 0.f ? 0.f : 1.f / Lr;
        uint16_t* to = p.out + ((long long)b * p.T + tok) * p.ldo + (long long)(h * p.G + r - tok * p.G) * HD + d0;
#pragma unroll
        for (int i = 0; i < kPer; i += 2)
          *reinterpret_cast<uint32_t*>(to + i) = p.bf16 ? q8_down2<true>(sum[i] * inv, sum[i + 1] * inv) : q8_down2<false>(sum[i] * inv, sum[i + 1] * inv);
      } else {
        float* to = p.part + (((long long)bh * p.rows + r) * p.ns + split) * (HD + 4);
        if (!(Lr == 0.f)) {
#pragma unroll
          for (int i = 0; i < kPer; ++i) to[d0 + i] = sum[i];
        }
        if (d0 == 0) to[HD] = Mr, to[HD + 1] = Lr;
      }
    }
    __syncthreads();
  }
}

// The splits of a row: a warp sums them.
template <int HD>
__global__ void __launch_bounds__(256) q8_combine_kernel(const __grid_constant__ Q8AttnParams p, long long total) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= total) return;
  const float* from = p.part + row * p.ns * (HD + 4);
  float M = -INFINITY, L = 0.f, sum[HD / 32] = {};
  for (int s = lane; s < p.ns; s += 32) M = fmaxf(M, from[s * (HD + 4) + HD]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  for (int s = 0; s < p.ns; ++s) {
    const float* x = from + s * (HD + 4);
    const float ls = x[HD + 1];
    if (ls == 0.f) continue;
    const float w = M == -INFINITY ? 1.f : ex2(x[HD] - M);
    L += ls * w;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) sum[i] += x[(HD / 32) * lane + i] * w;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const long long bh = row / p.rows, r = row - bh * p.rows, b = bh / p.c.kv_heads, h = bh - b * p.c.kv_heads, tok = r / p.G;
  uint16_t* to = p.out + (b * p.T + tok) * p.ldo + (h * p.G + r - tok * p.G) * HD + (HD / 32) * lane;
#pragma unroll
  for (int i = 0; i < HD / 32; i += 2)
    *reinterpret_cast<uint32_t*>(to + i) = p.bf16 ? q8_down2<true>(sum[i] * inv, sum[i + 1] * inv) : q8_down2<false>(sum[i] * inv, sum[i + 1] * inv);
}

// CTAs over which a row's keys are split: as many as fill the SMs, with at least 256 keys each (512 in the prompt kernel).
static int q8_splits(long long tiles, int slots, bool prompt) {
  const long long room = (prompt ? 1ll : 2ll) * sm_count(), least = prompt ? 512 : 256;
  long long ns = room / tiles;
  if (ns > (slots + least - 1) / least) ns = (slots + least - 1) / least;
  return ns < 1 ? 1 : ns > kMaxSplits ? kMaxSplits : (int)ns;
}
struct Q8Plan {
  int nt, q_tiles, ns;  // nt: column tiles of 8 rows of the kernel here, 0: the prompt kernel
  long long rows, tiles;
};
static Q8Plan q8_plan(const blr_q8_cache* c, int64_t n_tok, int heads) {
  Q8Plan a = {};
  a.rows = n_tok * (heads / c->kv_heads);
  a.nt = a.rows <= 8 ? 1 : a.rows <= 64 ? 2 : 0;
  const int per = a.nt ? 8 * a.nt : kQ8PromptRows;
  a.q_tiles = (int)((a.rows + per - 1) / per);
  a.tiles = c->n_seq * c->kv_heads * a.q_tiles;
  a.ns = a.tiles > 0 ? q8_splits(a.tiles, c->slots, a.nt == 0) : 1;
  return a;
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

size_t blr_attention_q8_scratch_bytes(const blr_q8_cache* cache, int64_t n_tok, int heads) {
  if (!cache || cache->n_seq <= 0 || cache->kv_heads <= 0 || cache->slots <= 0 || n_tok <= 0 || heads <= 0 || heads % cache->kv_heads != 0) return 0;
  const Q8Plan a = q8_plan(cache, n_tok, heads);
  return a.ns > 1 ? (size_t)cache->n_seq * cache->kv_heads * a.rows * a.ns * (cache->head_dim + 4) * sizeof(float) : 0;
}

int blr_attention_q8(const void* q, int64_t ldq, const blr_q8_cache* cache, const int64_t* start, const int64_t* n_new, int64_t n_tok, int heads,
                     float scale, int dtype, void* out, int64_t ldo, void* scratch, size_t scratch_bytes, void* ws, void* stream) {
  Q8AttnParams p = {};
  int rc;
  if ((rc = q8_view(cache, &p.c))) return rc;
  BLR_REQUIRE(dtype == BLR_DTYPE_F16 || dtype == BLR_DTYPE_BF16, BLR_ERR_ARG, "unknown dtype %d", dtype);
  BLR_REQUIRE(heads > 0 && heads % cache->kv_heads == 0, BLR_ERR_ARG, "attention_q8: %d heads are no multiple of %d kv heads", heads, cache->kv_heads);
  BLR_REQUIRE(n_tok >= 0 && n_tok * (heads / cache->kv_heads) < (1ll << 30), BLR_ERR_SHAPE, "attention_q8: n_tok = %lld", (long long)n_tok);
  BLR_REQUIRE((ldq | ldo) % 8 == 0, BLR_ERR_ARG, "attention_q8: row strides must be multiples of 8");
  BLR_REQUIRE(scale > 0.f && scale <= 3.0e38f, BLR_ERR_ARG, "attention_q8: the scale must be a positive number");
  if (cache->n_seq == 0 || n_tok == 0) return BLR_OK;
  BLR_REQUIRE(q && start && out, BLR_ERR_ARG, "null pointer");
  BLR_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(scratch)) & 15) == 0, BLR_ERR_ARG,
              "attention_q8 needs 16-byte aligned pointers");
  const Q8Plan a = q8_plan(cache, n_tok, heads);
  const size_t need = blr_attention_q8_scratch_bytes(cache, n_tok, heads);
  BLR_REQUIRE(need == 0 || (scratch && scratch_bytes >= need), BLR_ERR_WORKSPACE, "attention_q8: scratch of %zu bytes is too small", scratch_bytes);
  BLR_REQUIRE(a.tiles * a.ns < (1ll << 31), BLR_ERR_SHAPE, "attention_q8: too many rows");
  p.q = static_cast<const uint16_t*>(q), p.out = static_cast<uint16_t*>(out);
  p.ldq = ldq, p.ldo = ldo;
  p.start = reinterpret_cast<const long long*>(start), p.n_new = reinterpret_cast<const long long*>(n_new);
  p.part = static_cast<float*>(scratch);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.T = (int)n_tok, p.H = heads, p.G = heads / cache->kv_heads, p.rows = (int)a.rows, p.q_tiles = a.q_tiles, p.ns = a.ns, p.bf16 = dtype == BLR_DTYPE_BF16;
  p.n_bh = (int)(cache->n_seq * cache->kv_heads);
  p.status = ws == nullptr ? nullptr : static_cast<unsigned*>(ws) + 255;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)(a.tiles * a.ns)), block(32 * kQ8Warps);
  auto go = [&](auto kernel) { return launch(kernel, grid, block, st, p); };
#define BLR_Q8_ATTN(E4, HD) (a.nt == 1 ? go(q8_attention_kernel<E4, HD, 1>) : go(q8_attention_kernel<E4, HD, 2>))
  if (a.nt == 0) rc = q8_launch_prompt(p, cache->head_dim, cache->code, st);
  else if (cache->code == BLR_Q8_E4M3) rc = cache->head_dim == 128 ? BLR_Q8_ATTN(true, 128) : BLR_Q8_ATTN(true, 64);
  else rc = cache->head_dim == 128 ? BLR_Q8_ATTN(false, 128) : BLR_Q8_ATTN(false, 64);
#undef BLR_Q8_ATTN
  if (rc || a.ns == 1) return rc;
  const long long total = cache->n_seq * cache->kv_heads * a.rows;
  const dim3 cgrid((unsigned)((total + 7) / 8));
  return cache->head_dim == 128 ? launch(q8_combine_kernel<128>, cgrid, dim3(256), st, p, total) : launch(q8_combine_kernel<64>, cgrid, dim3(256), st, p, total);
}

}  // extern "C"
