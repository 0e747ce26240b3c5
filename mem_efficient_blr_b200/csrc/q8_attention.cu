// Causal attention of a sequence's newest tokens over an 8-bit cache (q8.cuh), a few rows at a time (sm_100a).
//
// A kv head's rows are its T tokens x (heads / kv_heads) query heads, token by token.  For 16 keys a warp computes S^T = K Q^T and O^T += V^T P^T with
// mma.sync (keys, then dimensions, as the 16 rows, 8 query rows as the columns), so that one query row costs what eight do and no operand is transposed in
// memory: the sum of the first product may run over the dimensions in any order, so a thread takes 16 neighbouring bytes of a key, and the second over the keys in
// any order, so it takes 16 neighbouring dimensions of four keys; P^T comes out of S^T by movmatrix.
//   s_j = ks_j c (q . k_j),  p_j = 2^(s_j - m),  l = sum p_j,  o = sum (p_j vs_j D) v_j  with codes k_j, v_j, the scales ks_j, vs_j of their blocks, and the row's own
// references m and D (q8_attention.h):
// codes are exact in fp16, q is too (bf16 rows are brought into its range by a power of two; what is 2^-38 of a row's largest value may be lost), so the only rounding to
// 16 bits is that of p_j vs_j D; sums are fp32.
// m follows the maximum only where it is more than 2^8 behind, D the heaviest p vs only where it has outgrown 2^15.
// Bound by HBM on the codes (a key and its value are 2 hd bytes): 64 sequences x 32 heads x 2048 keys of 128, 1.08 GB, 163 us in a graph, 6.6 TB/s (194 among calls
// from Python); by latency where they are few (1 sequence: 13 us for 17 MB: positions, codes, a few groups a warp, the second kernel).  The keys of a row are shared out over the warps of a CTA and
// over up to kMaxSplits CTAs.  A first version that loaded the groups into registers took 280 us for the former: 8 warps an SM instead of 16.
#include "../../include/blr_b200.h"
#include "q8_attention.h"
#include "tmap.h"

namespace blr {

static constexpr int kMaxSplits = 64;

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// CTA (row tile, sequence and kv head, split): a warp takes every fourth group of 16 keys and brings them into a ring of its own, kFewStages groups deep, with
// cp.async: no warp waits for another before the end.  A row's 16-byte pieces are written where the reads below meet no bank twice (heads of 64: twice for V).
static constexpr int kFewWarps = 4, kFewThreads = 32 * kFewWarps, kFewStages = 3;

template <int HD>
__host__ __device__ constexpr int few_ring_bytes() {  // (the warps' sums lie over it in the end)
  constexpr int ring = kFewWarps * kFewStages * 32 * HD, sums = kFewWarps * 8 * (HD + 4) * 4;
  return ring > sums ? ring : sums;
}
template <int HD, int NT>
__host__ __device__ constexpr int few_smem_bytes() { return few_ring_bytes<HD>() + (NT > 2 ? NT * HD / 16 * 256 : 0); }

__device__ __forceinline__ void cp_async16_cg(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// Where the 16-byte piece c of row `row` of a group lies.
template <int HD>
__device__ __forceinline__ uint32_t few_place(int row, int c) { return row * HD + ((c ^ (HD == 128 ? row & 7 : (row >> 1) & 3)) << 4); }

template <bool E4M3, int HD, int NT>
__global__ void __launch_bounds__(kFewThreads, NT == 1 ? 4 : NT == 2 ? 3 : 2) q8_attention_kernel(const __grid_constant__ Q8AttnParams p) {
  constexpr int kSteps = HD / 16, kRows = 8 * NT, kPitch = HD + 4, kPieces = HD / 16;
  constexpr bool kQShared = NT > 2;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float wm[kFewWarps][kRows], wl[kFewWarps][kRows], wu[kFewWarps][kRows];
  float(*const os)[8][kPitch] = reinterpret_cast<float(*)[8][kPitch]>(ring);
  uint2* const q_frag = reinterpret_cast<uint2*>(ring + few_ring_bytes<HD>());  // [tile][step][lane]
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tiles = p.n_bh * p.q_tiles, split = blockIdx.x / tiles, tile = blockIdx.x - split * tiles, qt = tile % p.q_tiles, bh = tile / p.q_tiles;
  const int b = bh / p.c.kv_heads, h = bh - b * p.c.kv_heads, r0 = qt * kRows;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long start = p.start[b], count = p.n_new == nullptr ? p.T : min((long long)p.T, p.n_new[b]);
  const int keys = q8_seen_by(p, start, count, r0, r0 + kRows);
  int share = keys;
  if (p.ns > 1 && p.n_seq == 1) {
    share = ((keys + p.ns - 1) / p.ns + 16 * kFewWarps - 1) / (16 * kFewWarps) * (16 * kFewWarps);
  } else if (p.ns > 1) {
    // as many keys for every CTA, whatever its sequence's length: all of them over the CTAs that the SMs hold, but a sequence has no more than ns CTAs
    float total = 0.f;
    for (int i = lane; i < p.n_seq; i += 32) {
      const long long n = p.n_new == nullptr ? p.T : min((long long)p.T, p.n_new[i]);
      total += (float)q8_seen_by(p, p.start[i], n, 0, p.rows);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    const float even = total * (float)(p.c.kv_heads * p.q_tiles) / (float)p.room;
    const int n = max(1, min(p.ns, (int)((float)keys / fmaxf(even, 1.f))));  // (rounded down: all of them together are no more than the SMs hold)
    share = ((keys + n - 1) / n + 16 * kFewWarps - 1) / (16 * kFewWarps) * (16 * kFewWarps);
  }
  const int k0 = (int)min((long long)keys, (long long)split * share), k1 = min(keys, k0 + min(share, keys - k0));
  if (p.ns > 1 && k0 >= k1) {  // no keys for this CTA: its rows say so
    if (threadIdx.x < kRows && r0 + threadIdx.x < p.rows)
      *reinterpret_cast<float2*>(p.part + (((long long)bh * p.rows + r0 + threadIdx.x) * p.ns + split) * (HD + 4) + HD) = make_float2(-INFINITY, 0.f);
    return;
  }
  // groups of this warp: 16 keys from first + 64 j on
  const int first = k0 + 16 * warp, steps = first < k1 ? (k1 - first + 16 * kFewWarps - 1) / (16 * kFewWarps) : 0;
  const uint32_t base = smem_u32(ring) + warp * kFewStages * 32 * HD;
  const uint8_t *const kh = p.c.k + (long long)bh * p.c.slots * HD, *const vh = p.c.v + (long long)bh * p.c.slots * HD;
  auto bring = [&](int j) {
    if (j < steps) {
      const uint32_t to = base + (j % kFewStages) * 32 * HD;
      const int j0 = first + 16 * kFewWarps * j, c = lane % kPieces;
#pragma unroll
      for (int i = 0; i < kPieces / 2; ++i) {
        const int row = lane / kPieces + i * (32 / kPieces);
        const long long off = (long long)min(j0 + row, p.c.slots - 1) * HD + 16 * c;
        cp_async16_cg(to + few_place<HD>(row, c), kh + off);
        cp_async16_cg(to + 16 * HD + few_place<HD>(row, c), vh + off);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int j = 0; j < kFewStages - 1; ++j) bring(j);
  const float *ksh = p.c.k_scale + (long long)bh * p.c.n_blocks, *vsh = p.c.v_scale + (long long)bh * p.c.n_blocks;
  auto block_of = [&](int j) { return (first + 16 * kFewWarps * j) >> p.c.block_log2; };
  float ks_next = steps > 0 ? ksh[block_of(0)] : 0.f, vs_next = steps > 0 ? vsh[block_of(0)] : 0.f;

  float o[NT][kSteps][4] = {}, m[NT][2], l[NT][2] = {}, D[NT][2], safe = INFINITY;  // safe: value scales up to it bring no row's P beyond 2^15 as long as its p is at most 2^8
  {
    // ---- the query rows as fp16 fragments, and what their dot products are to be multiplied with
    uint32_t qf[kQShared ? 1 : NT][kSteps][2];
    float factor[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + 8 * n + g;
      const bool live = r < p.rows && r / p.G < count;
      const int tok = live ? r / p.G : 0;
      const uint16_t* row = p.q + ((long long)b * p.T + tok) * p.ldq + (long long)(h * p.G + (live ? r - tok * p.G : 0)) * HD + (HD / 4) * t;
      float f[HD / 4];
      uint32_t most = 0;
#pragma unroll
      for (int w = 0; w < HD / 32; ++w) {
        const uint4 x = live ? *reinterpret_cast<const uint4*>(row + 8 * w) : make_uint4(0, 0, 0, 0);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = p.bf16 ? q8_up2<true>(xs[i]) : q8_up2<false>(xs[i]);
          f[8 * w + 2 * i] = v.x, f[8 * w + 2 * i + 1] = v.y;
          most = max(most, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
        }
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int up = q8_row_up(most, p.bf16);
      const float mul = __uint_as_float((uint32_t)up << 23), back = __uint_as_float((uint32_t)(254 - up) << 23);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t x = pack_half2(f[4 * s] * mul, f[4 * s + 1] * mul), y = pack_half2(f[4 * s + 2] * mul, f[4 * s + 3] * mul);
        if constexpr (kQShared) {
          if (warp == n % kFewWarps) q_frag[(n * kSteps + s) * 32 + lane] = make_uint2(x, y);
        } else {
          qf[n][s][0] = x, qf[n][s][1] = y;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        factor[n][i] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * i) * p.scale_log2;
        const int rc = r0 + 8 * n + 2 * t + i;
        lim[n][i] = rc < p.rows ? q8_seen(start, count, rc / p.G, p.c.slots) : 0;
      }
      m[n][0] = m[n][1] = -INFINITY, D[n][0] = D[n][1] = 1.f;
    }
    if constexpr (kQShared) __syncthreads();
    int lim_all = 0x7fffffff;  // keys below it are masked for no row of the warp (0 where its tiles have places without a row: leaving those out gained nothing for 20 rows of 32)
#pragma unroll
    for (int n = 0; n < NT; ++n) lim_all = min(lim_all, min(lim[n][0], lim[n][1]));
    lim_all = __reduce_min_sync(0xffffffffu, lim_all);

#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
      const int j0 = first + 16 * kFewWarps * j;
      const float ks = ks_next, vs = vs_next;
      if (j + 1 < steps) ks_next = ksh[block_of(j + 1)], vs_next = vsh[block_of(j + 1)];
      const uint32_t at = base + (j % kFewStages) * 32 * HD;
      asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 2) : "memory");
      __syncwarp();  // (everybody's pieces are there, and everybody has done with the group before, whose place the next one takes)
      bring(j + kFewStages - 1);
      {
        // ---- S^T: rows g and g + 8 of K, HD / 4 neighbouring dimensions of each
        uint32_t kw[2][kSteps];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = 8 * i + g;
          if constexpr (HD == 128) {
            lds128(at + few_place<HD>(row, 2 * t), kw[i][0], kw[i][1], kw[i][2], kw[i][3]);
            lds128(at + few_place<HD>(row, 2 * t + 1), kw[i][4], kw[i][5], kw[i][6], kw[i][7]);
          } else {
            lds128(at + few_place<HD>(row, t), kw[i][0], kw[i][1], kw[i][2], kw[i][3]);
          }
        }
        float sc[NT][4] = {};
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const uint32_t w0 = q8_bias<E4M3>(kw[0][st]), w1 = q8_bias<E4M3>(kw[1][st]);
          const uint32_t a0 = q8_half2<E4M3>(w0, false), a1 = q8_half2<E4M3>(w1, false), a2 = q8_half2<E4M3>(w0, true), a3 = q8_half2<E4M3>(w1, true);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (kQShared) {
              const uint2 q = q_frag[(n * kSteps + st) * 32 + lane];
              mma_16816<false>(sc[n], a0, a1, a2, a3, q.x, q.y);
            } else {
              mma_16816<false>(sc[n], a0, a1, a2, a3, qf[n][st][0], qf[n][st][1]);
            }
          }
        }
        // ---- V: keys 2t, 2t + 1, 2t + 8, 2t + 9, HD / 8 neighbouring dimensions of each
        uint32_t vw[4][HD / 32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 2 * t + (i & 1) + 8 * (i >> 1);
          if constexpr (HD == 128) lds128(at + 16 * HD + few_place<HD>(row, g), vw[i][0], vw[i][1], vw[i][2], vw[i][3]);
          else lds64(at + 16 * HD + few_place<HD>(row, g >> 1) + (g & 1) * 8, vw[i][0], vw[i][1]);
        }
        // ---- p
        const bool part = j0 + 16 > lim_all;
        uint32_t behind = vs > safe ? (1u << NT) - 1 : 0;  // a bit for each tile of rows
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float c[2] = {factor[n][0] * ks, factor[n][1] * ks};
          bool up = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sc[n][i] *= c[i & 1];
            if (part && j0 + g + 8 * (i >> 1) >= lim[n][i & 1]) sc[n][i] = -INFINITY;
            up |= sc[n][i] > m[n][i & 1] + 8.f;
          }
          behind |= up ? 1u << n : 0;
        }
        if (__any_sync(0xffffffffu, behind != 0)) {
          if (NT > 1) behind = __reduce_or_sync(0xffffffffu, behind);
          float least = INFINITY;  // of the rows' 2^d
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (NT == 1 || (behind >> n & 1)) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float mx = fmaxf(sc[n][i], sc[n][i + 2]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                // a row that the new keys do not ask stays as it is; a factor vs D that no fp32 holds asks too, as long as the row sees the block
                const float f = vs <= 3.402823466e38f ? vs * D[n][i] : 0.f, peak = ceilf(mx);
                const bool ask = mx > m[n][i] + 8.f || ex2(mx - m[n][i]) * f > 32768.f || (f > 3.402823466e38f && mx != -INFINITY);
                const float to = ask ? fmaxf(m[n][i], peak) : m[n][i];
                float to_m = m[n][i], to_D = D[n][i], down, corr;
                q8_move(to, fmaxf(peak - to, -123.f) + q8_above(vs), to_m, to_D, down, corr);
                if (!ask) to_D = D[n][i], down = corr = 1.f;
                m[n][i] = to, D[n][i] = to_D;
                l[n][i] *= down;
#pragma unroll
                for (int d = 0; d < kSteps; ++d) o[n][d][i] *= corr, o[n][d][i + 2] *= corr;
              }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (m[n][i] != -INFINITY) least = fminf(least, q8_unit(D[n][i]));
          }
          safe = 128.f * __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(least)));
        }
        uint32_t pt[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float e[4];
          const float mu[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
          const float f[2] = {vs * D[n][0], vs * D[n][1]};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = ex2(sc[n][i] - mu[i & 1]);
            l[n][i & 1] += v;
            e[i] = v * f[i & 1];
            if (part && j0 + g + 8 * (i >> 1) >= lim[n][i & 1]) e[i] = 0.f;  // (a masked place of a block that holds a NaN)
          }
          pt[n][0] = transpose8x8(pack_half2(e[0], e[1])), pt[n][1] = transpose8x8(pack_half2(e[2], e[3]));
        }
        if (j0 + 16 > keys) {  // (slots that nobody wrote may hold anything)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (j0 + 2 * t + (i & 1) + 8 * (i >> 1) >= keys)
#pragma unroll
              for (int w = 0; w < HD / 32; ++w) vw[i][w] = 0;
        }
        // ---- O^T
#pragma unroll
        for (int w = 0; w < HD / 32; ++w) {
          uint32_t pr[2][2];  // [keys][bytes 0, 1 | 2, 3], interleaved by key
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            pr[i][0] = q8_bias<E4M3>(prmt(vw[2 * i][w], vw[2 * i + 1][w], 0x5140u));
            pr[i][1] = q8_bias<E4M3>(prmt(vw[2 * i][w], vw[2 * i + 1][w], 0x7362u));
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
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], d);
        if (g == 0) wm[warp][8 * n + 2 * t + i] = m[n][i], wl[warp][8 * n + 2 * t + i] = l[n][i], wu[warp][8 * n + 2 * t + i] = q8_unit(D[n][i]);
      }
  }
  // ---- the warps' results meet, over the ring
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float M = -INFINITY;
        for (int w = 0; w < kFewWarps; ++w) M = fmaxf(M, wm[w][8 * n + 2 * t + i]);
        const float weight = m[n][i] == -INFINITY ? 0.f : ex2(m[n][i] - M);
#pragma unroll
        for (int d = 0; d < kSteps; ++d)  // dimensions HD / 8 g + 2 d, + 1
          *reinterpret_cast<float2*>(&os[warp][2 * t + i][(HD / 8) * g + 2 * d]) =
              m[n][i] == -INFINITY ? make_float2(0.f, 0.f) : make_float2(o[n][d][i] * weight, o[n][d][i + 2] * weight);
      }
    }
    __syncthreads();
    constexpr int kPer = 8 * HD / (32 * kFewWarps);  // values of a thread: 8 or 4 neighbours
    {
      const int row = threadIdx.x / (HD / kPer), d0 = (threadIdx.x - row * (HD / kPer)) * kPer, r = r0 + 8 * n + row;
      float Mr = -INFINITY, Lr = 0.f, sum[kPer] = {};
      for (int w = 0; w < kFewWarps; ++w) Mr = fmaxf(Mr, wm[w][8 * n + row]);
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        if (wm[w][8 * n + row] != -INFINITY || wl[w][8 * n + row] != 0.f) Lr += wl[w][8 * n + row] * (Mr == -INFINITY ? 1.f : ex2(wm[w][8 * n + row] - Mr));
        const float u = wu[w][8 * n + row];
#pragma unroll
        for (int i = 0; i < kPer; i += 4) {
          const float4 x = *reinterpret_cast<const float4*>(&os[w][row][d0 + i]);
          sum[i] = fmaf(x.x, u, sum[i]), sum[i + 1] = fmaf(x.y, u, sum[i + 1]), sum[i + 2] = fmaf(x.z, u, sum[i + 2]), sum[i + 3] = fmaf(x.w, u, sum[i + 3]);
        }
      }
      if (r < p.rows) {
        if (p.ns == 1) {
          const float inv = Lr == 0.f ? 0.f : 1.f / Lr;
          const int tok = r / p.G;
          uint16_t* to = p.out + ((long long)b * p.T + tok) * p.ldo + (long long)(h * p.G + r - tok * p.G) * HD + d0;
          uint32_t x[kPer / 2];
#pragma unroll
          for (int i = 0; i < kPer; i += 2) x[i / 2] = p.bf16 ? q8_down2<true>(sum[i] * inv, sum[i + 1] * inv) : q8_down2<false>(sum[i] * inv, sum[i + 1] * inv);
          if constexpr (kPer == 8) *reinterpret_cast<uint4*>(to) = make_uint4(x[0], x[1], x[2], x[3]);
          else *reinterpret_cast<uint2*>(to) = make_uint2(x[0], x[1]);
        } else {
          float* to = p.part + (((long long)bh * p.rows + r) * p.ns + split) * (HD + 4);
          if (!(Lr == 0.f)) {
#pragma unroll
            for (int i = 0; i < kPer; i += 4) *reinterpret_cast<float4*>(to + d0 + i) = make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
          }
          if (d0 == 0) to[HD] = Mr, to[HD + 1] = Lr;
        }
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
  // lane s has the weight of splits s and s + 32
  float w[2], M = -INFINITY, L = 0.f, sum[HD / 32] = {};
  float2 ml[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    ml[i] = lane + 32 * i < p.ns ? *reinterpret_cast<const float2*>(from + (lane + 32 * i) * (HD + 4) + HD) : make_float2(-INFINITY, 0.f);
    M = fmaxf(M, ml[i].x);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] = ml[i].y == 0.f ? 0.f : M == -INFINITY || ml[i].y != ml[i].y ? 1.f : ex2(ml[i].x - M);
    L += ml[i].y == 0.f ? 0.f : ml[i].y * w[i];
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
#pragma unroll 8
  for (int s = 0; s < p.ns; ++s) {
    const float ws = __shfl_sync(0xffffffffu, s < 32 ? w[0] : w[1], s & 31);
    float x[HD / 32];
    if constexpr (HD == 128) {
      const float4 v = *reinterpret_cast<const float4*>(from + s * (HD + 4) + 4 * lane);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(from + s * (HD + 4) + 2 * lane);
      x[0] = v.x, x[1] = v.y;
    }
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) sum[i] += ws == 0.f ? 0.f : x[i] * ws;  // (a split without keys has left its sums as they were)
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const long long bh = row / p.rows, r = row - bh * p.rows, b = bh / p.c.kv_heads, h = bh - b * p.c.kv_heads, tok = r / p.G;
  uint16_t* to = p.out + (b * p.T + tok) * p.ldo + (h * p.G + r - tok * p.G) * HD + (HD / 32) * lane;
#pragma unroll
  for (int i = 0; i < HD / 32; i += 2)
    *reinterpret_cast<uint32_t*>(to + i) = p.bf16 ? q8_down2<true>(sum[i] * inv, sum[i + 1] * inv) : q8_down2<false>(sum[i] * inv, sum[i + 1] * inv);
}

struct Q8Plan {
  int nt, q_tiles, ns, room;  // nt: column tiles of 8 rows of the kernel here, 0: the prompt kernel; ns: CTAs that may share a row tile's keys
  long long rows, tiles, wide_tiles;  // wide_tiles: of 128 slots of a head, whose codes are widened ahead (0: not)
};
// Row tiles of a kv head from which its codes are widened ahead of the prompt kernel, and the room that they may take.  us without | with, prompts from slot 0, heads of 128:
//   32 heads on 8   24 tiles, 1536 tokens 43 | 52   32, 2048: 60 | 67    40, 2560: 91 | 88    64, 4096: 184 | 179   128, 8192: 637 | 557
//   32 on 32        16 tiles, 4096 tokens 190 | 193  24, 6144: 381 | 368  32, 8192: 649 | 590  40, 10240: 972 | 914
//   8 on 1          40 tiles, 1280 tokens 31 | 34    64, 2048: 42 | 42
// of 64: 32 on 8, 40 tiles 74 | 74, 64 tiles 151 | 155; 32 on 32, 40 tiles 817 | 806.  With four times as many older keys, 40 tiles: 32 on 8 672 | 609 (of 64: 580 | 564), 8 on 1
// 64 | 64.  The launch and the pass cost 3 to 9 us, and the gain grows with the steps of an SM, which the host knows from the tokens alone: tiles are the simple measure, off by up
// to 9 % for long unshared prompts below it and for short ones of few heads above it.
static constexpr int kWideFrom = 40;
static constexpr long long kWideBytes = 256ll << 20;
// Few row tiles share their keys out over more CTAs, as many as the SMs hold at a time (4, 3, 2 or 1 of a kind); a second kernel sums the parts.  The host does not
// know the sequences' lengths: a tile may have half as many CTAs again as its even share, and the kernel here shares by the
// lengths.  Up to 512 slots a second launch (3 us) costs more than it saves (1 sequence x 32 heads x 300 keys of 2048 slots, shared and summed: 10 us, of which the second kernel 3).
static Q8Plan q8_plan(const blr_q8_cache* c, int64_t n_tok, int heads) {
  Q8Plan a = {};
  a.rows = n_tok * (heads / c->kv_heads);
  a.nt = a.rows <= 8 ? 1 : a.rows <= 16 ? 2 : a.rows <= 32 ? 4 : 0;
  const int per = a.nt ? 8 * a.nt : kQ8PromptRows;
  a.q_tiles = (int)((a.rows + per - 1) / per);
  a.tiles = c->n_seq * c->kv_heads * a.q_tiles;
  a.room = (a.nt == 1 ? 4 : a.nt == 2 ? 3 : a.nt == 4 ? 2 : 1) * sm_count();
  long long ns = a.tiles > 0 ? a.room / a.tiles : 1;
  const long long least = a.nt ? 128 : 512, most = (c->slots + least - 1) / least;  // keys of a CTA
  if (a.nt && ns > 1 && c->n_seq > 1) ns += ns / 2;
  if (c->slots <= 512) ns = 1;
  if (ns > most) ns = most;
  a.ns = ns < 1 ? 1 : ns > kMaxSplits ? kMaxSplits : (int)ns;
  const long long wide = (c->slots + 127) / 128;
  if (a.nt == 0 && a.q_tiles >= kWideFrom && c->n_seq * c->kv_heads * wide * 512 * c->head_dim <= kWideBytes) a.wide_tiles = wide;
  return a;
}
static size_t q8_wide_bytes(const Q8Plan& a, const blr_q8_cache* c) { return (size_t)(c->n_seq * c->kv_heads * a.wide_tiles) * 512 * c->head_dim; }

template <bool E4M3, int HD, int NT>
static int launch_few(const Q8AttnParams& p, long long ctas, cudaStream_t st) {
  static bool configured[64] = {};
  constexpr int smem = few_smem_bytes<HD, NT>();
  DeviceInfo di;
  int rc;
  if ((rc = device_info(&di))) return rc;
  if (!configured[di.dev]) {
    BLR_CUDA_OK(cudaFuncSetAttribute(q8_attention_kernel<E4M3, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    configured[di.dev] = true;
  }
  return q8_launch(q8_attention_kernel<E4M3, HD, NT>, dim3((unsigned)ctas), kFewThreads, smem, st, p);
}

}  // namespace blr

using namespace blr;

extern "C" {

size_t blr_attention_q8_scratch_bytes(const blr_q8_cache* cache, int64_t n_tok, int heads) {
  if (!cache || cache->n_seq <= 0 || cache->kv_heads <= 0 || cache->slots <= 0 || n_tok <= 0 || heads <= 0 || heads % cache->kv_heads != 0) return 0;
  const Q8Plan a = q8_plan(cache, n_tok, heads);
  return q8_wide_bytes(a, cache) + (a.ns > 1 ? (size_t)cache->n_seq * cache->kv_heads * a.rows * a.ns * (cache->head_dim + 4) * sizeof(float) : 0);
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
  p.wide = a.wide_tiles > 0 ? static_cast<uint8_t*>(scratch) : nullptr, p.wide_tiles = (int)a.wide_tiles;
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + q8_wide_bytes(a, cache));
  p.scale_log2 = scale * 1.4426950408889634f;
  p.T = (int)n_tok, p.H = heads, p.G = heads / cache->kv_heads, p.rows = (int)a.rows, p.q_tiles = a.q_tiles, p.ns = a.ns, p.bf16 = dtype == BLR_DTYPE_BF16;
  p.n_bh = (int)(cache->n_seq * cache->kv_heads), p.n_seq = (int)cache->n_seq, p.room = a.room;
  p.status = ws == nullptr ? nullptr : static_cast<unsigned*>(ws) + 255;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.nt == 0) {
    rc = q8_launch_prompt(p, cache->head_dim, cache->code, st);
  } else {
    const long long ctas = a.tiles * a.ns;
#define BLR_Q8_ATTN(E4, HD) \
  (a.nt == 1 ? launch_few<E4, HD, 1>(p, ctas, st) : a.nt == 2 ? launch_few<E4, HD, 2>(p, ctas, st) : launch_few<E4, HD, 4>(p, ctas, st))
    if (cache->code == BLR_Q8_E4M3) rc = cache->head_dim == 128 ? BLR_Q8_ATTN(true, 128) : BLR_Q8_ATTN(true, 64);
    else rc = cache->head_dim == 128 ? BLR_Q8_ATTN(false, 128) : BLR_Q8_ATTN(false, 64);
#undef BLR_Q8_ATTN
  }
  if (rc || a.ns == 1) return rc;
  const long long total = cache->n_seq * cache->kv_heads * a.rows;
  const dim3 cgrid((unsigned)((total + 7) / 8));
  return cache->head_dim == 128 ? q8_launch(q8_combine_kernel<128>, cgrid, 256, 0, st, p, total) : q8_launch(q8_combine_kernel<64>, cgrid, 256, 0, st, p, total);
}

}  // extern "C"
