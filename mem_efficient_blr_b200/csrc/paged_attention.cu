// Causal attention of a sequence's newest tokens over a cache in pages (paged.cuh), a few rows at a time (sm_100a).
//
//   s_j = c (q . k_j),  p_j = 2^(s_j - m),  l = sum p_j,  o = sum p_j v_j / l   over the slots j that the row sees and that have a page, c = scale log2 e
// m is the largest score when it was last moved, which is where one exceeds it by 8: p_j is at most 2^8 and sums are fp32.
//
// A kv head's rows are its T tokens x (heads / kv_heads) query heads, token by token.  For 16 keys, which share a page, a warp computes S^T = K Q^T and O^T += V^T P^T
// with mma.sync: keys, then dimensions, as the 16 rows, 8 query rows as the columns, so that one query row costs what eight do.  ldmatrix brings K as it lies and V
// transposed; P^T comes out of S^T by movmatrix.  The products' operands have 16 bits: q, k and v as they are, p rounded to fp16 for fp16 values (2^-11 of itself, or 2^-25
// below 2^-14 of the heaviest); for bf16 values, where that would be 2^-8, as the sum of two bf16 numbers (2^-15), by a second product.
// What a row does not see has no part in any bit of its result, whatever lies there: see "values that are no numbers" below.
// Bound by HBM: a key and its value are 4 hd bytes, read once for 8 to 32 rows.  64 sequences x 2048 keys, 32 heads of 128, fp16: 299 us, 7.2 TB/s; 7 x 16 to 32 k keys, 32 heads on 8,
// bf16: 107 us, 6.2 TB/s.  1 x 2048 keys, 10.2 us for 34 MB: launch, table, pages, four groups a warp and the second kernel follow each other.  8 x 5 tokens, 30 us where the bytes take
// 15.8: eight warps an SM (247 registers hold three tiles' sums) issue in 31 % of the cycles and wait for their products; bf16 weights are multiplied twice.
#include "../../include/blr_b200.h"
#include "paged.cuh"
#include "tmap.h"

namespace blr {

static constexpr int kPagedMaxSplits = 64;

__device__ __forceinline__ uint32_t paged_transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// CTA (split, row tile, sequence and kv head): a warp takes every fourth group of 16 keys and brings them into a ring of its own with cp.async: no warp waits
// for another before the end.
static constexpr int kFewWarps = 4, kFewThreads = 32 * kFewWarps, kFewStages = 3;

template <int HD>
__host__ __device__ constexpr int paged_ring_bytes() {  // (the warps' sums lie over it in the end)
  constexpr int ring = kFewWarps * kFewStages * 64 * HD, sums = kFewWarps * 8 * (HD + 4) * 4;
  return ring > sums ? ring : sums;
}
template <int HD, int NT>
__host__ __device__ constexpr int paged_few_smem() { return paged_ring_bytes<HD>() + (NT > 2 ? NT * HD / 16 * 256 : 0); }

__device__ __forceinline__ void cp_async16_cg(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// Where the 16-byte piece c of row `row` of a group lies: eight rows' pieces c in eight different banks' groups.
template <int HD>
__device__ __forceinline__ uint32_t paged_place(int row, int c) { return row * 2 * HD + ((c ^ (row & 7)) << 4); }

template <bool BF16>
__device__ __forceinline__ bool no_number2(uint32_t w) {  // either half of the pair
  constexpr uint32_t ex = BF16 ? 0x7f80u : 0x7c00u;
  return (w & ex) == ex || (w >> 16 & ex) == ex;
}

template <bool BF16, int HD, int NT>
__global__ void __launch_bounds__(kFewThreads, HD == 64 && NT < 3 ? 4 : 2) paged_attention_kernel(const __grid_constant__ PagedAttnParams p) {
  constexpr int kSteps = HD / 16, kRows = 8 * NT, kPitch = HD + 4, kPieces = HD / 8, kGroup = 64 * HD, kHalf = 32 * HD;  // bytes of a group, of its keys
  constexpr bool kQShared = NT > 2;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float wm[kFewWarps][kRows], wl[kFewWarps][kRows];
  float(*const os)[8][kPitch] = reinterpret_cast<float(*)[8][kPitch]>(ring);
  uint2* const q_frag = reinterpret_cast<uint2*>(ring + paged_ring_bytes<HD>());  // [tile][step][lane]
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tiles = p.n_bh * p.q_tiles, split = blockIdx.x / tiles, tile = blockIdx.x - split * tiles, qt = tile % p.q_tiles, bh = tile / p.q_tiles;
  const int b = bh / p.c.kv_heads, h = bh - b * p.c.kv_heads, r0 = qt * kRows;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long start = p.start[b], count = p.n_new == nullptr ? p.T : min((long long)p.T, p.n_new[b]);
  const int keys = paged_seen_by(p, start, count, r0, r0 + kRows);
  const int share = p.ns > 1 ? paged_share(p, keys, kRows, kRows, 0, 16 * kFewWarps, lane) : max(keys, 1);
  const int k0 = (int)min((long long)keys, (long long)split * share), k1 = min(keys, k0 + min(share, keys - k0));
  if (p.ns > 1 && k0 >= k1) {  // no keys for this CTA: its rows say so
    if (threadIdx.x < kRows && r0 + (int)threadIdx.x < p.rows)
      *reinterpret_cast<float2*>(p.part + (((long long)bh * p.rows + r0 + threadIdx.x) * p.ns + split) * (HD + 4) + HD) = make_float2(-INFINITY, 0.f);
    return;
  }
  // groups of this warp: 16 keys from first + 64 j on
  const int first = k0 + 16 * warp, steps = first < k1 ? (k1 - first + 16 * kFewWarps - 1) / (16 * kFewWarps) : 0;
  const uint32_t base = smem_u32(ring) + warp * kFewStages * kGroup;
  // lane i keeps the page of group 32 n + i, and that of 32 groups later
  const int* const table = p.c.table + (long long)b * p.c.ld_table;
  auto page_of = [&](int j) { return j < steps ? table[(first + 16 * kFewWarps * j) >> p.c.page_log2] : -1; };
  int page_now = page_of(lane), page_next = page_of(32 + lane);
  const uint16_t *const kh = p.c.k + (long long)h * p.c.k_head + 8 * (lane % kPieces), *const vh = p.c.v + (long long)h * p.c.v_head + 8 * (lane % kPieces);
  auto bring = [&](int j, int page) {
    if (j < steps && (unsigned)page < (unsigned)p.c.pages) {
      const uint32_t to = base + (j % kFewStages) * kGroup;
      const int in = (first + 16 * kFewWarps * j) & ((1 << p.c.page_log2) - 1), c = lane % kPieces, row0 = lane / kPieces;
      const uint16_t *ka = kh + page * p.c.k_page + (in + row0) * p.c.k_slot, *va = vh + page * p.c.v_page + (in + row0) * p.c.v_slot;
#pragma unroll
      for (int i = 0; i < kPieces / 2; ++i) {
        const int row = row0 + i * (32 / kPieces);
        cp_async16_cg(to + paged_place<HD>(row, c), ka + i * (32 / kPieces) * p.c.k_slot);
        cp_async16_cg(to + kHalf + paged_place<HD>(row, c), va + i * (32 / kPieces) * p.c.v_slot);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int j = 0; j < kFewStages - 1; ++j) bring(j, __shfl_sync(0xffffffffu, page_now, j));

  float o[NT][kSteps][4] = {}, m[NT][2], l[NT][2] = {};
  {
    // ---- the query rows as fragments: dimensions 16 s + 2 t, + 1 and 8 behind them
    uint32_t qf[kQShared ? 1 : NT][kSteps][2];
    int lim[NT][2], lim_all = 0x7fffffff;  // keys below lim_all are masked for no row of the warp (places without a row do not count)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + 8 * n + g;
      const bool live = r < p.rows && r / p.G < count;
      const int tok = live ? r / p.G : 0;
      const uint16_t* row = p.q + ((long long)b * p.T + tok) * p.ldq + (long long)(h * p.G + (live ? r - tok * p.G : 0)) * HD + 2 * t;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t x = live ? *reinterpret_cast<const uint32_t*>(row + 16 * s) : 0u, y = live ? *reinterpret_cast<const uint32_t*>(row + 16 * s + 8) : 0u;
        if constexpr (kQShared) {
          if (warp == n % kFewWarps) q_frag[(n * kSteps + s) * 32 + lane] = make_uint2(x, y);
        } else {
          qf[n][s][0] = x, qf[n][s][1] = y;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rc = r0 + 8 * n + 2 * t + i;
        lim[n][i] = rc < p.rows ? paged_seen(start, count, rc / p.G, p.c.slots) : 0;
        if (lim[n][i] > 0) lim_all = min(lim_all, lim[n][i]);
      }
      m[n][0] = m[n][1] = -INFINITY;
    }
    if constexpr (kQShared) __syncthreads();
    lim_all = __reduce_min_sync(0xffffffffu, lim_all);

#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
      const int j0 = first + 16 * kFewWarps * j;
      const uint32_t at = base + (j % kFewStages) * kGroup;
      const bool there = (unsigned)__shfl_sync(0xffffffffu, page_now, j & 31) < (unsigned)p.c.pages;
      const int ahead = j + kFewStages - 1, page = __shfl_sync(0xffffffffu, (ahead ^ j) & 32 ? page_next : page_now, ahead & 31);
      asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 2) : "memory");
      __syncwarp();  // (everybody's pieces are there, and everybody has done with the group before, whose place the next one takes)
      bring(ahead, page);
      if ((j & 31) == 31) page_now = page_next, page_next = page_of(j + 33 + lane);
      if (!there) continue;
      // ---- S^T
      float sc[NT][4] = {};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        uint32_t a0, a1, a2, a3;
        ldsm_x4(at + paged_place<HD>(lane & 15, 2 * s + (lane >> 4)), a0, a1, a2, a3);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (kQShared) {
            const uint2 q = q_frag[(n * kSteps + s) * 32 + lane];
            mma_16816<BF16>(sc[n], a0, a1, a2, a3, q.x, q.y);
          } else {
            mma_16816<BF16>(sc[n], a0, a1, a2, a3, qf[n][s][0], qf[n][s][1]);
          }
        }
      }
      // ---- p
      const bool part = j0 + 16 > lim_all;
      uint32_t behind = 0;  // a bit for each tile of rows
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        bool up = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[n][i] *= p.scale_log2;
          if (part && j0 + g + 8 * (i >> 1) >= lim[n][i & 1]) sc[n][i] = -INFINITY;
          up |= sc[n][i] > m[n][i & 1] + 8.f;
        }
        behind |= up ? 1u << n : 0;
      }
      if (__any_sync(0xffffffffu, behind != 0)) {
        if (NT > 1) behind = __reduce_or_sync(0xffffffffu, behind);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (NT == 1 || (behind >> n & 1)) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float mx = fmaxf(sc[n][i], sc[n][i + 2]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
              if (mx > m[n][i] + 8.f) {  // (a row that the new keys do not ask stays as it is)
                const float down = ex2(m[n][i] - mx);
                m[n][i] = mx;
                l[n][i] *= down;
#pragma unroll
                for (int d = 0; d < kSteps; ++d) o[n][d][i] *= down, o[n][d][i + 2] *= down;
              }
            }
          }
        }
      }
      uint32_t pt[NT][2], pl[BF16 ? NT : 1][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float mu[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[n][i] = ex2(sc[n][i] - mu[i & 1]);
          l[n][i & 1] += sc[n][i];
        }
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          if constexpr (BF16) {
            // p cut to bf16, and what is missing, never 0 where p is not: an infinite value must not meet a 0
            const uint32_t hi = prmt(__float_as_uint(sc[n][2 * z]), __float_as_uint(sc[n][2 * z + 1]), 0x7632u);
            const float2 f = q8_up2<true>(hi);
            pt[n][z] = paged_transpose8x8(hi);
            pl[n][z] = paged_transpose8x8(q8_down2<true>(fmaf(sc[n][2 * z], 1.00000012f, -f.x), fmaf(sc[n][2 * z + 1], 1.00000012f, -f.y)));
          } else {
            pt[n][z] = paged_transpose8x8(q8_down2<false>(sc[n][2 * z], sc[n][2 * z + 1]));
          }
        }
      }
      // ---- values that are no numbers where some of the rows must not see them (seldom): the tensor core would multiply them with 0, so they are added here and 0 put in their place
      if (part) {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kPieces / 2; ++i) {
          uint32_t w[4];
          lds128(at + kHalf + paged_place<HD>(lane / kPieces + i * (32 / kPieces), lane % kPieces), w[0], w[1], w[2], w[3]);
          bad |= no_number2<BF16>(w[0]) || no_number2<BF16>(w[1]) || no_number2<BF16>(w[2]) || no_number2<BF16>(w[3]);
        }
        if (__any_sync(0xffffffffu, bad)) {
#pragma unroll 1
          for (int k = 0; k < 16; ++k) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float w[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float x = __shfl_sync(0xffffffffu, sc[n][i], (k & 7) * 4 + t), y = __shfl_sync(0xffffffffu, sc[n][i + 2], (k & 7) * 4 + t);
                w[i] = k < 8 ? x : y;
              }
#pragma unroll
              for (int d = 0; d < kSteps; ++d)
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                  uint16_t raw;
                  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(raw) : "r"(at + kHalf + paged_place<HD>(k, 2 * d + z) + 2 * g) : "memory");
                  const float v = BF16 ? __uint_as_float((uint32_t)raw << 16) : __half2float(__ushort_as_half(raw));
#pragma unroll
                  for (int i = 0; i < 2; ++i)
                    if (no_number2<BF16>(raw) && j0 + k < lim[n][i]) o[n][d][2 * z + i] = fmaf(w[i], v, o[n][d][2 * z + i]);
                }
            }
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < kPieces / 2; ++i) {
            const uint32_t place = at + kHalf + paged_place<HD>(lane / kPieces + i * (32 / kPieces), lane % kPieces);
            uint32_t w[4];
            lds128(place, w[0], w[1], w[2], w[3]);
#pragma unroll
            for (int x = 0; x < 4; ++x) w[x] &= (no_number2<BF16>(w[x] & 0xffffu) ? 0u : 0xffffu) | (no_number2<BF16>(w[x] & 0xffff0000u) ? 0u : 0xffff0000u);
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(place), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
          }
          __syncwarp();
        }
      }
      // ---- O^T
#pragma unroll
      for (int d = 0; d < kSteps; ++d) {
        uint32_t a0, a1, a2, a3;
        ldsm_x4_t(at + kHalf + paged_place<HD>((lane & 7) + 8 * (lane >> 4), 2 * d + (lane >> 3 & 1)), a0, a1, a2, a3);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_16816<BF16>(o[n][d], a0, a1, a2, a3, pt[n][0], pt[n][1]);
          if constexpr (BF16) mma_16816<BF16>(o[n][d], a0, a1, a2, a3, pl[n][0], pl[n][1]);
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
        if (lim[n][i] == 0) {  // (no token, or one that sees nothing: masked nowhere, left out here)
          m[n][i] = -INFINITY, l[n][i] = 0.f;
#pragma unroll
          for (int d = 0; d < kSteps; ++d) o[n][d][i] = o[n][d][i + 2] = 0.f;
        }
        if (g == 0) wm[warp][8 * n + 2 * t + i] = m[n][i], wl[warp][8 * n + 2 * t + i] = l[n][i];
      }
  }
  // ---- the warps' results meet, over the ring
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float M = -INFINITY;
      for (int w = 0; w < kFewWarps; ++w) M = fmaxf(M, wm[w][8 * n + 2 * t + i]);
      // (a NaN among the scores is in l, and there in all that follows)
      const float weight = m[n][i] == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : ex2(m[n][i] - M);
#pragma unroll
      for (int d = 0; d < kSteps; ++d)
#pragma unroll
        for (int z = 0; z < 2; ++z) os[warp][2 * t + i][16 * d + 8 * z + g] = o[n][d][2 * z + i] * weight;
    }
    __syncthreads();
    constexpr int kPer = 8 * HD / kFewThreads;  // values of a thread: 8 or 4 neighbours
    {
      const int row = threadIdx.x / (HD / kPer), d0 = (threadIdx.x - row * (HD / kPer)) * kPer, r = r0 + 8 * n + row;
      float Mr = -INFINITY, Lr = 0.f, sum[kPer] = {};
      for (int w = 0; w < kFewWarps; ++w) Mr = fmaxf(Mr, wm[w][8 * n + row]);
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float lw = wl[w][8 * n + row];
        if (!(lw == 0.f)) Lr += lw * (wm[w][8 * n + row] == -INFINITY ? 1.f : ex2(wm[w][8 * n + row] - Mr));
#pragma unroll
        for (int i = 0; i < kPer; i += 4) {
          const float4 x = *reinterpret_cast<const float4*>(&os[w][row][d0 + i]);
          sum[i] += x.x, sum[i + 1] += x.y, sum[i + 2] += x.z, sum[i + 3] += x.w;
        }
      }
      if (r < p.rows) {
        if (p.ns == 1) {
          const float inv = 1.f / Lr;
          const int tok = r / p.G;
          uint16_t* to = p.out + ((long long)b * p.T + tok) * p.ldo + (long long)(h * p.G + r - tok * p.G) * HD + d0;
          uint32_t x[kPer / 2];
#pragma unroll
          for (int i = 0; i < kPer; i += 2) x[i / 2] = Lr == 0.f ? 0u : q8_down2<BF16>(sum[i] * inv, sum[i + 1] * inv);
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
template <bool BF16, int HD>
__global__ void __launch_bounds__(256) paged_combine_kernel(const __grid_constant__ PagedAttnParams p, long long total) {
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
    w[i] = ml[i].y == 0.f ? -1.f : ml[i].x == -INFINITY ? 1.f : ex2(ml[i].x - M);  // -1: a split without keys, which has left its sums as they were; (a sum without a maximum is NaN)
    L += ml[i].y == 0.f ? 0.f : ml[i].y * w[i];
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
#pragma unroll 8
  for (int s = 0; s < p.ns; ++s) {
    const float ws = __shfl_sync(0xffffffffu, s < 32 ? w[0] : w[1], s & 31);
    if (ws < 0.f) continue;
    float x[HD / 32];
    if constexpr (HD == 128) {
      const float4 v = *reinterpret_cast<const float4*>(from + s * (HD + 4) + 4 * lane);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(from + s * (HD + 4) + 2 * lane);
      x[0] = v.x, x[1] = v.y;
    }
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) sum[i] += x[i] * ws;
  }
  const float inv = 1.f / L;
  const long long bh = row / p.rows, r = row - bh * p.rows, b = bh / p.c.kv_heads, h = bh - b * p.c.kv_heads, tok = r / p.G;
  uint16_t* to = p.out + (b * p.T + tok) * p.ldo + (h * p.G + r - tok * p.G) * HD + (HD / 32) * lane;
#pragma unroll
  for (int i = 0; i < HD / 32; i += 2) *reinterpret_cast<uint32_t*>(to + i) = L == 0.f ? 0u : q8_down2<BF16>(sum[i] * inv, sum[i + 1] * inv);
}

struct PagedPlan {
  int nt, q_tiles, ns, room;  // nt: column tiles of 8 rows of the kernel here, 0: the prompt kernel; ns: CTAs that may share a row tile's keys
  long long rows, tiles;
};
// Few row tiles share their keys out over more CTAs, as many as the SMs hold at a time; a second kernel sums the parts.  The host does not know the sequences' lengths: a
// tile may have twice its even share of CTAs and one, and the kernels share by the lengths (paged_share); CTAs that are left over say so and end.
// Both sides of each rule, us from a graph, 32 heads of 128 on 8 unless said otherwise, fp16, pages of 16:
//   24 rows in three column tiles: 8 sequences x 6 tokens, 4096 keys at most, 29.4; in four 32.0; in the prompt kernel 45.9 (one sequence x 6: 18.5 | 20.0 | 20.1; x 8 tokens, 8192 keys,
//     32 rows: 24.8 here, 21.9 there, but 8 sequences x 8 33.5 | 46.2).
//   No CTA has fewer keys than `least`: with one column tile 128 (1 x 1000 keys 8.4; 64: 9.2, 256: 9.3), with more 256 (1 x 6 tokens, 4096 keys 15.5; 128: 18.5), in the prompt kernel 256 (1 x 40
//     tokens, 2048 keys 21.4; 512: 25.3, 1024: 32.7).
//   Up to 512 slots are not split: 8 x 500 keys 8.6, split 10.5; up to 1024: 1 x 1000 keys 11.9, split 8.4.
//   Twice the even share: 8 x 5 tokens over 2000 to 4001 keys 30.2, without 33.0; 3 x 257 tokens, 16 heads of 64 on 4, 50.7 | 65.8; but 8 x 1 over 500 to 1000 keys 13.2 | 11.9.
static PagedPlan paged_plan(const blr_paged_cache* c, int64_t n_tok, int heads) {
  PagedPlan a = {};
  const int64_t slots = c->pages_per_seq * c->page;
  a.rows = n_tok * (heads / c->kv_heads);
  a.nt = a.rows <= 8 ? 1 : a.rows <= 16 ? 2 : a.rows <= 24 ? 3 : a.rows <= 32 || !paged_prompt_fits(c) ? 4 : 0;
  const int per = a.nt ? 8 * a.nt : kPagedPromptRows;
  a.q_tiles = (int)((a.rows + per - 1) / per);
  a.tiles = c->n_seq * c->kv_heads * a.q_tiles;
  a.room = (a.nt == 0 ? 1 : c->head_dim == 64 && a.nt < 3 ? 4 : 2) * sm_count();
  long long ns = a.tiles > 0 ? a.room / a.tiles : 1;
  const long long least = a.nt == 1 ? 128 : 256, most = (slots + least - 1) / least;  // keys of a CTA
  if (ns > 1 && (c->n_seq > 1 || a.q_tiles > 1)) ns = 2 * ns + 1;
  if (slots <= 512) ns = 1;
  if (ns > most) ns = most;
  a.ns = ns < 1 ? 1 : ns > kPagedMaxSplits ? kPagedMaxSplits : (int)ns;
  return a;
}

template <bool BF16, int HD, int NT>
static int launch_paged_few(const PagedAttnParams& p, long long ctas, cudaStream_t st) {
  static bool configured[64] = {};
  constexpr int smem = paged_few_smem<HD, NT>();
  DeviceInfo di;
  int rc;
  if ((rc = device_info(&di))) return rc;
  if (!configured[di.dev]) {
    BLR_CUDA_OK(cudaFuncSetAttribute(paged_attention_kernel<BF16, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    configured[di.dev] = true;
  }
  return q8_launch(paged_attention_kernel<BF16, HD, NT>, dim3((unsigned)ctas), kFewThreads, smem, st, p);
}

}  // namespace blr

using namespace blr;

extern "C" {

size_t blr_attention_paged_scratch_bytes(const blr_paged_cache* cache, int64_t n_tok, int heads) {
  if (!cache || cache->n_seq <= 0 || cache->kv_heads <= 0 || cache->pages_per_seq <= 0 || cache->page <= 0 || n_tok <= 0 || heads <= 0 || heads % cache->kv_heads != 0) return 0;
  const PagedPlan a = paged_plan(cache, n_tok, heads);
  return a.ns > 1 ? (size_t)cache->n_seq * cache->kv_heads * a.rows * a.ns * (cache->head_dim + 4) * sizeof(float) : 0;
}

int blr_attention_paged(const void* q, int64_t ldq, const blr_paged_cache* cache, const int64_t* start, const int64_t* n_new, int64_t n_tok, int heads, float scale,
                        int dtype, void* out, int64_t ldo, void* scratch, size_t scratch_bytes, void* ws, void* stream) {
  PagedAttnParams p = {};
  int rc;
  if ((rc = paged_view(cache, &p.c))) return rc;
  BLR_REQUIRE(dtype == BLR_DTYPE_F16 || dtype == BLR_DTYPE_BF16, BLR_ERR_ARG, "unknown dtype %d", dtype);
  BLR_REQUIRE(heads > 0 && heads % cache->kv_heads == 0, BLR_ERR_ARG, "attention_paged: %d heads are no multiple of %d kv heads", heads, cache->kv_heads);
  BLR_REQUIRE(n_tok >= 0 && n_tok < (1ll << 30) && n_tok * (heads / cache->kv_heads) < (1ll << 30), BLR_ERR_SHAPE, "attention_paged: n_tok = %lld", (long long)n_tok);
  BLR_REQUIRE((ldq | ldo) % 8 == 0, BLR_ERR_ARG, "attention_paged: row strides must be multiples of 8");
  BLR_REQUIRE(scale > 0.f && scale <= 2.0e38f, BLR_ERR_ARG, "attention_paged: the scale must be a positive number");
  if (cache->n_seq == 0 || n_tok == 0) return BLR_OK;
  BLR_REQUIRE(q && start && out, BLR_ERR_ARG, "null pointer");
  BLR_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(scratch)) & 15) == 0, BLR_ERR_ARG,
              "attention_paged needs 16-byte aligned pointers");
  const PagedPlan a = paged_plan(cache, n_tok, heads);
  const size_t need = blr_attention_paged_scratch_bytes(cache, n_tok, heads);
  BLR_REQUIRE(need == 0 || (scratch && scratch_bytes >= need), BLR_ERR_WORKSPACE, "attention_paged: scratch of %zu bytes is too small", scratch_bytes);
  BLR_REQUIRE(a.tiles * a.ns < (1ll << 31), BLR_ERR_SHAPE, "attention_paged: too many rows");
  p.q = static_cast<const uint16_t*>(q), p.out = static_cast<uint16_t*>(out);
  p.ldq = ldq, p.ldo = ldo;
  p.start = reinterpret_cast<const long long*>(start), p.n_new = reinterpret_cast<const long long*>(n_new);
  p.part = static_cast<float*>(scratch);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.T = (int)n_tok, p.H = heads, p.G = heads / cache->kv_heads, p.rows = (int)a.rows, p.q_tiles = a.q_tiles, p.ns = a.ns;
  p.n_bh = (int)(cache->n_seq * cache->kv_heads), p.n_seq = (int)cache->n_seq, p.room = a.room;
  p.status = ws == nullptr ? nullptr : static_cast<unsigned*>(ws) + 255;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == BLR_DTYPE_BF16;
  const long long ctas = a.tiles * a.ns;
  if (a.nt == 0) {
    rc = paged_launch_prompt(p, cache, bf, st);
  } else {
#define BLR_PAGED(BF, HD) \
  (a.nt == 1 ? launch_paged_few<BF, HD, 1>(p, ctas, st) : a.nt == 2 ? launch_paged_few<BF, HD, 2>(p, ctas, st) : a.nt == 3 ? launch_paged_few<BF, HD, 3>(p, ctas, st) : launch_paged_few<BF, HD, 4>(p, ctas, st))
    if (cache->head_dim == 128) rc = bf ? BLR_PAGED(true, 128) : BLR_PAGED(false, 128);
    else rc = bf ? BLR_PAGED(true, 64) : BLR_PAGED(false, 64);
#undef BLR_PAGED
  }
  if (rc || a.ns == 1) return rc;
  const long long total = cache->n_seq * cache->kv_heads * a.rows;
  const dim3 cgrid((unsigned)((total + 7) / 8));
  if (cache->head_dim == 128)
    return bf ? q8_launch(paged_combine_kernel<true, 128>, cgrid, 256, 0, st, p, total) : q8_launch(paged_combine_kernel<false, 128>, cgrid, 256, 0, st, p, total);
  return bf ? q8_launch(paged_combine_kernel<true, 64>, cgrid, 256, 0, st, p, total) : q8_launch(paged_combine_kernel<false, 64>, cgrid, 256, 0, st, p, total);
}

}  // extern "C"
