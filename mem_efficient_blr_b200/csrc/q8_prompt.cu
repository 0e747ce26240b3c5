// Causal attention of many rows over an 8-bit cache (q8.cuh) on tcgen05 / TMEM (sm_100a).  One CTA takes 256 rows of a kv head (tokens x query heads, token by
// token) and walks the keys in tiles of 128, warp-specialised:
//   warps 0-3, 4-7  softmax of rows 0-127 and 128-255, a thread per row: S from TMEM, P back over it as fp16 pairs, O rescaled there when it has to be
//   warps 8-11      widen the codes of the next keys and values to fp16 (exact) into shared memory, as tcgen05.mma reads them
//   warps 12-15     one thread of the first issues the products: S = Q K^T (both from shared memory), O += P V (P from TMEM)
// The scales stay out of the products: a group of 16 keys has one for its keys, which multiplies S in the exponent's argument, and one for its values, which multiplies p.
// A thread keeps its row's references for both (q8_attention.h) and moves them when a step's sum of p, or that times the largest factor, has outgrown them.
// A step is half a tile, 64 keys, and a half's S alternates between two places of TMEM: S0 S0 S1 S1 first, then PV0 S0 | PV1 S1 | ... with the S two steps ahead of the PV, into
// the place that the PV's P has left (P lies over the S that it was made of; one queue, so in order).  Neither half waits for the other's softmax, or for its own scores.
// O is rescaled, seldom, when the last PV is known to be done.
// Bounds, a step of 256 x 64 scores of heads of 128: 1280 cycles of tensor core (2 x 256 for PV, 2 x 384 for S, which reads both operands from shared memory for 64 columns)
// and 1024 of ex2 (16 a cycle).  It takes 2140: the softmaxes of both halves share the schedulers for 1270 from scores in registers to P in TMEM, and spend 870 on barriers,
// factors and TMEM's latency.  8192 tokens, 32 heads on 8: 565 us in a graph, 608 among calls from Python, 904 TFLOP/s.  (One reference of value scales for all rows of a CTA, which
// later keys decided, took 1 % less.  What follows was measured on that form.  Steps of 128 keys, which leave no room for a second S: 600; back to back 571 against 561; and 3 x 257 tokens over up to 6001
// keys of heads of 64 71 instead of 67.  All ex2 left out: 12 % less time.  With the next scores loaded between the two halves of a step's: 610.)  Tried on steps of 128 without
// gain: part of ex2 as a polynomial on the FMA pipe (1/8: 617 us, 3/8: 623), four softmax warpgroups of half a tile's width each (771), vs / R in the exponent instead of a
// multiplication (610), scores read twice instead of held (697).
// All waits are bounded; a time-out is noted in *status, the rows of that CTA come out as NaN, and the kernel frees its TMEM and ends.
#include <math_constants.h>

#include "../../include/blr_b200.h"
#include "prompt.cuh"
#include "q8_attention.h"
#include "tmap.h"

namespace blr {

static constexpr int kKeys = 128, kStepKeys = 64;
// Threads, and registers of a thread at launch and from then on of the softmax warps (8), the widening ones (4, none where the codes have been widened) and the last
// four: setmaxnreg waits for ever for registers that the block was not launched with.
template <bool WIDE>
struct Split {
  static constexpr int kThreads = WIDE ? 384 : 512, kLaunch = WIDE ? 168 : 128, kSoftmax = WIDE ? 216 : 176, kWiden = 104, kIssue = 56;
  static_assert(8 * kSoftmax + (WIDE ? 0 : 4 * kWiden) + 4 * kIssue <= kThreads / 32 * kLaunch, "more registers than the block has");
};

// A thread has the 64 scores of its row for a step in registers, x, in four groups of 16 keys.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The factors of two groups: cg of their scores, fg of their weights.  Masked scores are -inf and their weights 0: a group that is masked as a whole has factors of its own for
// that (its scales may be NaN), and a key scale of 0 makes way for a number that its scores vanish under.
__device__ __forceinline__ void factors32(uint32_t fac, int c, float factor, float D, bool part, int left, float (&cg)[2], float (&fg)[2]) {
  uint64_t k, v;
  asm volatile("ld.shared.b64 %0, [%1];" : "=l"(k) : "r"(fac + 8 * c) : "memory");
  asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(fac + 32 + 8 * c) : "memory");
  unpair(mul2(k, pair(factor, factor)), cg[0], cg[1]);
  unpair(mul2(v, pair(D, D)), fg[0], fg[1]);
#pragma unroll
  for (int g = 0; g < 2; ++g) fg[g] = min_nan(fg[g], 3.402823466e38f);  // (a finite scale: no 0 times infinity)
  if (part) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      if (16 * g >= left) cg[g] = 1.f, fg[g] = 0.f;
      if (cg[g] == 0.f) cg[g] = 1e-37f;
    }
  }
}
// Moves a row's references to the maxima of its groups (q8_attention.h).
__device__ __forceinline__ void move_to(const uint32_t (&x)[2][32], uint32_t fac, float factor, bool part, int left, float& m, float& D, float& down, float& corr) {
  float peak[4], to = m;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float cg[2], fg[2];
    factors32(fac, c, factor, D, part, left - 32 * c, cg, fg);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      float top = __uint_as_float(x[c][16 * g]);
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, __uint_as_float(x[c][16 * g + i]));
      peak[2 * c + g] = ceilf(top * cg[g]);
      to = fmaxf(to, peak[2 * c + g]);
    }
  }
  if (to == -INFINITY) {
    // (no number among the row's first keys.  It counts as begun, or it would ask for a move at every step, and the rows beside it would not come to theirs; a number that follows is above
    // this by more than any sum has room for, and moves it)
    m = -3.402823466e38f;
    return;
  }
  uint32_t vs[4];
  lds128(fac + 32, vs[0], vs[1], vs[2], vs[3]);
  float heavy = -INFINITY;
#pragma unroll
  for (int g = 0; g < 4; ++g) heavy = fmaxf(heavy, peak[g] - to + q8_above(__uint_as_float(vs[g])));
  q8_move(to, heavy, m, D, down, corr);
}
// p = 2^(s - mu), and P = p vs D as fp16 pairs over the scores in TMEM; returns the sum of p, and the largest of the factors vs D.
__device__ __forceinline__ float weights(uint32_t s_at, const uint32_t (&x)[2][32], uint32_t fac, float factor, float D, float mu, bool part, int left, float& most) {
  uint64_t sum[2] = {0, 0};
  const uint64_t neg = pair(-mu, -mu);
  most = 0.f;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float cg[2], fg[2];
    uint32_t y[16];
    factors32(fac, c, factor, D, part, left - 32 * c, cg, fg);
    most = fmaxf(most, fmaxf(fg[0], fg[1]));
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const uint64_t c2 = pair(cg[g], cg[g]), f2 = pair(fg[g], fg[g]);
#pragma unroll
      for (int i = 16 * g; i < 16 * g + 16; i += 2) {
        float a, b, v, w;
        unpair(fma2(pair(__uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1])), c2, neg), a, b);
        const uint64_t e = pair(ex2(a), ex2(b));
        sum[g] = add2(sum[g], e);
        unpair(mul2(e, f2), v, w);
        y[i / 2] = pack_half2(v, w);
      }
    }
    tmem_st16(s_at + 16 * c, y);
  }
  float a, b;
  unpair(add2(sum[0], sum[1]), a, b);
  return a + b;
}

// What a CTA works on.  (Asked for anew where it is needed: kept in registers across the loops it would push others out of them.)
struct Place {
  int split, bh, b, h, r0;
};
__device__ __forceinline__ Place place_of(const Q8AttnParams& p) {
  int cta;
  asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(cta));
  Place a;
  const int tile = cta / p.ns;
  a.split = cta - tile * p.ns;
  a.bh = tile % p.n_bh;
  a.r0 = (p.q_tiles - 1 - tile / p.n_bh) * kQ8PromptRows;  // the last rows have the most keys: their CTAs come first
  a.b = a.bh / p.c.kv_heads;
  a.h = a.bh - a.b * p.c.kv_heads;
  return a;
}

// 128 rows of hd codes on their way to shared memory: a thread has 16 neighbouring codes of every (128 / kPasses)th row.
template <int HD>
struct Codes {
  static constexpr int kChunks = HD / 16, kPasses = kChunks, kStep = 128 / kPasses;
  uint4 w[kPasses];
  __device__ __forceinline__ void load(const uint8_t* head, int key0, int last, int idx) {
    const int c = idx % kChunks, row = idx / kChunks;
    const uint8_t* const at = head + (long long)(key0 + row) * HD + 16 * c;
    if (key0 + kKeys - 1 <= last) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) w[i] = *reinterpret_cast<const uint4*>(at + i * kStep * HD);
    } else {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {  // (behind the last slot: anything, as long as it is read inside the cache; masked as keys, zeros as values)
        const int over = max(0, key0 + row + i * kStep - last);
        w[i] = *reinterpret_cast<const uint4*>(at + (i * kStep - over) * HD);
      }
    }
  }
  // Rows of 64 values, 128 bytes, swizzled as tcgen05.mma expects them; rows from `live` on become zeros.
  template <bool E4M3>
  __device__ __forceinline__ void store(uint32_t to, int live, int idx) const {
    const int c = idx % kChunks, row0 = idx / kChunks, at = (c & 3) * 2, flip = HD == 128 ? c >> 2 : 0;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int row = row0 + i * kStep;
      const uint32_t ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
      uint32_t h[8];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint32_t b = q8_bias<E4M3>(ws[n]);
        h[2 * n] = q8_half2<E4M3>(b, false), h[2 * n + 1] = q8_half2<E4M3>(b, true);
      }
      if (row >= live)
#pragma unroll
        for (int n = 0; n < 8; ++n) h[n] = 0;
      const uint32_t base = to + (c >> 2) * 16384 + row * 128, x = base + (((at + flip) ^ (row & 7)) << 4), y = base + (((at + 1 - flip) ^ (row & 7)) << 4);
      // (the lanes of a row write all its eight 16-byte places at once, so that no two meet in a bank)
      if (flip) {
        sts128(x, h[4], h[5], h[6], h[7]);
        sts128(y, h[0], h[1], h[2], h[3]);
      } else {
        sts128(x, h[0], h[1], h[2], h[3]);
        sts128(y, h[4], h[5], h[6], h[7]);
      }
    }
  }
};

template <bool E4M3, int HD, bool WIDE>
__global__ void __launch_bounds__(Split<WIDE>::kThreads, 1) q8_prompt_kernel(const __grid_constant__ Q8AttnParams p) {
  constexpr int kLast = WIDE ? 8 : 12;  // the first of the last four warps
  extern __shared__ __align__(1024) uint8_t prompt_raw[];
  __shared__ __align__(16) float factors[4][16];
  constexpr uint32_t kTile = 128 * HD * 2;
  const uint32_t base = (smem_u32(prompt_raw) + 1023u) & ~1023u;
  const uint32_t qs = base, ks = base + 2 * kTile, vs = base + 4 * kTile, bars = base + 6 * kTile;
  const uint32_t kfull = bars, vfull = bars + 16, kempty = bars + 32, vempty = bars + 48, sfull = bars + 64, pfull = bars + 96, done = bars + 128, cfull = bars + 160;  // sfull, pfull, done: [half][place]
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int aborted;
  volatile int* const abort_flag = &aborted;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(kfull + 8 * i, WIDE ? 1 : 4);
      mbar_init(vfull + 8 * i, WIDE ? 1 : 4);
      mbar_init(kempty + 8 * i, 1);
      mbar_init(vempty + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(sfull + 8 * i, 1);
      mbar_init(pfull + 8 * i, 4);
      mbar_init(done + 8 * i, 1);
      mbar_init(cfull + 8 * i, 1);
    }
    mbar_init_fence();
  }
  if (warp == kLast) tmem_alloc(smem_u32(&tmem_slot), 512);

  asm volatile("griddepcontrol.wait;" ::: "memory");
  int keys, k0, n0, n1, lim = 0;
  float factor = p.scale_log2;
  const int wg = warp >> 2;
  {
    const Place at = place_of(p);
    const long long start = p.start[at.b], count = p.n_new == nullptr ? p.T : min((long long)p.T, p.n_new[at.b]);
    const int keys0 = q8_seen_by(p, start, count, at.r0, at.r0 + 128), keys1 = q8_seen_by(p, start, count, at.r0 + 128, at.r0 + 256);
    keys = max(keys0, keys1);
    const int share = ((keys + p.ns - 1) / p.ns + kKeys - 1) / kKeys * kKeys, k1 = min(keys, (at.split + 1) * share);
    k0 = min(keys, at.split * share);
    n0 = max(0, min(keys0, k1) - k0 + kStepKeys - 1) / kStepKeys;
    n1 = max(0, min(keys1, k1) - k0 + kStepKeys - 1) / kStepKeys;

  // ---- a softmax thread's row of q, as fp16
  const int row_i = (int)threadIdx.x & 127, r = at.r0 + (int)threadIdx.x;
  if (warp < 8) {
    const bool live = r < p.rows && r / p.G < count;
    const int tok = live ? r / p.G : 0;
    const uint4* const row = reinterpret_cast<const uint4*>(p.q + ((long long)at.b * p.T + tok) * p.ldq + (long long)(at.h * p.G + (live ? r - tok * p.G : 0)) * HD);
    float mul = 1.f;
    if (live) lim = q8_seen(start, count, tok, p.c.slots);
    if (live && p.bf16) {
      uint32_t most = 0;
#pragma unroll 4
      for (int i = 0; i < HD / 8; ++i) {
        const uint4 x = row[i];
        const uint32_t ws[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int n = 0; n < 4; ++n) most = max(most, max(ws[n] & 0x7fffu, (ws[n] >> 16) & 0x7fffu));
      }
      const int up = q8_row_up(most << 16, 1);
      mul = __uint_as_float((uint32_t)up << 23);
      factor *= __uint_as_float((uint32_t)(254 - up) << 23);
    }
    const uint32_t to = qs + wg * kTile + row_i * 128;
#pragma unroll 4
    for (int i = 0; i < HD / 8; ++i) {
      const uint4 x = live ? row[i] : make_uint4(0, 0, 0, 0);
      uint32_t ws[4] = {x.x, x.y, x.z, x.w};
      if (p.bf16) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float2 f = q8_up2<true>(ws[n]);
          ws[n] = pack_half2(f.x * mul, f.y * mul);
        }
      }
      sts128(to + (i >> 3) * 16384 + (((i & 7) ^ (row_i & 7)) << 4), ws[0], ws[1], ws[2], ws[3]);
    }
    fence_proxy_async_smem();
  }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int halves = max(n0, n1), steps = (halves + 1) / 2;  // (n0, n1, halves: of 64 keys; steps: tiles of 128)

  // (Few spills, 4 to 20 bytes in four of the six instances: what shared memory leaves of L1 does not keep them, and a reload from L2 inside a loop costs more than it saves.)
  // A step's factors: ks and vs of 8 groups of 16 keys (an infinite vs as a NaN).  One warp brings them, four steps deep (a step's are free when the S of the step after it
  // is done, and that warp is two steps ahead of that at most).
  float next_scale = 0.f;
  auto scale_at = [&](int j) {
    const float* const scales = (lane < 8 ? p.c.k_scale : p.c.v_scale) + (long long)place_of(p).bh * p.c.n_blocks;
    return scales[min((k0 + j * kKeys + 16 * (lane & 7)) >> p.c.block_log2, p.c.n_blocks - 1)];
  };
  auto make_factors = [&](int j) {
    const float scale = next_scale;
    if (j + 1 < steps) next_scale = scale_at(j + 1);
    if (lane < 16) factors[j & 3][lane] = lane < 8 || scale <= 3.402823466e38f ? scale : CUDART_NAN_F;
    __syncwarp();
    if (lane == 0) mbar_arrive(cfull + 8 * (j & 3));
  };
  if (warp >= kLast) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Split<WIDE>::kIssue));
    if (WIDE && warp == kLast + 1) {
      // tiles of widened keys and values as they are to lie in shared memory
      if (elect_one()) {
        const uint8_t* const from = p.wide + ((long long)place_of(p).bh * p.wide_tiles + k0 / kKeys) * 2 * kTile;
#pragma unroll 1
        for (int j = 0; j < steps; ++j) {
          const uint32_t s = j & 1, parity = ((j >> 1) & 1) ^ 1;
          if (j >= 2 && !mbar_wait(kempty + 8 * s, parity, abort_flag)) break;
          mbar_arrive_expect_tx(kfull + 8 * s, kTile);
          bulk_load(ks + s * kTile, from + (long long)j * 2 * kTile, kTile, kfull + 8 * s);
          if (j >= 2 && !mbar_wait(vempty + 8 * s, parity, abort_flag)) break;
          mbar_arrive_expect_tx(vfull + 8 * s, kTile);
          bulk_load(vs + s * kTile, from + (long long)j * 2 * kTile + kTile, kTile, vfull + 8 * s);
        }
      }
      __syncwarp();
    } else if (WIDE && warp == kLast + 2) {
      if (steps > 0) next_scale = scale_at(0);
#pragma unroll 1
      for (int j = 0; j < steps; ++j) {
        if (j >= 2 && !__all_sync(0xffffffffu, mbar_wait(kempty + 8 * (j & 1), ((j >> 1) & 1) ^ 1, abort_flag))) break;
        make_factors(j);
      }
    }
    if (warp == kLast && elect_one()) {
      const uint32_t id_s = umma_idesc(false, false, false, 128, kStepKeys), id_o = umma_idesc(false, false, true, 128, HD);
      auto product_s = [&](int i, int u) {
        uint32_t q_at = qs + i * kTile;
        asm volatile("" : "+r"(q_at));  // (sixteen descriptors kept across the loop would be spilled)
        const uint64_t a = umma_smem_desc(q_at, 16, 1024), k = umma_smem_desc(ks + ((u >> 1) & 1) * kTile + (u & 1) * 8192, 16, 1024);
        const uint32_t to = tmem + 128 * i + 64 * (u & 1);
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) umma_f16(to, a + (s >> 2) * 1024 + (s & 3) * 2, k + (s >> 2) * 1024 + (s & 3) * 2, id_s, s != 0);
        umma_commit(sfull + 16 * i + 8 * (u & 1));
      };
      auto product_o = [&](int i, int u) {
        const uint64_t v = umma_smem_desc(vs + ((u >> 1) & 1) * kTile + (u & 1) * 8192, 16384, 1024);
        const uint32_t from = tmem + 128 * i + 64 * (u & 1);
#pragma unroll
        for (int s = 0; s < kStepKeys / 16; ++s) umma_f16_ts(tmem + 256 + 128 * i, from + 8 * s, v + 128 * s, id_o, (u | s) != 0);
        umma_commit(done + 16 * i + 8 * (u & 1));  // (one for each place: behind the last P two products may be under way, and a barrier's parity tells two phases apart, not three)
      };
      bool ok = halves > 0 && mbar_poll(kfull, 0, abort_flag);
      if (ok) {
        tc_fence_after();
        if (n0 > 0) product_s(0, 0);
        if (n0 > 1) product_s(0, 1);
        if (n1 > 0) product_s(1, 0);
        if (n1 > 1) product_s(1, 1);
        umma_commit(kempty);
      }
#pragma unroll 1
      for (int u = 0; ok && u < halves; ++u) {
        const int j = u >> 1, next = u + 2;
        // (written out: a loop around the products costs the elected thread hundreds of cycles a step)
        if ((u & 1) == 0) {
          if (!mbar_poll(vfull + 8 * (j & 1), (j >> 1) & 1, abort_flag)) { ok = false; break; }
          if (next < halves && !mbar_poll(kfull + 8 * ((j + 1) & 1), ((j + 1) >> 1) & 1, abort_flag)) { ok = false; break; }
        }
        if (u < n0) {
          if (!mbar_poll(pfull + 8 * (u & 1), j & 1, abort_flag)) { ok = false; break; }
          tc_fence_after();
          product_o(0, u);
          if (next < n0) product_s(0, next);
        }
        if (u < n1) {
          if (!mbar_poll(pfull + 16 + 8 * (u & 1), j & 1, abort_flag)) { ok = false; break; }
          tc_fence_after();
          product_o(1, u);
          if (next < n1) product_s(1, next);
        }
        if (u & 1) {
          if (next < halves) umma_commit(kempty + 8 * ((j + 1) & 1));
          umma_commit(vempty + 8 * (j & 1));
        }
      }
    }
    __syncwarp();
  } else if (!WIDE && warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Split<WIDE>::kWiden));
    const int idx = threadIdx.x & 127, last = p.c.slots - 1;
    const long long head = (long long)place_of(p).bh * p.c.slots * HD;
    const uint8_t *const kh = p.c.k + head, *const vh = p.c.v + head;
    if (warp == 8 && steps > 0) next_scale = scale_at(0);
    Codes<HD> kc, vc;
    if (steps > 0) kc.load(kh, k0, last, idx), vc.load(vh, k0, last, idx);
#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
      const uint32_t s = j & 1, parity = ((j >> 1) & 1) ^ 1;
      if (j >= 2 && !__all_sync(0xffffffffu, mbar_wait(kempty + 8 * s, parity, abort_flag))) break;
      if (warp == 8) make_factors(j);
      kc.template store<E4M3>(ks + s * kTile, 128, idx);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(kfull + 8 * s);
      if (j + 1 < steps) kc.load(kh, k0 + (j + 1) * kKeys, last, idx);
      if (j >= 2 && !__all_sync(0xffffffffu, mbar_wait(vempty + 8 * s, parity, abort_flag))) break;
      vc.template store<E4M3>(vs + s * kTile, keys - k0 - j * kKeys, idx);  // (slots that nobody wrote may hold anything)
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(vfull + 8 * s);
      if (j + 1 < steps) vc.load(vh, k0 + (j + 1) * kKeys, last, idx);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Split<WIDE>::kSoftmax));
    const int n = wg ? n1 : n0;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, o_at = tmem + lanes + 256 + 128 * wg;
    float m = -INFINITY, l = 0.f, D = 1.f;
    const int lim_all = __reduce_min_sync(0xffffffffu, lim);
    bool ok = true;
#pragma unroll 1
    for (int u = 0; u < n; ++u) {
      const int j = u >> 1, key0 = k0 + u * kStepKeys;
      const uint32_t s_at = tmem + lanes + 128 * wg + 64 * (u & 1);
      const bool part = key0 + kStepKeys > lim_all;  // some of these keys are masked for a row of the warp
      if ((u & 1) == 0 && !__all_sync(0xffffffffu, mbar_wait(cfull + 8 * (j & 3), (j >> 2) & 1, abort_flag))) { ok = false; break; }
      const uint32_t fac = smem_u32(factors[j & 3]) + 16 * (u & 1);  // (of the step's four groups; those of their values 32 bytes behind)
      if (!__all_sync(0xffffffffu, mbar_wait(sfull + 16 * wg + 8 * (u & 1), j & 1, abort_flag))) { ok = false; break; }
      tc_fence_after();
      uint32_t x[2][32];
      tmem_ld32(s_at, x[0]);
      tmem_ld32(s_at + 32, x[1]);
      tmem_ld_wait();
      tmem_ready(x[0]);
      tmem_ready(x[1]);
      if (part) {
        mask32(x[0], lim - key0);
        mask32(x[1], lim - key0 - 32);
      }
      // against the references so far, which are seldom left behind: a sum above 2^11, or one that may bring a P above 2^15, tells of it, and all is done once more.  The rows that
      // ask for it move theirs, the others come out as they were.
      float total = 0.f;
      bool ask = m == -INFINITY && lim > key0;  // (a row's first keys)
#pragma unroll 1
      for (bool moved = __any_sync(0xffffffffu, ask);; moved = true) {
        if (moved) {
          float down = 1.f, corr = 1.f;
          if (ask) move_to(x, fac, factor, part, lim - key0, m, D, down, corr);
          __syncwarp();  // (what follows in TMEM is the whole warp's)
          l *= down;
          if (u > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
            if (!__all_sync(0xffffffffu, mbar_wait(done + 16 * wg + 8 * ((u - 1) & 1), ((u - 1) >> 1) & 1, abort_flag))) { ok = false; break; }
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < HD / 8; ++k) {
              uint32_t o[8];
              tmem_ld8(o_at + 8 * k, o);
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
              tmem_st8(o_at + 8 * k, o);
            }
          }
        }
        float most;
        total = weights(s_at, x, fac, factor, D, m == -INFINITY ? 0.f : m, part, lim - key0, most);
        ask = total > 2048.f || total * most > 32768.f;
        if (moved || !__any_sync(0xffffffffu, ask)) break;
      }
      if (!ok) break;
      l += total;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull + 16 * wg + 8 * (u & 1));
    }
    if (ok && n > 0 && !__all_sync(0xffffffffu, mbar_wait(done + 16 * wg + 8 * ((n - 1) & 1), ((n - 1) >> 1) & 1, abort_flag))) ok = false;
    tc_fence_after();
    const Place at = place_of(p);
    const int r = at.r0 + (int)threadIdx.x;
    const bool live = r < p.rows;
    const float fin = !ok ? CUDART_NAN_F : p.ns > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l, unit = q8_unit(D);
    const int tok = live ? r / p.G : 0;
    uint16_t* const to = p.out + ((long long)at.b * p.T + tok) * p.ldo + (long long)(at.h * p.G + r - tok * p.G) * HD;
    float* const to32 = p.part + (((long long)at.bh * p.rows + r) * p.ns + at.split) * (HD + 4);
#pragma unroll 1
    for (int c = 0; c < HD / 32; ++c) {
      __syncwarp();  // (rows that are none leave a turn early, and the load is the whole warp's)
      uint32_t x[32];
      if (n > 0 && ok) {
        tmem_ld32(o_at + 32 * c, x);
        tmem_ld_wait();
        tmem_ready(x);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = 0;
      }
      if (!live) continue;
#pragma unroll
      for (int i = 0; i < 32; ++i)  // (a row that sees nothing: zeros, whatever its products were)
        x[i] = ok && l == 0.f ? 0u : __float_as_uint(__uint_as_float(x[i]) * fin * unit);
      if (p.ns > 1) {
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<float4*>(to32 + 32 * c + i) = make_float4(__uint_as_float(x[i]), __uint_as_float(x[i + 1]), __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
      } else {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          uint32_t o[4];
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            const float u = __uint_as_float(x[i + 2 * z]), v = __uint_as_float(x[i + 2 * z + 1]);
            o[z] = p.bf16 ? q8_down2<true>(u, v) : q8_down2<false>(u, v);
          }
          *reinterpret_cast<uint4*>(to + 32 * c + i) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
    }
    if (live && p.ns > 1) to32[HD] = m, to32[HD + 1] = ok ? l : CUDART_NAN_F;
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 1u);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // (products in flight end before their operands' memory is given back)
  }
  if (warp == kLast) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The codes of 128 slots of a head as fp16, in the very order that a tile has in shared memory; zeros behind a sequence's last slot.  Where a tile of keys is read by
// several CTAs it is widened once like this, instead of by each: 2 bytes a code written and read through L2.
template <bool E4M3, int HD>
__global__ void __launch_bounds__(256) q8_widen_kernel(const __grid_constant__ Q8AttnParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kChunks = HD / 16;
  const int tile = blockIdx.x % p.wide_tiles, bh = blockIdx.x / p.wide_tiles, b = bh / p.c.kv_heads, key0 = tile * kKeys;
  const long long count = p.n_new == nullptr ? p.T : min((long long)p.T, p.n_new[b]);
  const int keys = q8_seen_by(p, p.start[b], count, 0, p.rows);
  if (key0 >= keys) return;
  uint8_t* const to = p.wide + ((long long)bh * p.wide_tiles + tile) * 2 * (128 * HD * 2);
#pragma unroll
  for (int i = threadIdx.x; i < 2 * 128 * kChunks; i += 256) {
    const int which = i / (128 * kChunks), at = i - which * (128 * kChunks), row = at / kChunks, c = at - row * kChunks;
    uint4 w = make_uint4(0, 0, 0, 0);
    const bool live = key0 + row < keys;
    if (live) w = *reinterpret_cast<const uint4*>((which ? p.c.v : p.c.k) + ((long long)bh * p.c.slots + key0 + row) * HD + 16 * c);
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    uint32_t h[8];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint32_t v = q8_bias<E4M3>(ws[n]);
      h[2 * n] = live ? q8_half2<E4M3>(v, false) : 0u, h[2 * n + 1] = live ? q8_half2<E4M3>(v, true) : 0u;
    }
    uint8_t* const line = to + which * (128 * HD * 2) + (c >> 2) * 16384 + row * 128;
    *reinterpret_cast<uint4*>(line + ((((c & 3) * 2) ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(line + ((((c & 3) * 2 + 1) ^ (row & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
  }
}

template <bool E4M3, int HD, bool WIDE>
static int launch_prompt(const Q8AttnParams& p, cudaStream_t stream) {
  static bool configured[64] = {};
  DeviceInfo di;
  int rc;
  if ((rc = device_info(&di))) return rc;
  const int smem = 6 * 128 * HD * 2 + 1024 + 256 < 120 * 1024 ? 120 * 1024 : 6 * 128 * HD * 2 + 1024 + 256;  // one CTA per SM: a second one would only wait for TMEM
  if (!configured[di.dev]) {
    BLR_CUDA_OK(cudaFuncSetAttribute(q8_prompt_kernel<E4M3, HD, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaFuncAttributes fa;
    BLR_CUDA_OK(cudaFuncGetAttributes(&fa, q8_prompt_kernel<E4M3, HD, WIDE>));
    BLR_REQUIRE(fa.numRegs == Split<WIDE>::kLaunch, BLR_ERR_UNSUPPORTED, "the prompt kernel was built with %d registers, its split is made for %d", fa.numRegs,
                Split<WIDE>::kLaunch);
    configured[di.dev] = true;
  }
  return q8_launch(q8_prompt_kernel<E4M3, HD, WIDE>, dim3((unsigned)p.n_bh * p.q_tiles * p.ns), Split<WIDE>::kThreads, smem, stream, p);
}

int q8_launch_prompt(const Q8AttnParams& p, int head_dim, int code, cudaStream_t stream) {
  const bool e4 = code == BLR_Q8_E4M3;
  if (p.wide == nullptr) {
    if (head_dim == 128) return e4 ? launch_prompt<true, 128, false>(p, stream) : launch_prompt<false, 128, false>(p, stream);
    return e4 ? launch_prompt<true, 64, false>(p, stream) : launch_prompt<false, 64, false>(p, stream);
  }
  auto widen = [&](auto kernel) { return q8_launch(kernel, dim3((unsigned)p.n_bh * p.wide_tiles), 256, 0, stream, p); };
  const int rc = head_dim == 128 ? (e4 ? widen(q8_widen_kernel<true, 128>) : widen(q8_widen_kernel<false, 128>))
                                 : (e4 ? widen(q8_widen_kernel<true, 64>) : widen(q8_widen_kernel<false, 64>));
  if (rc) return rc;
  return head_dim == 128 ? launch_prompt<false, 128, true>(p, stream) : launch_prompt<false, 64, true>(p, stream);
}

}  // namespace blr
