// Causal attention of many rows over a cache in pages (paged.cuh) on tcgen05 / TMEM (sm_100a).  One CTA takes 256 rows of a kv head (tokens x query heads, token by
// token) and walks the keys in tiles of 128, warp-specialised:
//   warps 0-3, 4-7  softmax of rows 0-127 and 128-255, a thread per row: S from TMEM, P back over it as 16-bit pairs, O rescaled there when it has to be
//   warp 8          one thread issues the products: S = Q K^T (both from shared memory), O += P V (P from TMEM)
//   warp 9          looks up the pages of the next tiles and has them copied, a box of a page's slots and 64 dimensions at a time; "no page" is a box outside the pool, zeros
//   warps 10, 11    look through the values of the tiles that not all rows see: what is no number there, and what lies behind the last key, becomes 0 for the product
//                   (which would multiply it with 0 for the rows that must not see it), and is added by the rows that do see it in the end
// p = 2^(s - m): m, a whole number, is the row's own and moves when a step's sum of p has outgrown 2^11, so that nothing but P is rounded (fp16: 2^-11 of itself, or
// 2^-25 below 2^-14 of the heaviest; bf16: 2^-8), and no bit of a row depends on what it does not see.  P has the values' type because the product's operands must have one type; what bf16
// leaves of it (2^-15, as the kernel for few rows has it) would be a second product, 524 cycles to a step's 1440, and as many conversions again in the softmax, which is what a step waits for.
// A step is half a tile, 64 keys, and a half's S alternates between two places of TMEM: S0 S0 S1 S1 first, then PV0 S0 | PV1 S1 | ... with the S two steps ahead of the PV, into
// the place that the PV's P has left (P lies over the S that it was made of; one queue, so in order).  Neither half waits for the other's softmax, or for its own scores.
// O is rescaled, seldom, when the last PV is known to be done.
// 8192 tokens, 32 heads of 128 on 8, fp16: 530 us, 1037 TFLOP/s, for some 10 ms; 600 to 615 us when it goes on and the power limit lowers the clock.  A step's products take 1440 cycles (S has 64
// columns, whose Q and K come out of shared memory: 476 of a half's 720) and a step 2000: the two halves' softmaxes, which run side by side (1470 for the weights of both, 500 from their
// scores to the weights and from the weights to the products).  Tried: the halves by turns 713 us; S of 128 keys in one place 583; fewer registers in the softmax 532; a polynomial for ex2, below.
// 3 x 257 tokens over up to 6001 keys, 16 heads of 64 on 4: 50 us; the longest of 136 shares has 16 tiles of keys where even ones would have 13, and a sequence's fifth row tile has 4 rows.
// All waits are bounded; a time-out is noted in *status, the rows of that CTA come out as NaN, and the kernel frees its TMEM and ends.
#include <math_constants.h>

#include "../../include/blr_b200.h"
#include "paged.cuh"
#include "prompt.cuh"
#include "tmap.h"

namespace blr {

static constexpr int kKeys = 128, kStepKeys = 64, kRows = kPagedPromptRows;
// Threads, and registers of a thread at launch and from then on of the softmax warps (8) and the last four: setmaxnreg waits for ever for registers that the block was
// not launched with.
static constexpr int kPromptThreads = 384, kLaunchRegs = 168, kSoftmaxRegs = 216, kOtherRegs = 56;
static_assert(8 * kSoftmaxRegs + 4 * kOtherRegs <= kPromptThreads / 32 * kLaunchRegs, "more registers than the block has");

struct PagedPromptParams {
  CUtensorMap k, v;
  PagedAttnParams a;
  int k_head_at, k_page_at, v_head_at, v_page_at;  // which of the maps' outer dimensions has the heads, the pages
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}

// Slots in groups of 16: those of `groups` without a page (a bit each) are masked.
__device__ __forceinline__ void mask_groups(uint32_t (&x)[32], uint32_t groups) {
#pragma unroll
  for (int g = 0; g < 2; ++g)
    if (!(groups >> g & 1)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[16 * g + i] = 0xff800000u;
    }
}
// Moves a row's m to the largest of its scores, rounded up.  l and O are to be multiplied with the result, a power of two.
__device__ __forceinline__ float prompt_move(const uint32_t (&x)[2][32], float factor, float& m) {
  float top = -INFINITY;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(x[c][i]));
  const float to = fmaxf(m, ceilf(top * factor));
  if (to == -INFINITY) return 1.f;
  const float down = ex2(m - to);
  m = to;
  return down;
}
// p = 2^(s - mu) as 16-bit pairs over the scores in TMEM; returns their sum.  The arguments one number at a time: with the instruction for pairs of floats ex2 has to wait for
// its register pairs (1003 cycles for a warp's 64 numbers, and 605 without; 562 us for a prompt of 8192 tokens with 32 heads on 8, and 534 without); the sums, whose operands come out of
// ex2, by pairs (531 us).  A polynomial in place of ex2 for a sixteenth, an eighth and a quarter of the numbers: 538, 554 and 567 us, the warps are short of turns, not of ex2.
template <bool BF16>
__device__ __forceinline__ float prompt_weights(uint32_t s_at, const uint32_t (&x)[2][32], float factor, float mu) {
  uint64_t sum[2] = {};
  uint32_t yy[2][16];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t (&y)[16] = yy[c];
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float a = ex2(fmaf(__uint_as_float(x[c][i]), factor, -mu)), b = ex2(fmaf(__uint_as_float(x[c][i + 1]), factor, -mu));
      sum[(i & 2) / 2] = add2(sum[(i & 2) / 2], pair(a, b));
      y[i / 2] = q8_down2<BF16>(a, b);
    }
  }
  tmem_st16(s_at, yy[0]);
  tmem_st16(s_at + 16, yy[1]);
  float a, b;
  unpair(add2(sum[0], sum[1]), a, b);
  return a + b;
}

template <bool BF16>
__device__ __forceinline__ uint32_t not_numbers(uint32_t w) {  // a mask of the halves of a pair that are NaN or infinite
  constexpr uint32_t ex = BF16 ? 0x7f80u : 0x7c00u;
  return ((w & ex) == ex ? 0xffffu : 0u) | ((w >> 16 & ex) == ex ? 0xffff0000u : 0u);
}

// What a CTA works on.  (Asked for anew where it is needed: kept in registers across the loops it would push others out of them.)
struct Place {
  int split, bh, b, h, r0;
};
__device__ __forceinline__ Place place_of(const PagedAttnParams& p) {
  int cta;
  asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(cta));
  Place a;
  const int tiles = p.n_bh * p.q_tiles;
  a.split = cta / tiles;
  const int tile = cta - a.split * tiles;
  a.bh = tile % p.n_bh;
  a.r0 = (p.q_tiles - 1 - tile / p.n_bh) * kRows;  // the last rows have the most keys: their CTAs come first
  a.b = a.bh / p.c.kv_heads;
  a.h = a.bh - a.b * p.c.kv_heads;
  return a;
}

template <bool BF16, int HD>
__global__ void __launch_bounds__(kPromptThreads, 1) paged_prompt_kernel(const __grid_constant__ PagedPromptParams pp) {
  extern __shared__ __align__(1024) uint8_t prompt_raw[];
  const PagedAttnParams& p = pp.a;
  constexpr uint32_t kTile = 128 * HD * 2;
  const uint32_t base = (smem_u32(prompt_raw) + 1023u) & ~1023u;
  const uint32_t qs = base, ks = base + 2 * kTile, vs = base + 4 * kTile, bars = base + 6 * kTile;
  // sfull, pfull, done: [half][place]; zfull: the values of a tile that not all rows see are there (its own count: those who wait for it
  // begin with the first such tile), vclean: they have been looked through
  const uint32_t kfull = bars, vfull = bars + 16, kempty = bars + 32, vempty = bars + 48, sfull = bars + 64, pfull = bars + 96, done = bars + 128, vclean = bars + 192, zfull = bars + 208;
  __shared__ uint32_t tmem_slot, there[4], any_bad;
  __shared__ volatile int aborted;
  volatile int* const abort_flag = &aborted;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    *abort_flag = 0, any_bad = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(kfull + 8 * i, 1);
      mbar_init(vfull + 8 * i, 1);
      mbar_init(kempty + 8 * i, 1);
      mbar_init(vempty + 8 * i, 1);
      mbar_init(vclean + 8 * i, 2);
      mbar_init(zfull + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(sfull + 8 * i, 1);
      mbar_init(pfull + 8 * i, 4);
      mbar_init(done + 8 * i, 1);
    }
    mbar_init_fence();
  }
  __syncthreads();  // (the barriers are there)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int k0, k1, n0, n1, lim = 0, clean0;  // clean0: the first tile that not all rows see
  const int wg = warp >> 2;
  {
    const Place at = place_of(p);
    const long long start = p.start[at.b], count = p.n_new == nullptr ? p.T : min((long long)p.T, p.n_new[at.b]);
    // ---- a softmax thread's row of q
    const int row_i = (int)threadIdx.x & 127, r = at.r0 + (int)threadIdx.x;
    if (warp < 8) {
      const bool live = r < p.rows && r / p.G < count;
      const int tok = live ? r / p.G : 0;
      const uint4* const row = reinterpret_cast<const uint4*>(p.q + ((long long)at.b * p.T + tok) * p.ldq + (long long)(at.h * p.G + (live ? r - tok * p.G : 0)) * HD);
      if (live) lim = paged_seen(start, count, tok, p.c.slots);
      const uint32_t to = qs + wg * kTile + row_i * 128;
#pragma unroll 4
      for (int i = 0; i < HD / 8; ++i) {
        const uint4 x = live ? row[i] : make_uint4(0, 0, 0, 0);
        sts128(to + (i >> 3) * 16384 + (((i & 7) ^ (row_i & 7)) << 4), x.x, x.y, x.z, x.w);
      }
      fence_proxy_async_smem();
    }
    const int keys0 = paged_seen_by(p, start, count, at.r0, at.r0 + 128), keys1 = paged_seen_by(p, start, count, at.r0 + 128, at.r0 + 256);
    const int keys = max(keys0, keys1), share = p.ns > 1 ? paged_share(p, keys, p.rows - at.r0, kRows, kRows / 2, kKeys, lane) : max(keys, 1);
    k0 = (int)min((long long)keys, (long long)at.split * share), k1 = min(keys, k0 + min(share, keys - k0));
    if (p.ns > 1 && k0 >= k1) {  // no keys for this CTA: its rows say so
      const int r = at.r0 + (int)threadIdx.x;
      if ((int)threadIdx.x < kRows && r < p.rows) *reinterpret_cast<float2*>(p.part + (((long long)at.bh * p.rows + r) * p.ns + at.split) * (HD + 4) + HD) = make_float2(-INFINITY, 0.f);
      return;
    }
    n0 = max(0, min(keys0, k1) - k0 + kStepKeys - 1) / kStepKeys;
    n1 = max(0, min(keys1, k1) - k0 + kStepKeys - 1) / kStepKeys;
    clean0 = max(0, max(1, paged_seen(start, count, at.r0 / p.G, p.c.slots)) - k0) / kKeys;
  }
  if (warp == 8) tmem_alloc(smem_u32(&tmem_slot), 512);
  if (warp < 9) {  // (q and the room in TMEM; the copies begin meanwhile)
    tc_fence_before();
    asm volatile("bar.sync 2, 288;" ::: "memory");
    tc_fence_after();
  }
  const uint32_t tmem = tmem_slot;
  const int halves = max(n0, n1), steps = (halves + 1) / 2;  // (n0, n1, halves: of 64 keys; steps: tiles of 128)

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 9) {
      // lane i < 128 / page has the page of that part of a tile
      const Place at = place_of(p);
      const int parts = kKeys >> p.c.page_log2, part_bytes = 128 << p.c.page_log2;
      const int* const table = p.c.table + (long long)at.b * p.c.ld_table;
      auto page_of = [&](int j) {
        const int slot = k0 + j * kKeys + (lane << p.c.page_log2);
        const int page = lane < parts && slot < k1 ? table[slot >> p.c.page_log2] : -1;
        return (unsigned)page < (unsigned)p.c.pages ? page : p.c.pages;
      };
      auto copy = [&](uint32_t to, const CUtensorMap* map, int page, int head_at, int page_at, uint32_t bar) {
        if (elect_one()) mbar_arrive_expect_tx(bar, kTile);
        __syncwarp();
#pragma unroll 1
        for (int i = 0; i < parts; ++i) {
          const int one = __shfl_sync(0xffffffffu, page, i);
          if (elect_one()) {
            const int c1 = head_at == 1 ? at.h : page_at == 1 ? one : 0, c2 = head_at == 2 ? at.h : page_at == 2 ? one : 0, c3 = head_at == 3 ? at.h : page_at == 3 ? one : 0;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) tma_load_4d(to + c * 16384 + i * part_bytes, map, 64 * c, c1, c2, c3, bar);
          }
          __syncwarp();
        }
      };
      int next = page_of(0);
#pragma unroll 1
      for (int j = 0; j < steps; ++j) {
        const uint32_t s = j & 1, parity = ((j >> 1) & 1) ^ 1;
        const int page = next;
        if (j + 1 < steps) next = page_of(j + 1);
        if (j >= 2 && !__all_sync(0xffffffffu, mbar_wait(kempty + 8 * s, parity, abort_flag))) break;
        // (a tile's word is free when the S of the tile after it is done, and this warp is two tiles ahead of that at most)
        const unsigned parts_there = __ballot_sync(0xffffffffu, page < p.c.pages);
        if (lane == 0) {
          uint32_t groups = 0;
          for (int g = 0; g < 8; ++g) groups |= (parts_there >> (g * 16 >> p.c.page_log2) & 1u) << g;
          there[j & 3] = groups;
        }
        copy(ks + s * kTile, &pp.k, page, pp.k_head_at, pp.k_page_at, kfull + 8 * s);
        if (j >= 2 && !__all_sync(0xffffffffu, mbar_wait(vempty + 8 * s, parity, abort_flag))) break;
        copy(vs + s * kTile, &pp.v, page, pp.v_head_at, pp.v_page_at, (j >= clean0 ? zfull : vfull) + 8 * s);
      }
    } else if (warp >= 10) {
      uint32_t bad = 0;
#pragma unroll 1
      for (int j = clean0; j < steps; ++j) {
        const uint32_t s = j & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(zfull + 8 * s, ((j - clean0) >> 1) & 1, abort_flag))) break;
        const int live = k1 - (k0 + j * kKeys);  // rows of the tile that hold a key
#pragma unroll 1
        for (int i = (warp - 10) * 32 + lane; i < 128 * HD / 8; i += 64) {
          const uint32_t place = vs + s * kTile + 16 * i;
          const int row = (i >> 3) & 127;
          uint32_t w[4];
          lds128(place, w[0], w[1], w[2], w[3]);
          uint32_t any = 0;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t no = row < live ? not_numbers<BF16>(w[x]) : 0xffffffffu;
            any |= no;
            if (row < live) bad |= no;
            w[x] &= ~no;
          }
          if (any) sts128(place, w[0], w[1], w[2], w[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(vclean + 8 * s);
      }
      if (__any_sync(0xffffffffu, bad != 0) && lane == 0) {
        atomicOr(&any_bad, 1u);
        __threadfence_block();
      }
    } else if (elect_one()) {
      const uint32_t id_s = umma_idesc(BF16, false, false, 128, kStepKeys), id_o = umma_idesc(BF16, false, true, 128, HD);
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
          const bool clean = j >= clean0;
          if (!mbar_poll((clean ? vclean : vfull) + 8 * (j & 1), (clean ? (j - clean0) >> 1 : j >> 1) & 1, abort_flag)) { ok = false; break; }
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
    asm volatile("bar.arrive 1, 384;" ::: "memory");  // (what warps 10 and 11 found is known)
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int n = wg ? n1 : n0;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, o_at = tmem + lanes + 256 + 128 * wg;
    const float factor = p.scale_log2;
    float m = -INFINITY, l = 0.f;
    const int lim_all = __reduce_min_sync(0xffffffffu, lim);
    uint32_t groups = 0xffu;  // of the tile's keys by 16: which have a page
    bool ok = true, fresh = true;  // fresh: a row of the warp has yet to see its first keys
#pragma unroll 1
    for (int u = 0; u < n; ++u) {
      const int j = u >> 1, key0 = k0 + u * kStepKeys;
      const uint32_t s_at = tmem + lanes + 128 * wg + 64 * (u & 1);
      const bool part = key0 + kStepKeys > lim_all;  // some of these keys are masked for a row of the warp
      if (!__all_sync(0xffffffffu, mbar_wait(sfull + 16 * wg + 8 * (u & 1), j & 1, abort_flag))) { ok = false; break; }
      if ((u & 1) == 0) groups = *(volatile uint32_t*)&there[j & 3];  // (written ahead of the copy of the keys that these scores are of)
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
      if (groups != 0xffu) {
        mask_groups(x[0], groups >> 4 * (u & 1));
        mask_groups(x[1], groups >> (4 * (u & 1) + 2));
      }
      // against the m so far, which is seldom left behind: a sum above 2^11 tells of it, and all is done once more.  The rows that ask for it move theirs, the others come out as
      // they were.  The first keys of a row are a pass of their own, ahead of that: a row without a number among its scores takes all of its keys for the first, and the rows beside it are not
      // to wait for it.
      float total = 0.f;
      bool ask = fresh && m == -INFINITY && lim > key0;  // (a row's first keys)
      if (fresh) fresh = __any_sync(0xffffffffu, m == -INFINITY && lim > 0);
#pragma unroll 1
      for (int pass = fresh && __any_sync(0xffffffffu, ask) ? 1 : 0;; pass = 2) {  // 0: nothing moves, 1: a row's first keys, 2: what is behind
        if (pass != 0) {
          float down = 1.f;
          if (ask) down = prompt_move(x, factor, m);
          __syncwarp();  // (what follows in TMEM is the whole warp's)
          l *= down;
          if (u > 0 && __any_sync(0xffffffffu, down != 1.f)) {
            if (!__all_sync(0xffffffffu, mbar_wait(done + 16 * wg + 8 * ((u - 1) & 1), ((u - 1) >> 1) & 1, abort_flag))) { ok = false; break; }
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < HD / 8; ++k) {
              uint32_t o[8];
              tmem_ld8(o_at + 8 * k, o);
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * down);
              tmem_st8(o_at + 8 * k, o);
            }
          }
        }
        total = prompt_weights<BF16>(s_at, x, factor, m == -INFINITY ? 0.f : m);
        ask = total > 2048.f;
        if (pass == 2 || !__any_sync(0xffffffffu, ask)) break;
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
    asm volatile("bar.sync 1, 384;" ::: "memory");
    const bool spoilt = ok && *(volatile uint32_t*)&any_bad != 0;
    const Place at = place_of(p);
    const int r = at.r0 + (int)threadIdx.x;
    const bool live = r < p.rows;
    const float fin = !ok ? CUDART_NAN_F : p.ns > 1 ? 1.f : 1.f / l;
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
      if (spoilt && lim > 0) {
        // (seldom) values that are no numbers, of the keys from tile clean0 on that this row sees
        const uint16_t* const q = p.q + ((long long)at.b * p.T + tok) * p.ldq + (long long)(at.h * p.G + r - tok * p.G) * HD;
#pragma unroll 1
        for (int key = k0 + clean0 * kKeys; key < min(lim, k1); ++key) {
          const int page = p.c.table[(long long)at.b * p.c.ld_table + (key >> p.c.page_log2)], in = key & ((1 << p.c.page_log2) - 1);
          if ((unsigned)page >= (unsigned)p.c.pages) continue;
          const uint32_t* const v = reinterpret_cast<const uint32_t*>(p.c.v + page * p.c.v_page + at.h * p.c.v_head + in * p.c.v_slot) + 16 * c;
          uint32_t bad = 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) bad |= not_numbers<BF16>(v[i]);
          if (bad == 0) continue;
          const uint32_t *const k = reinterpret_cast<const uint32_t*>(p.c.k + page * p.c.k_page + at.h * p.c.k_head + in * p.c.k_slot), *const qw = reinterpret_cast<const uint32_t*>(q);
          float s = 0.f;
#pragma unroll 4
          for (int i = 0; i < HD / 2; ++i) {
            const float2 a = q8_up2<BF16>(qw[i]), b = q8_up2<BF16>(k[i]);
            s = fmaf(a.x, b.x, s), s = fmaf(a.y, b.y, s);
          }
          const float w = ex2(fmaf(s, factor, m == -INFINITY ? 0.f : -m));
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t no = not_numbers<BF16>(v[i]);
            const float2 f = q8_up2<BF16>(v[i]);
            if (no & 0xffffu) x[2 * i] = __float_as_uint(fmaf(w, f.x, __uint_as_float(x[2 * i])));
            if (no >> 16) x[2 * i + 1] = __float_as_uint(fmaf(w, f.y, __uint_as_float(x[2 * i + 1])));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 32; ++i)  // (a row that sees nothing: zeros, whatever its products were)
        x[i] = ok && l == 0.f ? 0u : __float_as_uint(__uint_as_float(x[i]) * fin);
      if (p.ns > 1) {
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<float4*>(to32 + 32 * c + i) = make_float4(__uint_as_float(x[i]), __uint_as_float(x[i + 1]), __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
      } else {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          uint32_t o[4];
#pragma unroll
          for (int z = 0; z < 4; ++z) o[z] = q8_down2<BF16>(__uint_as_float(x[i + 2 * z]), __uint_as_float(x[i + 2 * z + 1]));
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
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // (copies and products in flight end before their operands' memory is given back)
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// A pool as the copy engine sees it: 64 of a head's values, and the slots, heads and pages by rising strides, each a multiple of the one before it.  Where a pool's layout is
// another (or there is no page) the rows go through the kernel for few.
struct PoolDims {
  uint64_t dims[4], strides[3];
  uint32_t box[4];
  int at[3];  // of slots, heads, pages
};
static bool pool_dims(const int64_t strides[3], const blr_paged_cache* c, PoolDims* o) {
  const int64_t size[3] = {c->page, c->kv_heads, c->pages}, stride[3] = {strides[2], strides[1], strides[0]};
  int order[3] = {0, 1, 2};
  auto later = [&](int a, int b) { return size[a] == 1 || (size[b] != 1 && stride[a] > stride[b]); };  // (a dimension of one has no stride of its own)
  for (int i = 0; i < 2; ++i)
    for (int k = 0; k < 2 - i; ++k)
      if (later(order[k], order[k + 1]) && !(size[order[k + 1]] == 1 && size[order[k]] == 1)) {
        const int t = order[k];
        order[k] = order[k + 1], order[k + 1] = t;
      }
  o->dims[0] = (uint64_t)c->head_dim, o->box[0] = 64;
  uint64_t before = 0;
  for (int i = 0; i < 3; ++i) {
    const int w = order[i];
    const uint64_t bytes = size[w] == 1 && before != 0 ? before : 2 * (uint64_t)stride[w];
    if ((before != 0 && bytes % before != 0) || bytes >= (1ull << 40)) return false;
    o->dims[i + 1] = (uint64_t)size[w], o->strides[i] = before = bytes, o->box[i + 1] = w == 0 ? (uint32_t)c->page : 1u;
    o->at[w] = i + 1;
  }
  return true;
}

bool paged_prompt_fits(const blr_paged_cache* c) {
  PoolDims d;
  return c->pages > 0 && pool_dims(c->k_strides, c, &d) && pool_dims(c->v_strides, c, &d);
}

template <bool BF16, int HD>
static int launch_prompt(const PagedPromptParams& p, cudaStream_t stream) {
  static bool configured[64] = {};
  DeviceInfo di;
  int rc;
  if ((rc = device_info(&di))) return rc;
  const int smem = 6 * 128 * HD * 2 + 1024 + 256 < 120 * 1024 ? 120 * 1024 : 6 * 128 * HD * 2 + 1024 + 256;  // one CTA per SM: a second one would only wait for TMEM
  if (!configured[di.dev]) {
    BLR_CUDA_OK(cudaFuncSetAttribute(paged_prompt_kernel<BF16, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaFuncAttributes fa;
    BLR_CUDA_OK(cudaFuncGetAttributes(&fa, paged_prompt_kernel<BF16, HD>));
    BLR_REQUIRE(fa.numRegs == kLaunchRegs, BLR_ERR_UNSUPPORTED, "the prompt kernel was built with %d registers, its split is made for %d", fa.numRegs, kLaunchRegs);
    configured[di.dev] = true;
  }
  return q8_launch(paged_prompt_kernel<BF16, HD>, dim3((unsigned)p.a.n_bh * p.a.q_tiles * p.a.ns), kPromptThreads, smem, stream, p);
}

int paged_launch_prompt(const PagedAttnParams& a, const blr_paged_cache* c, bool bf16, cudaStream_t stream) {
  PagedPromptParams p = {};
  p.a = a;
  const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  PoolDims d;
  int rc;
  pool_dims(c->k_strides, c, &d);
  p.k_head_at = d.at[1], p.k_page_at = d.at[2];
  if ((rc = encode_tmap_4d(&p.k, dt, c->k, d.dims, d.strides, d.box, Swz::B128))) return rc;
  pool_dims(c->v_strides, c, &d);
  p.v_head_at = d.at[1], p.v_page_at = d.at[2];
  if ((rc = encode_tmap_4d(&p.v, dt, c->v, d.dims, d.strides, d.box, Swz::B128))) return rc;
  if (c->head_dim == 128) return bf16 ? launch_prompt<true, 128>(p, stream) : launch_prompt<false, 128>(p, stream);
  return bf16 ? launch_prompt<true, 64>(p, stream) : launch_prompt<false, 64>(p, stream);
}

}  // namespace blr
