// Log probabilities of given tokens, entropy and likeliest tokens of rows of logits.
//   M = max x,  S = sum e^(x - M),  log p(i) = (x_i - M) - log S,  H = log S - (sum e^(x - M) (x - M)) / S
// in fp32: e^(x - M) = 2^t for t = (x - M) log2 e, and H = log S - log 2 (sum 2^t t) / S.  The difference comes first: it is all that counts, and is exact for
// values next to M however far from 0 they lie (a row that is masked throughout with -1e10, say), where a product of M would be off by any number.  It costs nothing,
// since pairs of values share an instruction (add, mul, add, fma for two, beside two ex2 and two clamps).
// Order of the likeliest: falling value (NaN above everything, -0 equal to 0), ties by rising id.
//
// A cluster of 1 to 8 CTAs takes a row: each reads its part once into shared memory, keeping the maximum of what every thread reads, and works from there.
// The smallest of the maxima of as many groups of threads as tokens are asked for is a number that at least so many values reach: only values that reach it
// (some tens) are kept and ordered.  A list that overflows is made anew of those above that number and the first of those that equal it (2047 rows of 32000 bf16 with 3 tokens
// that are not ruled out, 8 alternatives: 89 us, by one search for each token 497); one that overflows again by searches.
// Bound by HBM (each logit once), closely followed by ex2 (16 a cycle and SM).
#include <cooperative_groups.h>
#include <math_constants.h>

#include "../../include/blr_b200.h"
#include "logits.cuh"
#include "tmap.h"

namespace cg = cooperative_groups;

namespace blr {

static constexpr int kLpMaxTop = 64, kLpGroups = 128, kLpMaxPart = 200 * 1024;
typedef unsigned long long Ranked;  // order_of(value) << 32 | ~id: larger is likelier

__device__ __forceinline__ Ranked ranked(float x, int id) { return (Ranked)order_of(x) << 32 | (0xffffffffu - (uint32_t)id); }

// Of the largest values that groups of threads have seen, the `top`-th (by one warp): at least so many of a row's values reach it, and seldom many more.
// 0: there are fewer.
__device__ __forceinline__ uint32_t reached_by(const uint32_t* group, int groups, int top, int lane) {
  uint32_t found = 0;
  for (int i = lane; i < groups; i += 32) {
    const uint32_t v = group[i];
    int ahead = 0;
    for (int k = 0; k < groups; ++k) ahead += group[k] > v || (group[k] == v && k < i);
    if (ahead == top - 1) found = v;
  }
  return __reduce_max_sync(0xffffffffu, found);
}
// The groups of a CTA's warps, a warp each or equal parts of one: as few as make a group that has seen something for each token asked for, twice as many in a CTA of few warps,
// which has less room for what reaches the threshold.  The first thread of each leaves what its group has seen.
template <int WARPS>
__device__ __forceinline__ int leave_group(uint32_t seen, uint32_t* group, int vectors, int top, int warp, int lane) {
  int parts = 1;
  while (parts < 32 && parts * WARPS < kLpGroups && (min(vectors, 32 * WARPS) * parts + 31) / 32 < (WARPS == 16 ? top : 2 * top)) parts *= 2;
  uint32_t g = seen;
  for (int d = 1; d < 32 / parts; d <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, d));
  if (lane % (32 / parts) == 0) group[warp * parts + lane / (32 / parts)] = g;
  return WARPS * parts;
}

struct LpParams {
  const void* logits;
  long long ld;
  const long long* ids;
  float *logprob, *entropy, *top_lp;
  long long* top_ids;
  int vocab, top, part;  // part: vectors of a CTA
};

// What a CTA of THREADS threads keeps beside its part of the row; kKept: room for values that reach the threshold.
template <int THREADS>
struct LpShared {
  static constexpr int kWarps = THREADS / 32, kKept = THREADS == 512 ? 1024 : 4 * THREADS;
  Ranked kept[kKept], best[kLpMaxTop], red[kWarps];
  float edge[16], sums[2][kWarps], S, D;  // edge: values of the row ahead of its first whole vector and behind its last
  uint32_t most, least, count;
  uint32_t group[kLpGroups];
};

template <int KIND, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 3 : 1536 / THREADS < 32 ? 1536 / THREADS : 32) token_logprobs_kernel(const __grid_constant__ LpParams p) {
  extern __shared__ __align__(16) uint4 part[];
  typedef LpShared<THREADS> Shared;
  constexpr int kLpThreads = THREADS, kLpWarps = Shared::kWarps, kLpKept = Shared::kKept;
  __shared__ Shared sh;
  constexpr int kPer = Vec<KIND>::kPer, kSize = KIND == 2 ? 4 : 2;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = cluster.block_rank(), n_cta = cluster.num_blocks();
  const long long r = blockIdx.x / n_cta;
  const char* const row = static_cast<const char*>(p.logits) + r * p.ld * kSize;
  // whole vectors of the row, this CTA's of them, and the values around them (the first CTA's)
  const int head = min(p.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / kSize), vecs = (p.vocab - head) / kPer, tail = p.vocab - head - vecs * kPer;
  const int v0 = min(vecs, rank * p.part), mine = min(vecs, v0 + p.part) - v0, id0 = head + v0 * kPer, edges = rank == 0 ? head + tail : 0;
  auto edge_id = [&](int i) { return i < head ? i : p.vocab - tail + (i - head); };
  if (tid == 0) sh.count = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const bool writes = rank == 0 && tid == kLpThreads - 1;  // (its loads are on their way long before they are used)
  const long long id = writes ? p.ids[r] : -1;

  // ---- the row into shared memory, and the largest value that each thread has seen (0: none)
  uint32_t seen = 0;
  {
    const uint4* const from = reinterpret_cast<const uint4*>(row + (size_t)head * kSize) + v0;
    constexpr int kAhead = 4;
    uint32_t top = Vec<KIND>::kLowest;
    int i = tid;
    for (; i + (kAhead - 1) * kLpThreads < mine; i += kAhead * kLpThreads) {
      uint4 w[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) w[u] = from[i + u * kLpThreads];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        part[i + u * kLpThreads] = w[u];
        top = Vec<KIND>::larger(top, Vec<KIND>::largest(w[u]));
      }
    }
    uint4 w[kAhead - 1];
#pragma unroll
    for (int u = 0; u < kAhead - 1; ++u)
      if (i + u * kLpThreads < mine) w[u] = from[i + u * kLpThreads];
#pragma unroll
    for (int u = 0; u < kAhead - 1; ++u)
      if (i + u * kLpThreads < mine) {
        part[i + u * kLpThreads] = w[u];
        top = Vec<KIND>::larger(top, Vec<KIND>::largest(w[u]));
      }
    if (tid < mine) seen = order_of(Vec<KIND>::most(top));
    if (tid < edges) {
      const float x = logit<KIND>(row, edge_id(tid));
      sh.edge[tid] = x;
      seen = max(seen, order_of(x));
    }
  }
  const float given = id >= 0 && id < p.vocab ? logit<KIND>(row, id) : 0.f;
  const int groups = leave_group<kLpWarps>(seen, sh.group, mine, p.top, warp, lane);
  __syncthreads();
  if (warp == 0) {
    uint32_t most = 0;
    for (int i = lane; i < groups; i += 32) most = max(most, sh.group[i]);
    most = __reduce_max_sync(0xffffffffu, most);
    const uint32_t least = p.top > 0 ? reached_by(sh.group, groups, p.top, lane) : 0u;
    if (lane == 0) sh.most = most, sh.least = least;
  }
  if (n_cta > 1) cluster.sync();
  else __syncthreads();
  uint32_t most = 0, least = 0;
  for (int o = 0; o < n_cta; ++o) {
    const Shared* other = cluster.map_shared_rank(&sh, o);
    most = max(most, other->most), least = max(least, other->least);
  }
  const float M = value_of(most), reach = value_of(least);
  const bool finite = M <= 3.402823466e38f && M >= -3.402823466e38f, empty = M == -CUDART_INF_F;
  const bool all = least == 0;  // (too few groups have seen anything: keep everything)

  // ---- the sums, and the values that reach the threshold
  float S = 0.f, D = 0.f;
  auto keep = [&](float x, int id) {
    const uint32_t at = atomicAdd(&sh.count, 1u);
    if (at < kLpKept) sh.kept[at] = ranked(x, id);
  };
  if (finite) {
    const uint64_t low = pair(-M, -M), log2e = pair(1.4426950408889634f, 1.4426950408889634f);
    uint64_t s2 = 0, d2 = 0;
    auto add = [&](float x, float y) {
      float t[2];
      unpair(mul2(add2(pair(x, y), low), log2e), t[0], t[1]);
      t[0] = fmaxf(t[0], -1e30f), t[1] = fmaxf(t[1], -1e30f);  // (-inf: a weight of 0, and of a number)
      const uint64_t e = pair(ex2(t[0]), ex2(t[1]));
      s2 = add2(s2, e);
      d2 = fma2(e, pair(t[0], t[1]), d2);
    };
    int i = tid;
    auto vec = [&](const uint4& w) {
      float f[kPer];
      Vec<KIND>::floats(w, f);
#pragma unroll
      for (int k = 0; k < kPer; k += 2) add(f[k], f[k + 1]);
    };
    for (; i + kLpThreads < mine; i += 2 * kLpThreads) {
      const uint4 w = part[i], v = part[i + kLpThreads];
      vec(w);
      vec(v);
    }
    if (i < mine) vec(part[i]);
    if (tid < edges) add(sh.edge[tid], -CUDART_INF_F);
    float odd;
    unpair(s2, S, odd), S += odd;
    unpair(d2, D, odd), D += odd;
    if (p.top > 0 && (all || seen >= least)) {  // (few threads)
      for (int i = tid; i < mine; i += kLpThreads) {
        const uint4 w = part[i];
        if (!all && !(Vec<KIND>::most(Vec<KIND>::largest(w)) >= reach)) continue;
        if (*(volatile uint32_t*)&sh.count > kLpKept) break;  // (too many: made anew below)
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const float x = Vec<KIND>::value(w, k);
          if (all || x >= reach) keep(x, id0 + i * kPer + k);
        }
      }
      if (tid < edges && (all || sh.edge[tid] >= reach)) keep(sh.edge[tid], edge_id(tid));
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) S += __shfl_xor_sync(0xffffffffu, S, d), D += __shfl_xor_sync(0xffffffffu, D, d);
  if (lane == 0) sh.sums[0][warp] = S, sh.sums[1][warp] = D;
  __syncthreads();
  if (warp == 0) {
    S = lane < kLpWarps ? sh.sums[0][lane] : 0.f, D = lane < kLpWarps ? sh.sums[1][lane] : 0.f;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) S += __shfl_xor_sync(0xffffffffu, S, d), D += __shfl_xor_sync(0xffffffffu, D, d);
    if (lane == 0) sh.S = S, sh.D = D;
  }

  // ---- this CTA's likeliest, in order (0: no more)
  int kept = (int)sh.count;
  for (int i = tid; i < kLpMaxTop; i += kLpThreads) sh.best[i] = 0;
  __syncthreads();
  if (finite && !all && kept > kLpKept) {
    // Many values are equal to the threshold (tokens that are ruled out, where fewer are left than asked for): those above it, and by rising id those on it until there are enough.
    if (tid == 0) sh.count = 0;
    __syncthreads();
    for (int i = tid; i < mine; i += kLpThreads) {
      const uint4 w = part[i];
      if (!(Vec<KIND>::most(Vec<KIND>::largest(w)) > reach)) continue;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const float x = Vec<KIND>::value(w, k);
        if (x > reach) keep(x, id0 + i * kPer + k);
      }
    }
    if (tid < edges && sh.edge[tid] > reach) keep(sh.edge[tid], edge_id(tid));
    if (warp == 0) {
      int found = 0;
      auto look = [&](bool there, float x, int id) {
        const bool on = there && x == reach;
        if (on) keep(x, id);
        found += __popc(__ballot_sync(0xffffffffu, on));
      };
      const int ahead = min(edges, head);
      look(lane < ahead, lane < ahead ? sh.edge[lane] : 0.f, lane);
      for (int i0 = 0; i0 < mine && found < p.top; i0 += 32) {
        const int i = i0 + lane;
        const uint4 w = i < mine ? part[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < kPer; ++k) look(i < mine, Vec<KIND>::value(w, k), id0 + i * kPer + k);
      }
      if (found < p.top) look(ahead + lane < edges, ahead + lane < edges ? sh.edge[ahead + lane] : 0.f, edge_id(ahead + lane));
    }
    __syncthreads();
    kept = (int)sh.count;
  }
  if (finite && kept <= kLpKept) {
    for (int i = tid; i < kept; i += kLpThreads) {
      const Ranked v = sh.kept[i];
      int before = 0;
      for (int k = 0; k < kept; ++k) before += sh.kept[k] > v;
      if (before < p.top) sh.best[before] = v;
    }
  } else {
    Ranked last = ~0ull;
    for (int k = 0; k < p.top && last != 0; ++k) {  // (too many all the same, or a row with values that are no numbers: one search each)
      Ranked v = 0;
      auto look = [&](float x, int id) {
        const Ranked c = ranked(x, id);
        if (c < last) v = max(v, c);
      };
      for (int i = tid; i < mine; i += kLpThreads) {
        const uint4 w = part[i];
#pragma unroll
        for (int z = 0; z < kPer; ++z) look(Vec<KIND>::value(w, z), id0 + i * kPer + z);
      }
      if (tid < edges) look(sh.edge[tid], edge_id(tid));
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
      if (lane == 0) sh.red[warp] = v;
      __syncthreads();
      v = sh.red[0];
      for (int w = 1; w < kLpWarps; ++w) v = max(v, sh.red[w]);
      if (tid == 0) sh.best[k] = v;
      last = v;
      __syncthreads();
    }
  }
  if (n_cta > 1) cluster.sync();
  else __syncthreads();

  // ---- the first CTA puts the row together
  if (rank == 0) {
    S = D = 0.f;
    for (int o = 0; o < n_cta; ++o) {
      const Shared* other = cluster.map_shared_rank(&sh, o);
      S += other->S, D += other->D;
    }
    const float log_s = logf(S);
    // (a row of -inf alone: every log probability -inf, entropy 0; a NaN or +inf: NaN)
    auto lp = [&](float x) { return finite ? (x - M) - log_s : empty ? -CUDART_INF_F : CUDART_NAN_F; };
    if (writes) {
      p.logprob[r] = id < 0 ? 0.f : id >= p.vocab ? CUDART_NAN_F : lp(given);
      p.entropy[r] = finite ? log_s - D / S * 0.69314718055994531f : empty ? 0.f : CUDART_NAN_F;
    }
    for (int i = tid; i < n_cta * p.top; i += kLpThreads) {
      const int from = i / p.top, k = i - from * p.top;
      const Ranked v = cluster.map_shared_rank(&sh, from)->best[k];
      if (v == 0) continue;
      int before = k;  // (lists are in order: a binary search in each of the others)
      for (int o = 0; o < n_cta; ++o) {
        if (o == from) continue;
        const Ranked* list = cluster.map_shared_rank(&sh, o)->best;
        int a = 0, z = p.top;
        while (a < z) {
          const int m = (a + z) >> 1;
          if (list[m] > v) a = m + 1;
          else z = m;
        }
        before += a;
      }
      if (before < p.top) p.top_lp[r * p.top + before] = lp(value_of((uint32_t)(v >> 32))), p.top_ids[r * p.top + before] = 0xffffffffu - (uint32_t)v;
    }
  }
  if (n_cta > 1) cluster.sync();  // (a CTA's memory is there until the first one has read it)
}

template <int KIND, int THREADS>
static int launch_logprobs(const LpParams& p, int64_t rows, int ctas, int smem, cudaStream_t stream) {
  static bool configured[64] = {};
  DeviceInfo di;
  int rc;
  if ((rc = device_info(&di))) return rc;
  if (!configured[di.dev]) {
    BLR_CUDA_OK(cudaFuncSetAttribute(token_logprobs_kernel<KIND, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLpMaxPart));
    configured[di.dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)ctas;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  BLR_CUDA_OK(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<KIND, THREADS>, p));
  return BLR_OK;
}

// Rows of at most so many vectors of 16 bytes that one CTA takes whole: a warp's, four warps'.  (4000 rows, us with 512 | 128 | 32 threads: 300 values of fp16 and 20 alternatives
// 150 | 40 | 22, 300 of fp32 144 | 37 | 21, 500 of fp32 235 | 22 | 24; 2000 of fp16 and 5 alternatives 45 | 20 | 32, 8000 of fp32 70 | 62 | 97.)  A warp has 32 groups at most for its
// threshold: for more alternatives four take the row (300 of fp16, 64 alternatives 151 | 99 | 180).
static constexpr int kWarpVecs = 96, kWarpTop = 32, kFourWarpVecs = 2048;

}  // namespace blr

using namespace blr;

extern "C" {

int blr_token_logprobs(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int kind, const int64_t* ids, int top, float* logprob,
                       float* entropy, float* top_logprob, int64_t* top_ids, void* stream) {
  BLR_REQUIRE(kind >= 0 && kind <= 2, BLR_ERR_ARG, "unknown kind of logits %d", kind);
  const int64_t size = kind == 2 ? 4 : 2;
  BLR_REQUIRE(rows >= 0 && rows < (1ll << 28) && vocab > 0 && (rows <= 1 || ld >= vocab), BLR_ERR_ARG, "token_logprobs: %lld rows of %lld", (long long)rows,
              (long long)vocab);
  BLR_REQUIRE(vocab * size <= 8ll * kLpMaxPart, BLR_ERR_UNSUPPORTED, "token_logprobs keeps a row in the shared memory of 8 SMs: at most %lld bytes, not %lld",
              8ll * kLpMaxPart, (long long)(vocab * size));
  BLR_REQUIRE(top >= 0 && top <= kLpMaxTop && top <= vocab, BLR_ERR_ARG, "token_logprobs gives 0 to %d tokens (and no more than there are), not %d", kLpMaxTop, top);
  if (rows == 0) return BLR_OK;
  BLR_REQUIRE(logits && ids && logprob && entropy && (top == 0 || (top_logprob && top_ids)), BLR_ERR_ARG, "null pointer");
  BLR_REQUIRE(reinterpret_cast<uintptr_t>(logits) % size == 0, BLR_ERR_ARG, "token_logprobs: logits must be aligned to their size");
  // a row's part of at most 64 KB, so that three CTAs share an SM; few rows: over more CTAs, as long as each has 4 KB
  int ctas = 1;
  while (ctas < 8 && vocab * size > ctas * 65536ll) ctas *= 2;
  while (ctas < 8 && rows * ctas < 2ll * sm_count() && vocab * size >= ctas * 8192ll) ctas *= 2;
  LpParams p = {};
  p.logits = logits, p.ld = ld, p.ids = reinterpret_cast<const long long*>(ids);
  p.logprob = logprob, p.entropy = entropy, p.top_lp = top_logprob, p.top_ids = reinterpret_cast<long long*>(top_ids);
  const int64_t per = 16 / size, vecs = vocab / per;  // (as many vectors as a row can have, however it is aligned)
  p.vocab = (int)vocab, p.top = top, p.part = (int)((vecs + ctas - 1) / ctas);
  if (p.part < 1) p.part = 1;
  const int smem = p.part * 16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define BLR_LP(THREADS) \
  (kind == 0 ? launch_logprobs<0, THREADS>(p, rows, ctas, smem, st) : kind == 1 ? launch_logprobs<1, THREADS>(p, rows, ctas, smem, st) : launch_logprobs<2, THREADS>(p, rows, ctas, smem, st))
  if (ctas == 1 && p.part <= kWarpVecs && top <= kWarpTop) return BLR_LP(32);
  if (ctas == 1 && p.part <= kFourWarpVecs) return BLR_LP(128);
  return BLR_LP(512);
#undef BLR_LP
}

}  // extern "C"
