// The next token of rows of logits from a given uniform number u in [0, 1), with temperature T, top-k, top-p and min-p.
//   M = max x,  w_i = e^((x_i - M) / T)  (T = 0: 1 for the first of the largest, 0 else);  order: falling x, equal ones by rising id
//   kept: the first k; of those the fewest first ones whose weights reach p times their sum; of those the ones with w_i >= min_p
//   id = the least kept i with  sum of kept w_j, j <= i  >  u times the sum of all kept,   logprob = log(w_id / that sum)
// Each filter keeps the beginning of the order: what lies above a threshold, and the first few that equal it.  The last one goes by ids, so that nothing is sorted.
// A sum may end next to a border (p times the whole, u times the kept), and the token depends on which side: weights and sums are in 64 bits, in an order that depends on the
// row's length and place alone.
//
// A cluster of 1 to 8 CTAs takes a row: each reads its part once into shared memory and works from there.
#include <cooperative_groups.h>
#include <math_constants.h>

#include "../../include/blr_b200.h"
#include "logits.cuh"
#include "tmap.h"

namespace cg = cooperative_groups;

namespace blr {

static constexpr int kSampleMaxPart = 192 * 1024;  // bytes of a row that a CTA takes

struct SampleParams {
  const void* logits;
  long long ld;
  const float* uniform;
  blr_sampling s;
  long long* ids;
  float* logprob;
  int vocab, part;  // part: vectors of 16 bytes of a CTA, a multiple of 32
};

// What the CTAs of a row tell each other.
struct SampleSum {
  double mass;
  int count;
};

template <int KIND, int THREADS>
struct SampleShared {
  static constexpr int kWarps = THREADS / 32;
  SampleSum warp[kWarps], sum[2];
  uint32_t most[kWarps], top;
};

template <int KIND>
__device__ __forceinline__ uint32_t raw_logit(const char* row, int id) {  // its bits
  if constexpr (KIND == 2) return reinterpret_cast<const uint32_t*>(row)[id];
  else return reinterpret_cast<const uint16_t*>(row)[id];
}

template <int KIND, int THREADS>
__global__ void __launch_bounds__(THREADS) sample_kernel(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) uint4 part[];
  typedef SampleShared<KIND, THREADS> Shared;
  __shared__ Shared sh;
  constexpr int kPer = Vec<KIND>::kPer, kSize = KIND == 2 ? 4 : 2, kWarps = Shared::kWarps;
  // orders of 16-bit values differ in their upper bits alone
  constexpr int kDrop = KIND == 0 ? 13 : KIND == 1 ? 16 : 0;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = cluster.block_rank(), n_cta = cluster.num_blocks();
  const long long r = blockIdx.x / n_cta;
  const char* const row = static_cast<const char*>(p.logits) + r * p.ld * kSize;
  // vector i of the row has the values from id i kPer - shift on; -inf where there is none
  const int shift = (int)(reinterpret_cast<uintptr_t>(row) & 15) / kSize, vecs = (p.vocab + shift + kPer - 1) / kPer;
  const int v0 = min(vecs, rank * p.part), mine = min(vecs, v0 + p.part) - v0, chunks = (mine + 31) / 32;
  double* const chunk_mass = reinterpret_cast<double*>(part + p.part);
  int* const chunk_ties = reinterpret_cast<int*>(chunk_mass + p.part / 32);
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- the row into shared memory, and its largest value
  uint32_t top = Vec<KIND>::kLowest;
  for (int i = tid; i < mine; i += THREADS) {
    const int id = (v0 + i) * kPer - shift;
    uint4 w;
    if (id >= 0 && id + kPer <= p.vocab) {
      w = *reinterpret_cast<const uint4*>(row + (long long)id * kSize);
    } else {
      uint32_t x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = Vec<KIND>::kLowest;
#pragma unroll
        for (int z = 0; z < kPer / 4; ++z) {
          const int at = id + k * (kPer / 4) + z;
          if (at < 0 || at >= p.vocab) continue;
          const uint32_t v = raw_logit<KIND>(row, at);
          if constexpr (KIND == 2) x[k] = v;
          else x[k] = z ? (x[k] & 0xffffu) | v << 16 : (x[k] & 0xffff0000u) | v;
        }
      }
      w = make_uint4(x[0], x[1], x[2], x[3]);
    }
    part[i] = w;
    top = Vec<KIND>::larger(top, Vec<KIND>::largest(w));
  }
  uint32_t most = __reduce_max_sync(0xffffffffu, order_of(Vec<KIND>::most(top)));
  if (lane == 0) sh.most[warp] = most;
  __syncthreads();
  if (warp == 0) {
    most = __reduce_max_sync(0xffffffffu, lane < kWarps ? sh.most[lane] : 0u);
    if (lane == 0) sh.top = most;
  }
  auto meet = [&]() {
    if (n_cta > 1) cluster.sync();
    else __syncthreads();
  };
  meet();
  most = 0;
  for (int o = 0; o < n_cta; ++o) most = max(most, cluster.map_shared_rank(&sh, o)->top);
  const float M = value_of(most);

  // ---- the row's settings
  const float T = p.s.temperature ? p.s.temperature[r] : p.s.temperature_all, top_p = p.s.top_p ? p.s.top_p[r] : p.s.top_p_all;
  const float min_p = p.s.min_p ? p.s.min_p[r] : p.s.min_p_all, u = p.uniform[r];
  const long long top_k = p.s.top_k ? p.s.top_k[r] : p.s.top_k_all;
  // (a NaN among the logits or the settings, nothing above -inf, a temperature below 0)
  const bool none = M != M || M == -CUDART_INF_F || !(T >= 0.f) || top_p != top_p || min_p != min_p || u != u;
  const bool first = T == 0.f || top_k == 1 || top_p <= 0.f;  // the first of the largest alone
  const double inv = T > 0.f ? 1.0 / (double)T : 0.0, least = fmin((double)min_p, 1.0);
  auto weight = [&](float x) {
    if (x == M) return 1.0;
    if (x == -CUDART_INF_F || M == CUDART_INF_F) return 0.0;
    return exp(((double)x - (double)M) * inv);
  };
  auto key_of = [&](float x) { return order_of(x) >> kDrop; };

  // ---- sums over the row, the same in all threads
  int turn = 0;
  auto total = [&](double mass, int count) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, d);
    count = __reduce_add_sync(0xffffffffu, count);
    if (lane == 0) sh.warp[warp].mass = mass, sh.warp[warp].count = count;
    __syncthreads();
    if (warp == 0) {
      mass = lane < kWarps ? sh.warp[lane].mass : 0.0, count = lane < kWarps ? sh.warp[lane].count : 0;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, d);
      count = __reduce_add_sync(0xffffffffu, count);
      if (lane == 0) sh.sum[turn].mass = mass, sh.sum[turn].count = count;
    }
    meet();
    SampleSum s = {0.0, 0};
    for (int o = 0; o < n_cta; ++o) {
      const SampleSum t = cluster.map_shared_rank(&sh, o)->sum[turn];
      s.mass += t.mass, s.count += t.count;
    }
    turn ^= 1;  // (the next sum is written elsewhere: another CTA may still be reading this one)
    return s;
  };
  auto each = [&](auto f) {  // of this thread's values
    for (int i = tid; i < mine; i += THREADS) {
      const uint4 w = part[i];
#pragma unroll
      for (int k = 0; k < kPer; ++k) f(Vec<KIND>::value(w, k));
    }
  };

  // ---- the threshold: values above it are kept, and the first `ties` of those that equal it
  uint32_t edge = 0;  // (below everything)
  int ties = 0;
  const uint32_t edge_most = most >> kDrop;
  if (!none && first) {
    edge = edge_most, ties = 1;
  } else if (!none) {
    if (top_k > 0 && top_k < p.vocab) {  // at least top_k values reach lo, fewer reach hi
      uint32_t lo = 0, hi = edge_most + 1;
      int above = 0;  // that reach hi
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        int n = 0;
        each([&](float x) { n += key_of(x) >= mid; });
        n = total(0.0, n).count;
        if (n >= top_k) lo = mid;
        else hi = mid, above = n;
      }
      edge = lo, ties = (int)top_k - above;
    }
    if (top_p < 1.f) {
      double mass = 0.0;
      each([&](float x) {
        if (key_of(x) > edge) mass += weight(x);
      });
      const double tie = edge == 0 ? 0.0 : weight(value_of(edge << kDrop | (edge << kDrop & 0x80000000u ? 0u : (1u << kDrop) - 1u)));
      const double want = (double)top_p * (total(mass, 0).mass + ties * tie);
      // the weights that reach lo (or equal `edge` and count) are enough, those that reach hi are not
      uint32_t lo = edge, hi = edge_most + 1;
      double above = 0.0;  // that reach hi
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        mass = 0.0;
        each([&](float x) {
          const uint32_t k = key_of(x);
          if (k >= mid && k < hi) mass += weight(x);
        });
        mass = total(mass, 0).mass;
        if (above + mass >= want) lo = mid;
        else hi = mid, above += mass;
      }
      const double one = lo == edge ? tie : weight(value_of(lo << kDrop | (lo << kDrop & 0x80000000u ? 0u : (1u << kDrop) - 1u)));
      double n = one > 0.0 ? ceil((want - above) / one) : 0.0;
      if (n > 1.0 && above + (n - 1.0) * one >= want) n -= 1.0;
      else if (above + n * one < want) n += 1.0;
      const int enough = n < 1.0 ? 1 : n > 1e9 ? 1000000000 : (int)n;
      ties = lo == edge && edge != 0 ? min(ties, enough) : enough;
      edge = lo;
    }
  }

  // ---- what is kept, chunk by chunk (of 32 vectors: neighbouring ids)
  const float edge_value = value_of(edge << kDrop | (edge << kDrop & 0x80000000u ? 0u : (1u << kDrop) - 1u));
  const double edge_weight = edge == 0 ? 0.0 : first ? 1.0 : weight(edge_value) >= least ? weight(edge_value) : 0.0;
  auto above_edge = [&](float x) {  // its weight, if it counts
    if (first || key_of(x) <= edge) return 0.0;
    const double w = weight(x);
    return w >= least ? w : 0.0;
  };
  double mass = 0.0;
  int count = 0;
  if (!none)
    for (int c = warp; c < chunks; c += kWarps) {
      const int i = c * 32 + lane;
      double m = 0.0;
      int n = 0;
      if (i < mine) {
        const uint4 w = part[i];
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const float x = Vec<KIND>::value(w, k);
          m += above_edge(x);
          n += key_of(x) == edge;
        }
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) m += __shfl_xor_sync(0xffffffffu, m, d);
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) chunk_mass[c] = m, chunk_ties[c] = n, mass += m, count += n;
    }
  total(mass, count);
  turn ^= 1;
  // (each CTA's share: its mass above the edge and its ties, of which the first of the row count)
  double all = 0.0, before = 0.0, own = 0.0;
  int ties_left = ties, last = 0;
  int own_ties = 0;  // ties that count from this CTA's first on
  for (int o = 0; o < n_cta; ++o) {
    const SampleSum t = cluster.map_shared_rank(&sh, o)->sum[turn];
    const double m = t.mass + min(t.count, ties_left) * edge_weight;
    if (o == rank) before = all, own = m, own_ties = ties_left;
    if (m > 0.0) last = o;
    ties_left -= min(t.count, ties_left);
    all += m;
  }
  const double want = (double)fmaxf(u, 0.f) * all;
  const bool here = u >= 1.f ? rank == last : want >= before && (want < before + own) && own > 0.0;
  if (none) {
    if (rank == 0 && tid == 0) p.ids[r] = -1, p.logprob[r] = CUDART_NAN_F;
  } else if (here && warp == 0) {
    // the chunk, then the lane, then the value
    double run = before, m = 0.0;
    int left = own_ties, found = -1, found_left = 0;
    double found_run = 0.0;
    for (int c0 = 0; c0 < chunks; c0 += 32) {
      const int c = c0 + lane;
      const int n = c < chunks ? chunk_ties[c] : 0;
      int n_sum = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, n_sum, d);
        if (lane >= d) n_sum += v;
      }
      const int n_before = n_sum - n, counted = min(max(left - n_before, 0), n);
      m = c < chunks ? chunk_mass[c] + counted * edge_weight : 0.0;
      double sum = m;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += v;
      }
      const bool hit = m > 0.0 && (u >= 1.f || run + sum > want);
      const unsigned hits = __ballot_sync(0xffffffffu, hit), some = __ballot_sync(0xffffffffu, m > 0.0);
      const int at = u >= 1.f ? (some ? 31 - __clz(some) : -1) : hits ? __ffs(hits) - 1 : some ? 31 - __clz(some) : -1;
      if (at >= 0) {  // (the last one with a weight, should rounding leave none)
        found = c0 + at;
        found_run = run + __shfl_sync(0xffffffffu, sum - m, at), found_left = left - __shfl_sync(0xffffffffu, n_before, at);
        if (u < 1.f && hits) break;
      }
      run += __shfl_sync(0xffffffffu, sum, 31);
      left -= __shfl_sync(0xffffffffu, n_sum, 31);
    }
    const int i = found * 32 + lane;
    const bool there = found >= 0 && i < mine;
    const uint4 w = there ? part[i] : make_uint4(0, 0, 0, 0);
    int n = 0;
    if (there)
#pragma unroll
      for (int k = 0; k < kPer; ++k) n += key_of(Vec<KIND>::value(w, k)) == edge;
    int n_sum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, n_sum, d);
      if (lane >= d) n_sum += v;
    }
    const int mine_left = found_left - (n_sum - n);
    auto counted = [&](float x, int& left) {
      if (key_of(x) == edge) return left-- > 0 ? edge_weight : 0.0;
      return above_edge(x);
    };
    m = 0.0;
    if (there) {
      int left = mine_left;
#pragma unroll
      for (int k = 0; k < kPer; ++k) m += counted(Vec<KIND>::value(w, k), left);
    }
    double sum = m;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    const unsigned hits = u >= 1.f ? 0u : __ballot_sync(0xffffffffu, m > 0.0 && found_run + sum > want), some = __ballot_sync(0xffffffffu, m > 0.0);
    const int at = hits ? __ffs(hits) - 1 : 31 - __clz(some);
    if (lane == at) {
      double run = found_run + (sum - m), taken = 0.0;
      int left = mine_left, id = -1;
      bool done = false;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const double v = counted(Vec<KIND>::value(w, k), left);
        run += v;
        if (v > 0.0 && !done) {
          taken = v, id = (v0 + i) * kPer - shift + k;
          done = u < 1.f && run > want;
        }
      }
      p.ids[r] = id;
      p.logprob[r] = (float)log(taken / all);
    }
  }
  if (n_cta > 1) cluster.sync();  // (a CTA's memory is there until everybody has read it)
}

template <int KIND, int THREADS>
static int launch_sample(const SampleParams& p, int64_t rows, int ctas, cudaStream_t stream) {
  static bool configured[64] = {};
  const int smem = p.part * 16 + p.part / 32 * 12;
  DeviceInfo di;
  int rc;
  if ((rc = device_info(&di))) return rc;
  if (!configured[di.dev]) {
    BLR_CUDA_OK(cudaFuncSetAttribute(sample_kernel<KIND, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleMaxPart + 512 * 16 + (kSampleMaxPart / 512 + 16) * 12));
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
  BLR_CUDA_OK(cudaLaunchKernelEx(&cfg, sample_kernel<KIND, THREADS>, p));
  return BLR_OK;
}

}  // namespace blr

using namespace blr;

extern "C" {

int blr_sample(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int kind, const float* uniform, const blr_sampling* s, int64_t* ids, float* logprob,
               void* stream) {
  BLR_REQUIRE(kind >= 0 && kind <= 2, BLR_ERR_ARG, "unknown kind of logits %d", kind);
  const int64_t size = kind == 2 ? 4 : 2;
  BLR_REQUIRE(rows >= 0 && rows < (1ll << 28) && vocab > 0 && (rows <= 1 || ld >= vocab), BLR_ERR_ARG, "sample: %lld rows of %lld", (long long)rows, (long long)vocab);
  BLR_REQUIRE(vocab * size <= 8ll * kSampleMaxPart, BLR_ERR_UNSUPPORTED, "sample keeps a row in the shared memory of 8 SMs: at most %lld bytes, not %lld", 8ll * kSampleMaxPart,
              (long long)(vocab * size));
  BLR_REQUIRE(s, BLR_ERR_ARG, "null pointer");
  BLR_REQUIRE(s->temperature || s->temperature_all >= 0.f, BLR_ERR_ARG, "sample: the temperature must not be negative");
  BLR_REQUIRE((s->top_p || s->top_p_all == s->top_p_all) && (s->min_p || s->min_p_all == s->min_p_all), BLR_ERR_ARG, "sample: top_p and min_p must be numbers");
  if (rows == 0) return BLR_OK;
  BLR_REQUIRE(logits && uniform && ids && logprob, BLR_ERR_ARG, "null pointer");
  BLR_REQUIRE(reinterpret_cast<uintptr_t>(logits) % size == 0, BLR_ERR_ARG, "sample: logits must be aligned to their size");
  // a row's part of at most 64 KB, so that three CTAs share an SM; few rows: over more CTAs, as long as each has 4 KB
  int ctas = 1;
  while (ctas < 8 && vocab * size > ctas * 65536ll) ctas *= 2;
  while (ctas < 8 && rows * ctas < 2ll * sm_count() && vocab * size >= ctas * 8192ll) ctas *= 2;
  SampleParams p = {};
  p.logits = logits, p.ld = ld, p.uniform = uniform, p.s = *s;
  p.ids = reinterpret_cast<long long*>(ids), p.logprob = logprob;
  const int64_t per = 16 / size, vecs = (vocab + 2 * per - 2) / per;  // (as many vectors as a row can have, however it is aligned)
  p.vocab = (int)vocab, p.part = (int)(((vecs + ctas - 1) / ctas + 31) / 32 * 32);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define BLR_SAMPLE(THREADS) \
  (kind == 0 ? launch_sample<0, THREADS>(p, rows, ctas, st) : kind == 1 ? launch_sample<1, THREADS>(p, rows, ctas, st) : launch_sample<2, THREADS>(p, rows, ctas, st))
  return p.part <= 2048 ? BLR_SAMPLE(128) : BLR_SAMPLE(512);
#undef BLR_SAMPLE
}

}  // extern "C"
