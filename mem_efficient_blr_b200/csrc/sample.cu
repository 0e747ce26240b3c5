// The next token of rows of logits from a given uniform number u in [0, 1), with temperature T, top-k, top-p and min-p.
//   M = max x,  w_i = e^((x_i - M) / T)  (T = 0: 1 for the first of the largest, 0 else);  order: falling x, equal ones by rising id
//   kept: the first k; of those the fewest first ones whose weights reach p times their sum; of those the ones with w_i >= min_p
//   id = the least kept i with  sum of kept w_j, j <= i  >  u times the sum of all kept,   logprob = log(w_id / that sum)
// Each filter keeps the beginning of the order: what lies above an edge, and the first few that equal it.  The last one goes by ids, so that the row is never sorted.
// A sum may end next to a border (p times the whole, u times the kept), and the token depends on which side: weights and sums are in 64 bits, in an order that depends on the
// row's length and place alone.
//
// One CTA takes a row and keeps it in shared memory, where it fits, or reads it again from L2.
//   The edge of small k, or of short nuclei, is among the few hundred values that reach a number which enough groups of threads have seen reached: they are put in order.  (128 threads, which
//   rows of up to 512 vectors have, are too few groups for a nucleus or k above 128.)
//   Where it is not (long nuclei), a histogram of the row says between which values the edge lies, those above are summed, and so on with those between until they can be
//   put in order or are one value.
//   Where that does not end in a few rounds, the edge is searched for bit by bit, a pass over the row each.  That is every row whose k is more than its threads (the histogram then begins at the
//   lowest number there is, and its bins are even in value), or more than a mask leaves: 4 | 256 rows of 32000 bf16 numbers, k = 1000, 96 | 136 us, k = 50 of 20 that are left 44 | 68 (of 32000:
//   8 | 12), k = 200 of 2000 40 | 47; 256 rows of 150000 fp32 numbers, which do not stay on the chip, k = 1000, 1.9 ms.
// Bound by instructions, not by HBM: 1024 rows of 50001 fp32 numbers drawn from as a whole take 112 us for 31.5 of bytes, 42 instructions a value, 10 of them in 64 bits, at 2.3 a cycle and SM;
// 256 nuclei of 0.9 of 32000 bf16 numbers 36 to 86 us by the inputs, 52 on average, the slowest row counts (2.5): rounds behind barriers, each over the row (256 rows are one wave).  4 rows, k = 50 and p = 0.95: 8.8 us, launch, row, list, order, sums.
// The likeliest alone, 600 rows of 32000: 26 us (5.9 of bytes): behind the row's maximum a second pass over it with the sums' chunks, scans and barriers finds the id.
// A row on a cluster of CTAs: 13 to 22 us for 4 rows, 72 to 150 for the nuclei, 200 to 220 for the whole.
#include <math_constants.h>

#include <type_traits>

#include "../../include/blr_b200.h"
#include "logits.cuh"
#include "tmap.h"

namespace blr {

static constexpr int kStaged = 88 * 1024;          // bytes of a row that is kept in shared memory: two CTAs to an SM
static constexpr int kListed = 512, kBins = 2048;  // values that can be put in order; bins of the histogram
typedef unsigned long long Listed;                 // order_of(value) << 32 | ~id: larger comes first
static constexpr float kSpan = 24.f;               // what the histogram of a nucleus covers: weights from 1 to e^-24

static constexpr int kSampleDynamic = 100 * 1024;                // shared memory of a CTA at most
static constexpr int64_t kSampleMostBytes = 4ll << 20;            // of a row: its chunks' sums fit there

struct SampleParams {
  const void* logits;
  long long ld;
  const float* uniform;
  blr_sampling s;
  long long* ids;
  float* logprob;
  int vocab, chunks;  // chunks: of 32 vectors of 16 bytes, that a row can have
  double series[5];   // log(2) / 256 to the powers 1 to 4 over their factorials; 1.5 2^52
};

struct SampleSum {
  double mass, likely;
  int count;
};

template <int THREADS>
struct SampleShared {
  static constexpr int kWarps = THREADS / 32;
  union alignas(16) {
    struct {
      Listed list[kListed], sorted[kListed];
      double upto[kListed];  // sums over what is sorted
    };
    int hist[kBins];
    uint32_t groups[33 * kWarps];  // (a warp's 32 a word apart from the next one's: lane i reads warp i's)
  };
  double table[256];  // 2^(j / 256)
  SampleSum warp[2][kWarps];
  uint32_t most[kWarps], reach[kWarps], listed;
  float estimate[kWarps];
  int ties, kept, bin, inside, at[2];
};

// e^((x - M) / T) in 64 bits, to 2^-50 of itself and 2^-52 for each unit of (M - x) / T: 2^(n / 256) from the table times the Taylor series of 2^(r / 256), |r| <= 1/2, up to the fourth power,
// which leaves 2^-54 (of 2^(r / 32), with a table of 32 numbers, it left 2^-39, and one more power to 2^-48 cost 1 % of a row that is summed as a whole: 113.8 us for 112.7).  Exactly 1
// at M; for x above `low`, which is next below M, or where e^-700 is.  (A call of exp has three times the instructions, and they are what bounds such a row.)
// (The series' numbers come as the kernel's parameters, where an instruction reads them: as literals each takes two more.)
struct Weight {
  float low;
  double most, c;  // 256 log2(e) / T
  const double *table, *series;
  __device__ __forceinline__ double operator()(float x) const {
    const double d = (double)x - most, s = fma(d, c, series[4]);  // 1.5 2^52: whole numbers end in the last bits
    const int n = __double2loint(s);
    const double r = fma(d, c, -(s - series[4]));
    double e = fma(r, series[3], series[2]);
    e = fma(r, e, series[1]);
    e = fma(r, e, series[0]);
    e = fma(r, e, 1.0) * table[n & 255];
    return __hiloint2double(__double2hiint(e) + ((n & ~255) << 12), __double2loint(e));
  }
  __device__ __forceinline__ double or_zero(float x) const { return x > low ? (*this)(x) : 0.0; }
};

constexpr double power_of_two(double x) {  // its Taylor series, 0 <= x < 1
  double term = 1.0, sum = 1.0;
  for (int i = 1; i < 24; ++i) term *= x * 0.69314718055994530942 / i, sum += term;
  return sum;
}
struct Powers {
  double of[256];
  constexpr Powers() : of() {
    for (int j = 0; j < 256; ++j) of[j] = power_of_two(j / 256.0);
  }
};
__device__ const Powers kPowers = Powers();

template <int KIND>
__device__ __forceinline__ uint32_t raw_logit(const char* row, int id) {  // its bits
  if constexpr (KIND == 2) return reinterpret_cast<const uint32_t*>(row)[id];
  else return reinterpret_cast<const uint16_t*>(row)[id];
}
__device__ __forceinline__ uint32_t sort_falling(uint32_t v, int lane) {  // a warp's values, the largest in lane 0
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const uint32_t o = __shfl_xor_sync(0xffffffffu, v, j);
      v = ((lane & j) == 0) == ((lane & k) == 0) ? max(v, o) : min(v, o);
    }
  return v;
}

// A CTA's row.
template <int KIND, int THREADS, bool STAGED>
struct SampleRow {
  typedef SampleShared<THREADS> Shared;
  static constexpr int kPer = Vec<KIND>::kPer, kSize = KIND == 2 ? 4 : 2, kWarps = Shared::kWarps;
  static constexpr int kDrop = KIND == 0 ? 13 : KIND == 1 ? 16 : 0;  // orders of 16-bit values differ in their upper bits alone
  Shared& sh;
  uint4* const part;
  const char* const row;
  int tid, warp, lane, vecs, id0, vocab, turn;  // vector i has the values from id id0 + i kPer on; -inf where there is none
  float M;
  Weight weight;

  __device__ __forceinline__ static float value_of_key(uint32_t k) { return value_of(k << kDrop | (k << kDrop & 0x80000000u ? 0u : (1u << kDrop) - 1u)); }

  __device__ __forceinline__ uint4 load(int i) const {
    const int id = id0 + i * kPer;
    if (id >= 0 && id + kPer <= vocab) return *reinterpret_cast<const uint4*>(row + (long long)id * kSize);
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = Vec<KIND>::kLowest;
#pragma unroll
      for (int z = 0; z < kPer / 4; ++z) {
        const int at = id + k * (kPer / 4) + z;
        if (at < 0 || at >= vocab) continue;
        const uint32_t v = raw_logit<KIND>(row, at);
        if constexpr (KIND == 2) x[k] = v;
        else x[k] = z ? (x[k] & 0xffffu) | v << 16 : (x[k] & 0xffff0000u) | v;
      }
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
  }
  // inner: known not to be the first or the last
  __device__ __forceinline__ uint4 load_inner(int i) const { return reinterpret_cast<const uint4*>(row + (long long)id0 * kSize)[i]; }
  __device__ __forceinline__ uint4 vec(int i, bool inner = false) const {
    if constexpr (STAGED) return part[i];
    else return inner ? load_inner(i) : load(i);
  }
  // f(vector, its number) of this thread's vectors, AHEAD of them loaded at a time
  template <int AHEAD, typename F>
  __device__ __forceinline__ void each_vector(F f) const {
    for (int i0 = 0; i0 < vecs; i0 += AHEAD * THREADS) {
      const int i = i0 + tid;
      uint4 w[AHEAD];
      if (i0 > 0 && i0 + AHEAD * THREADS < vecs) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) w[a] = vec(i + a * THREADS, true);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) f(w[a], i + a * THREADS);
      } else {
#pragma unroll 1
        for (int k = i; k < min(vecs, i0 + AHEAD * THREADS); k += THREADS) f(vec(k), k);
      }
    }
  }
  // f(value) of this thread's values, in few instructions: what few rows come to is not to push the rest out of the instruction cache
  template <typename F>
  __device__ __forceinline__ void each_seldom(F f) const {
    for (int i = tid; i < vecs; i += THREADS) {
      const uint4 w = vec(i);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (KIND == 2) {
          f(__uint_as_float(ws[k]));
        } else {
          const float2 v = q8_up2<KIND == 1>(ws[k]);
          f(v.x), f(v.y);
        }
      }
    }
  }
  // Sums over the row, the same in all threads.
  template <bool LIKELY = false>
  __device__ __forceinline__ SampleSum total(double mass, double likely, int count) {
    auto add_up = [](double& a, double& b, int& n) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, d);
        if constexpr (LIKELY) b += __shfl_xor_sync(0xffffffffu, b, d);
      }
      n = __reduce_add_sync(0xffffffffu, n);
    };
    add_up(mass, likely, count);
    if (lane == 0) sh.warp[turn][warp] = {mass, likely, count};
    __syncthreads();
    SampleSum s = lane < kWarps ? sh.warp[turn][lane] : SampleSum{0.0, 0.0, 0};
    add_up(s.mass, s.likely, s.count);
    turn ^= 1;  // (the next sums go elsewhere: others may still be reading these)
    return s;
  }
  // What comes before this thread's v, thread by thread, and the sum of all.
  __device__ __forceinline__ double before(double v, double& all) {
    double upto = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 31) sh.warp[turn][warp].mass = upto;
    __syncthreads();
    double warps = lane < kWarps ? sh.warp[turn][lane].mass : 0.0;
#pragma unroll
    for (int d = 1; d < kWarps; d <<= 1) {
      const double o = __shfl_up_sync(0xffffffffu, warps, d);
      if (lane >= d) warps += o;
    }
    turn ^= 1;
    all = __shfl_sync(0xffffffffu, warps, kWarps - 1);
    const double ahead = __shfl_sync(0xffffffffu, warps, (warp + 31) & 31);
    return (warp > 0 ? ahead : 0.0) + (upto - v);
  }
  // This thread's `n` values for the list: where they go (beyond kListed: nowhere).  All threads of a warp come here.
  __device__ __forceinline__ uint32_t reserve(int n) const {
    int upto = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    uint32_t at = 0;
    if (lane == 31 && upto > 0) at = atomicAdd(&sh.listed, (uint32_t)upto);
    return __shfl_sync(0xffffffffu, at, 31) + (uint32_t)(upto - n);
  }

  // Looks for the edge among the n listed values: what is above them in the order has mass `sum`.  Kept are the first `left` of the list, and of those, with what is above,
  // the fewest that reach `share` of their sum (of `whole`, where that is known, >= 0).  False: the list does not reach it; `sum` is then that with the list's.
  __device__ __forceinline__ bool cut(int n, long long left, double& sum, float share, double whole, uint32_t& edge, int& ties) {
    __syncthreads();  // (the list is complete)
    if (n < 1 || n > kListed) return false;
    if (tid == 0) {
      if (n < kListed) sh.list[n] = 0;  // (below all)
      sh.kept = n, sh.ties = 0;
    }
    __syncthreads();
    if (THREADS < kListed || 16 * n <= 5 * THREADS) {
      // each value's place: how many come before it; as many threads to a value as there are
      int by = 1;
      while (by < 32 && 2 * by * n <= THREADS) by *= 2;
      for (int i0 = 0; i0 < n; i0 += THREADS / by) {
        const int i = i0 + tid / by, end = i < n ? (n + 1) / 2 : 0;
        const Listed v = i < n ? sh.list[i] : 0;
        int before = 0;
#pragma unroll 4
        for (int q = tid % by; q < end; q += by) {
          const ulonglong2 o = reinterpret_cast<const ulonglong2*>(sh.list)[q];
          before += (o.x > v) + (o.y > v);
        }
        for (int d = 1; d < by; d <<= 1) before += __shfl_xor_sync(0xffffffffu, before, d);
        if (i < n && tid % by == 0) sh.sorted[before] = v;
      }
    } else {
      // a value for each thread, sorted by comparisons in pairs (cycles by places | like this: 60 values 1900 | 2900, 250 by 1024 threads 4500 | 7400, 300 by 512 14800 | 8900)
      Listed v = tid < n ? sh.list[tid] : 0, *at = sh.sorted;
      __syncthreads();
      for (int k = 2; k <= kListed; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
          Listed o;
          if (j >= 32) {
            if (tid < kListed) at[tid] = v;
            __syncthreads();
            o = tid < kListed ? at[tid ^ j] : 0;
            at = at == sh.sorted ? sh.list : sh.sorted;  // (what has been written here two steps ago has been read by everybody)
          } else {
            o = __shfl_xor_sync(0xffffffffu, v, j);
          }
          if ((o > v) == (((tid & j) == 0) == ((tid & k) == 0))) v = o;
        }
      __syncthreads();
      if (tid < n) sh.sorted[tid] = v;
    }
    __syncthreads();
    bool reaches = left <= n;
    if (share < 1.f) {
      constexpr int kOwn = (kListed + THREADS - 1) / THREADS;  // a thread's neighbours in order
      double run[kOwn], own = 0.0;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int at = tid * kOwn + i;
        own += at < n && at < left ? weight.or_zero(value_of((uint32_t)(sh.sorted[at] >> 32))) : 0.0;
        run[i] = own;
      }
      double all;
      const double ahead = sum + before(own, all);
      all += sum;
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
        if (tid * kOwn + i < kListed) sh.upto[tid * kOwn + i] = ahead + run[i];
      __syncthreads();
      const double want = share * (whole < 0.0 ? all : whole);
      int end = kListed;  // the first one that is not needed
#pragma unroll
      for (int i = kOwn - 1; i >= 0; --i) {
        const int at = tid * kOwn + i;
        if (at > 0 && at < n && (at >= left || sh.upto[at - 1] >= want)) end = at;
      }
      end = __reduce_min_sync(0xffffffffu, end);
      if (lane == 0 && end < kListed) atomicMin(&sh.kept, end);
      if (whole >= 0.0) reaches = all >= want;
      sum = all;
    } else if (tid == 0 && left < n) {
      sh.kept = (int)left;
    }
    __syncthreads();
    if (!reaches) return false;
    const uint32_t e = (uint32_t)(sh.sorted[sh.kept - 1] >> 32);
    int same = 0;
    for (int i = tid; i < sh.kept; i += THREADS) same += (uint32_t)(sh.sorted[i] >> 32) == e;
    same = __reduce_add_sync(0xffffffffu, same);
    if (lane == 0 && same > 0) atomicAdd(&sh.ties, same);
    __syncthreads();
    edge = e >> kDrop, ties = sh.ties;
    return true;
  }

  // The token, where all that is kept are the first sh.kept of the sorted: by their ids.
  __device__ __forceinline__ void pick(double least, float u, long long* id_out, float* logprob_out) {
    const int n = sh.kept;
    double* const mass = reinterpret_cast<double*>(sh.list);
    uint32_t* const ids = reinterpret_cast<uint32_t*>(sh.upto);
    if (tid == 0) sh.at[0] = 0x7fffffff, sh.at[1] = -1;
    int by = 1;
    while (by < 32 && 2 * by * n <= THREADS) by *= 2;
    for (int i0 = 0; i0 < n; i0 += THREADS / by) {
      const int i = i0 + tid / by, end = i < n ? n : 0;
      const Listed v = i < n ? sh.sorted[i] : 0;
      int before = 0;
#pragma unroll 4
      for (int k = tid % by; k < end; k += by) before += (uint32_t)sh.sorted[k] > (uint32_t)v;  // (~id)
      for (int d = 1; d < by; d <<= 1) before += __shfl_xor_sync(0xffffffffu, before, d);
      if (i < n && tid % by == 0) {
        const double w = weight.or_zero(value_of((uint32_t)(v >> 32)));
        mass[before] = w >= least ? w : 0.0, ids[before] = ~(uint32_t)v;
      }
    }
    __syncthreads();
    constexpr int kOwn = (kListed + THREADS - 1) / THREADS;
    double w[kOwn], own = 0.0, all;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int at = tid * kOwn + i;
      w[i] = at < n ? mass[at] : 0.0;
      own += w[i];
    }
    double run = before(own, all);
    const double want = (double)fmaxf(u, 0.f) * all;
    // the first one that goes beyond, or (u = 1, or should rounding leave none) the last one with a weight
    int beyond = 0x7fffffff, with = -1;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      run += w[i];
      if (w[i] > 0.0) {
        with = tid * kOwn + i;
        if (beyond == 0x7fffffff && u < 1.f && run > want) beyond = with;
      }
    }
    beyond = __reduce_min_sync(0xffffffffu, beyond), with = __reduce_max_sync(0xffffffffu, with);
    if (lane == 0 && beyond != 0x7fffffff) atomicMin(&sh.at[0], beyond);
    if (lane == 0 && with >= 0) atomicMax(&sh.at[1], with);
    __syncthreads();
    if (tid == 0) {
      const int at = sh.at[0] != 0x7fffffff ? sh.at[0] : sh.at[1];
      *id_out = ids[at], *logprob_out = (float)log(mass[at] / all);
    }
  }

  // What is known of the edge: it is a value from lo to hi, above hi lies `over` (by count: its mass is not looked after).
  struct Bracket {
    float lo, hi;
    SampleSum over;
  };
  // Counts what lies in the bracket, bin by bin, and says between which values the k-th lies, or those lie at which the weights, as far as counts tell, reach `want`: 0 .. 4 bins; and how
  // many are there at most.  False: it is not among the bins.
  __device__ __forceinline__ bool close_in(const Bracket& b, bool by_count, double want, float log2_per, float& lo, float& hi, int& inside) {
    const float scale = kBins * 0.9999f / (b.hi - b.lo);
    if (!(scale <= 3.0e38f) || !(scale > 0.f)) return false;
    auto bin_of = [&](float x) { return (int)((b.hi - x) * scale); };  // (0 .. kBins - 1 from hi to lo; rises with falling x)
    __syncthreads();
    for (int i = tid; i < kBins; i += THREADS) sh.hist[i] = 0;
    if (tid == 0) sh.bin = kBins, sh.at[0] = -1;
    __syncthreads();
    each_seldom([&](float x) {
      if (x <= b.hi && x >= b.lo) atomicAdd(&sh.hist[bin_of(x)], 1);
    });
    __syncthreads();
    constexpr int kOwn = kBins / THREADS;
    float m[kOwn], run = 0.f;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int bin = tid * kOwn + i;
      const float n = (float)sh.hist[bin];
      float at = b.hi - (bin + 0.5f) / scale;
      if constexpr (KIND != 2) {  // (the 16-bit value in the bin, where they are so far apart that there is one)
        const uint32_t key = order_of(b.hi - bin / scale) >> kDrop;
        const float v0 = value_of_key(key), v1 = value_of_key(key - 1);
        if (v0 <= b.hi && bin_of(v0) == bin) at = v0;
        else if (bin_of(v1) == bin) at = v1;
      }
      m[i] = by_count ? n : n * ex2((at - M) * log2_per);
      run += m[i];
    }
    float upto = run;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    if (lane == 31) sh.estimate[warp] = upto;
    __syncthreads();
    float ahead = upto - run;
    const float need = (float)(want - (by_count ? (double)b.over.count : b.over.mass));
    for (int i = 0; i < warp; ++i) ahead += sh.estimate[i];
    int here = kBins;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      ahead += m[i];
      if (here == kBins && ahead >= need && m[i] > 0.f) here = tid * kOwn + i;
    }
    here = __reduce_min_sync(0xffffffffu, here);
    if (lane == 0 && here < kBins) atomicMin(&sh.bin, here);
    // (where the estimate does not get there: the last bin that has something)
    int last = -1;
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
      if (m[i] > 0.f) last = tid * kOwn + i;
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0) atomicMax(&sh.at[0], last);
    __syncthreads();
    const int bin = sh.bin < kBins ? sh.bin : sh.at[0];
    if (bin < 0) return false;
    // (a bin more on either side than are meant, since the borders of bins are rounded: by count the bin itself is meant, else its neighbours too)
    const int aside = by_count ? 1 : 2;
    inside = 0;
    for (int i = max(bin - aside, 0); i <= min(bin + aside, kBins - 1); ++i) inside += sh.hist[i];
    hi = bin <= aside ? b.hi : fminf(b.hi, b.hi - (bin - aside + 0.5f) / scale);
    lo = bin >= kBins - 1 - aside ? b.lo : fmaxf(b.lo, b.hi - (bin + aside + 0.5f) / scale);
    return true;
  }

  // A few rounds of closing in on the edge, until what is left can be put in order or is one value.  by_count: the k-th value; else the one at which the weights reach `want`.
  __device__ __forceinline__ bool search(Bracket b, bool by_count, long long k, double want, float share, double whole, float log2_per, uint32_t& edge, int& ties) {
#pragma unroll 1
    for (int round = 0; round < 8; ++round) {
      float lo, hi;
      int inside = 0;
      const uint32_t key_lo = order_of(b.lo) >> kDrop, key_hi = order_of(b.hi) >> kDrop;
      const bool single = key_lo == key_hi;
      if (single) {
        lo = b.lo, hi = b.hi;
      } else if (!close_in(b, by_count, want, log2_per, lo, hi, inside)) {
        return false;
      }
      const bool fits = !single && inside <= kListed;
      __syncthreads();  // (the bins make way for the list)
      if (tid == 0) sh.listed = 0;
      __syncthreads();
      // what lies above the new bracket, and in it
      double mass = 0.0, mass_in = 0.0;
      int count = 0, count_in = 0;
      each_seldom([&](float x) {
        if (x < lo || x > b.hi) return;
        const double w = by_count ? 0.0 : weight.or_zero(x);
        if (x > hi) {
          mass += w, ++count;
        } else {
          mass_in += w, ++count_in;
          if (fits) {
            const uint32_t at = atomicAdd(&sh.listed, 1u);
            if (at < kListed) sh.list[at] = (Listed)order_of(x) << 32 | (0xffffffffu - at);  // (in any order among equal ones: only values count here)
          }
        }
      });
      const SampleSum s = total<true>(mass, mass_in, count);
      const int in = total(0.0, 0.0, count_in).count;
      const bool above = by_count ? b.over.count + s.count >= k : b.over.mass + s.mass >= want;
      const bool below = by_count ? b.over.count + s.count + in < k : b.over.mass + s.mass + s.likely < want;
      if (above) {  // (the estimate was too low: it lies above hi)
        if (single) return false;
        b.lo = value_of(order_of(hi) + 1);
        continue;
      }
      b.over.mass += s.mass, b.over.count += s.count;
      if (below) {
        if (single) return false;
        b.over.mass += s.likely, b.over.count += in;
        b.hi = value_below(order_of(lo));
        if (!(b.hi >= b.lo)) return false;
        continue;
      }
      if (fits) return cut(in, by_count ? k - b.over.count : (long long)in, b.over.mass, share, whole, edge, ties);
      if (single) {
        edge = key_hi;
        const double one = weight.or_zero(value_of_key(edge));
        double n = by_count ? (double)(k - b.over.count) : ceil((want - b.over.mass) / one);
        if (!by_count && n > 1.0 && b.over.mass + (n - 1.0) * one >= want) n -= 1.0;
        if (!by_count && b.over.mass + n * one < want) n += 1.0;
        ties = (int)fmin(fmax(n, 1.0), 1e9);
        return true;
      }
      b.lo = lo, b.hi = hi;
    }
    return false;
  }
};

template <int KIND, int THREADS, bool STAGED>
__global__ void __launch_bounds__(THREADS, THREADS == 1024 ? 1 : THREADS == 512 ? 2 : 8) sample_kernel(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) uint4 dynamic[];
  typedef SampleRow<KIND, THREADS, STAGED> Row;
  __shared__ typename Row::Shared sh;
  constexpr int kPer = Row::kPer, kSize = Row::kSize, kWarps = Row::kWarps, kDrop = Row::kDrop;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long r = blockIdx.x;
  const char* const row = static_cast<const char*>(p.logits) + r * p.ld * kSize;
  const int shift = (int)(reinterpret_cast<uintptr_t>(row) & 15) / kSize, vecs = (p.vocab + shift + kPer - 1) / kPer, chunks = (vecs + 31) / 32;
  double* const chunk_mass = reinterpret_cast<double*>(dynamic);
  int* const chunk_ties = reinterpret_cast<int*>(chunk_mass + p.chunks);
  uint4* const part = dynamic + (p.chunks * 12 + 15) / 16;
  Row R = {sh, part, row, tid, warp, lane, vecs, -shift, p.vocab, 0, 0.f, {}};
  for (int i = tid; i < 256; i += THREADS) sh.table[i] = kPowers.of[i];
  if (tid == 0) sh.listed = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float T = p.s.temperature ? p.s.temperature[r] : p.s.temperature_all, top_p = p.s.top_p ? p.s.top_p[r] : p.s.top_p_all;
  const float min_p = p.s.min_p ? p.s.min_p[r] : p.s.min_p_all, u = p.uniform[r];
  const long long top_k = p.s.top_k ? p.s.top_k[r] : p.s.top_k_all;

  // ---- the row, and the largest value that each thread has seen
  uint32_t seen;
  {
    uint32_t top = Vec<KIND>::kLowest;
    constexpr int kAhead = 4;
    for (int i0 = 0; i0 < vecs; i0 += kAhead * THREADS) {
      const int i = i0 + tid;
      const bool inner = i0 > 0 && i0 + kAhead * THREADS < vecs;
      uint4 w[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
        if (inner || i + a * THREADS < vecs) w[a] = inner ? R.load_inner(i + a * THREADS) : R.load(i + a * THREADS);
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
        if (inner || i + a * THREADS < vecs) {
          if constexpr (STAGED) part[i + a * THREADS] = w[a];
          top = Vec<KIND>::larger(top, Vec<KIND>::largest(w[a]));
        }
    }
    seen = tid < vecs ? order_of(Vec<KIND>::most(top)) : 0u;
  }
  bool first = T == 0.f || top_k == 1 || top_p <= 0.f;  // the first of the largest alone
  const bool k_mode = !first && top_k > 0 && top_k < p.vocab, p_mode = !first && top_p < 1.f, listing = k_mode || p_mode;
  // A number that some hundred values reach: of the groups' (threads') largest the one that so many groups reach (0: all values do).
  const int want_listed = k_mode && (top_k <= kListed / 2 || !p_mode) ? (int)min(top_k, (long long)kListed) : 192;
  uint32_t ranked = 0;
  if (listing) {
    ranked = sort_falling(seen, lane);
    sh.groups[33 * warp + lane] = ranked;
  }
  const uint32_t warp_most = __reduce_max_sync(0xffffffffu, seen);
  if (lane == 0) sh.most[warp] = warp_most;
  __syncthreads();
  const uint32_t most = __reduce_max_sync(0xffffffffu, lane < kWarps ? sh.most[lane] : 0u);
  uint32_t reached = 0;
  if (listing) {
    // each warp tries one of its own: the one that has its share of the groups above it; lane i counts those of warp i that reach it
    const uint32_t v = __shfl_sync(0xffffffffu, ranked, min(31, (want_listed + kWarps - 1) / kWarps - 1));
    int n = 0;
    if (lane < kWarps) {
#pragma unroll
      for (int step = 16; step > 0; step >>= 1)
        if (sh.groups[33 * lane + n + step - 1] >= v) n += step;
      n += sh.groups[33 * lane + n] >= v;
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) sh.reach[warp] = n >= want_listed ? v : 0u;
    __syncthreads();
    reached = __reduce_max_sync(0xffffffffu, lane < kWarps ? sh.reach[lane] : 0u);
  }
  const float M = value_of(most);

  // (a NaN among the logits or the settings, nothing above -inf, a temperature below 0)
  if (M != M || M == -CUDART_INF_F || !(T >= 0.f) || top_p != top_p || min_p != min_p || u != u) {
    if (tid == 0) p.ids[r] = -1, p.logprob[r] = CUDART_NAN_F;
    return;
  }
  const double least = fmin((double)min_p, 1.0);
  const Weight weight = {fminf(M - 700.f * T, value_below(most)), (double)M, T > 0.f ? 256.0 * 1.4426950408889634074 / (double)T : 0.0, sh.table, p.series};
  R.M = M, R.weight = weight;
  const float low_p = least > 0.0 ? M + T * 1.0001f * (logf((float)least) - 1e-3f) - 1e-6f * fabsf(M) : -CUDART_INF_F;  // what lies below weighs less than min_p

  // ---- the edge: values above it are kept, and the first `ties` of those that equal it
  const uint32_t edge_most = most >> kDrop, edge_least = order_of(-CUDART_INF_F) >> kDrop;
  uint32_t edge = 0;  // (below everything)
  int ties = 0;
  if (first) {
    edge = edge_most, ties = 1;
  } else if (M == CUDART_INF_F) {  // (the infinite ones share the row)
    int n = 0;
    R.each_seldom([&](float x) { n += x == M; });
    n = R.total(0.0, 0.0, n).count;
    if (k_mode && top_k < n) n = (int)top_k;
    edge = edge_most, ties = p_mode ? (int)ceil((double)top_p * n) : n, first = true;
  } else if (listing) {
    const float reach = value_of(reached), log2_per = 1.44269504f / T;
    // those that reach it: how many, then into the list
    auto reaches = [&](float x, int id) { return (reached == 0 || x >= reach) && id >= 0 && id < p.vocab; };
    int n = 0, at_vector = 0;
    uint32_t vectors = 0;  // of this thread's first 32 that have any; the rest is looked at twice
    if (seen >= reached)
      R.template each_vector<4>([&](const uint4& w, int i) {
        const int v = at_vector++;
        if (reached != 0 && !(Vec<KIND>::most(Vec<KIND>::largest(w)) >= reach)) return;
        if (v < 32) vectors |= 1u << v;
#pragma unroll
        for (int k = 0; k < kPer; ++k) n += reaches(Vec<KIND>::value(w, k), R.id0 + i * kPer + k);
      });
    __syncthreads();  // (the groups make way for the list)
    uint32_t at = R.reserve(n);
    if (n > 0 && at < kListed) {
      auto put = [&](int i) {
        const uint4 w = R.vec(i);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const float x = Vec<KIND>::value(w, k);
          const int id = R.id0 + i * kPer + k;
          if (reaches(x, id) && at < kListed) sh.list[at++] = (Listed)order_of(x) << 32 | (0xffffffffu - (uint32_t)id);
        }
      };
      for (; vectors != 0; vectors &= vectors - 1) put(tid + (__ffs(vectors) - 1) * THREADS);
      for (int i = tid + 32 * THREADS; i < vecs; i += THREADS) put(i);
    }
    bool found = false, with_share = false;
    if (k_mode) {
      // by count; with a share of the first k, if the list has them all
      __syncthreads();
      double none = 0.0;
      found = R.cut((int)min(sh.listed, 0x7fffffffu), top_k, none, p_mode ? top_p : 1.f, -1.0, edge, ties);
      with_share = found;
      if (found) return R.pick(least, u, p.ids + r, p.logprob + r);
      if (!found) {
        // as many values as there are threads that have seen some reach the least of what they have seen
        uint32_t low = __reduce_min_sync(0xffffffffu, tid < vecs ? seen : 0xffffffffu);
        if (lane == 0) sh.reach[warp] = low;
        __syncthreads();
        for (int i = 0; i < kWarps; ++i) low = min(low, sh.reach[i]);
        const float from = top_k <= min(THREADS, vecs) ? value_of(low) : -3.402823466e38f;
        found = R.search({fmaxf(from, -3.402823466e38f), M, {0.0, 0.0, 0}}, true, top_k, (double)top_k, 1.f, -1.0, log2_per, edge, ties);
        if (!found) {
          uint32_t lo = edge_least, hi = edge_most + 1;  // at least top_k values reach lo, fewer reach hi
          int over = 0;                                  // that reach hi
          while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const float at = Row::value_of_key(mid);
            int n = 0;
            R.each_seldom([&](float x) { n += x >= at; });
            n = R.total(0.0, 0.0, n).count;
            if (n >= top_k) lo = mid;
            else hi = mid, over = n;
          }
          edge = lo, ties = (int)top_k - over;
        }
      }
    }
    if (p_mode && !with_share) {
      const uint32_t k_edge = edge;
      const int k_ties = ties;
      const float k_value = k_edge == 0 ? -CUDART_INF_F : Row::value_of_key(k_edge), over_k = fmaxf(k_value, weight.low);
      const double tie = k_edge == 0 ? 0.0 : weight.or_zero(k_value);
      double mass[2] = {}, likely = 0.0;
      R.template each_vector<STAGED ? 1 : 2>([&](const uint4& w, int) {
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const float x = Vec<KIND>::value(w, k);
          const double v = weight(x), c = x > over_k ? v : 0.0;
          mass[k & 1] += c;
          if (x >= low_p) likely += c;  // (or a little less than min_p)
        }
      });
      SampleSum whole = R.template total<true>(mass[0] + mass[1], likely, 0);
      if (k_value >= low_p) whole.likely += k_ties * tie;
      whole.mass += k_ties * tie;
      const double want = (double)top_p * whole.mass;
      if (!(least > 0.0 && whole.likely < want)) {  // (where what min-p keeps does not reach the share, the nucleus has no part in it)
        const int listed = (int)min(sh.listed, 0x7fffffffu);
        found = false;
        SampleSum over = {0.0, 0.0, 0};
        float below = M;
        if (!k_mode) {
          found = R.cut(listed, listed, over.mass, top_p, whole.mass, edge, ties);
          if (found) return R.pick(least, u, p.ids + r, p.logprob + r);
          if (over.mass > 0.0) over.count = listed, below = value_below(reached);  // (it goes on below what was listed)
        }
        const float from = fmaxf(fmaxf(k_value, M - kSpan * T), -3.402823466e38f);
        if (!found && below >= from) found = R.search({from, below, over}, false, 0, want, top_p, whole.mass, log2_per, edge, ties);
        if (!found) {
          // the weights that reach lo (or equal k_edge and count) are enough, those that reach hi are not
          uint32_t lo = max(k_edge, edge_least), hi = edge_most + 1;
          double over = 0.0;  // that reach hi
          while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const float at = Row::value_of_key(mid), end = Row::value_of_key(hi);
            double m = 0.0;
            R.each_seldom([&](float x) {
              if (x >= at && (hi > edge_most || x < end)) m += weight.or_zero(x);
            });
            m = R.total(m, 0.0, 0).mass;
            if (over + m >= want) lo = mid;
            else hi = mid, over += m;
          }
          const double one = weight.or_zero(Row::value_of_key(lo));
          double n = one > 0.0 ? ceil((want - over) / one) : 0.0;
          if (n > 1.0 && over + (n - 1.0) * one >= want) n -= 1.0;
          else if (over + n * one < want) n += 1.0;
          ties = (int)fmin(fmax(n, 1.0), 1e9);
          edge = lo;
        }
        if (edge == k_edge && k_edge != 0) ties = min(ties, k_ties);
      }
    }
  }

  // ---- what is kept, chunk by chunk (of 32 vectors: neighbouring ids)
  const float edge_value = edge == 0 ? -CUDART_INF_F : Row::value_of_key(edge), over_edge = first ? CUDART_INF_F : fmaxf(edge_value, weight.low);
  const double edge_alone = edge == 0 ? 0.0 : first ? 1.0 : weight.or_zero(edge_value), edge_weight = edge_alone >= least ? edge_alone : 0.0;
  const float pass = fmaxf(edge_value, first ? -CUDART_INF_F : low_p);  // (what lies clearly below the edge or min-p is passed over by the vector)
  auto above_edge = [&](float x) {  // its weight, if it counts
    const double w = weight(x);
    return x > over_edge && w >= least ? w : 0.0;
  };
  double mass = 0.0;
  int count = 0;
  auto sum_chunks = [&](auto all_of_it) {  // all_of_it: no edge, no min-p
    constexpr bool kAll = decltype(all_of_it)::value;
    for (int c0 = warp; c0 < chunks; c0 += 4 * kWarps) {  // four chunks of a warp at a time
      double m[4] = {};
      uint32_t n[2] = {};  // a half for each chunk
      uint4 w[4];
      bool any = false;
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int i = (c0 + a * kWarps) * 32 + lane;
        constexpr uint32_t low = Vec<KIND>::kLowest;
        if (c0 > 0 && c0 + 3 * kWarps < chunks - 1) w[a] = R.vec(i, true);
        else w[a] = i < vecs ? R.vec(i) : make_uint4(low, low, low, low);
        if constexpr (!kAll) {
          if (i < vecs && Vec<KIND>::most(Vec<KIND>::largest(w[a])) >= pass) any = true;
          else w[a] = make_uint4(low, low, low, low);
        }
      }
      if (kAll || __any_sync(0xffffffffu, any)) {
        if (kAll || any) {
#pragma unroll
          for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
              const float x = Vec<KIND>::value(w[a], k);
              if constexpr (kAll) {
                m[a] += weight.or_zero(x);
              } else {
                m[a] += above_edge(x);
                n[a >> 1] += x == edge_value ? 1u << 16 * (a & 1) : 0u;
              }
            }
        }
        // each lane goes on with half of what it has: eight lanes have a chunk in the end
        const bool high = lane & 16, odd = lane & 8;
        double e = high ? m[2] : m[0], o = high ? m[3] : m[1];
        e += __shfl_xor_sync(0xffffffffu, high ? m[0] : m[2], 16);
        o += __shfl_xor_sync(0xffffffffu, high ? m[1] : m[3], 16);
        m[0] = (odd ? o : e) + __shfl_xor_sync(0xffffffffu, odd ? e : o, 8);
#pragma unroll
        for (int d = 4; d > 0; d >>= 1) m[0] += __shfl_xor_sync(0xffffffffu, m[0], d);
        if constexpr (!kAll) {
          n[0] = __reduce_add_sync(0xffffffffu, n[0]), n[1] = __reduce_add_sync(0xffffffffu, n[1]);
          n[0] = (high ? n[1] : n[0]) >> (odd ? 16 : 0) & 0xffffu;
        }
      }
      const int c = c0 + (lane >> 3) * kWarps;
      if ((lane & 7) == 0 && c < chunks) chunk_mass[c] = m[0], chunk_ties[c] = (int)n[0], mass += m[0], count += (int)n[0];
    }
  };
  if (edge == 0 && !(least > 0.0)) sum_chunks(std::true_type());
  else sum_chunks(std::false_type());
  const SampleSum kept = R.total(mass, 0.0, count);
  const double all = kept.mass + min(kept.count, ties) * edge_weight, want = (double)fmaxf(u, 0.f) * all;
  const bool to_end = u >= 1.f;

  // ---- the chunk: a thread has some neighbours, their ties that count and their masses, and what comes before both
  const int each = (chunks + THREADS - 1) / THREADS, c0 = min(tid * each, chunks), c1 = min(c0 + each, chunks);
  int n = 0;
  for (int c = c0; c < c1; ++c) n += chunk_ties[c];
  int n_upto = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, n_upto, d);
    if (lane >= d) n_upto += v;
  }
  if (lane == 31) sh.reach[warp] = n_upto;
  if (tid == 0) sh.at[0] = 0x7fffffff, sh.at[1] = -1;
  __syncthreads();
  int left = ties - (n_upto - n);
  for (int i = 0; i < warp; ++i) left -= (int)sh.reach[i];
  double m = 0.0;
  {
    int l = left;
    for (int c = c0; c < c1; ++c) m += chunk_mass[c] + min(max(l, 0), chunk_ties[c]) * edge_weight, l -= chunk_ties[c];
  }
  double sum;
  double run = R.before(m, sum);
  // the first thread that goes beyond, or, should rounding leave none, the last one with a mass
  const unsigned hits = __ballot_sync(0xffffffffu, m > 0.0 && !to_end && run + m > want), some = __ballot_sync(0xffffffffu, m > 0.0);
  if (lane == 0 && hits) atomicMin(&sh.at[0], tid + __ffs(hits) - 1);
  if (lane == 0 && some) atomicMax(&sh.at[1], tid + 31 - __clz(some));
  __syncthreads();
  const int owner = sh.at[0] != 0x7fffffff ? sh.at[0] : sh.at[1];
  if (owner >> 5 != warp) return;
  int chunk = c0;
  {  // (of the owner's chunks, the first that goes beyond, or the last one with a mass)
    double before = run;
    int l = left, best = -1, best_left = 0;
    double best_run = 0.0;
    for (int c = c0; c < c1; ++c) {
      const double v = chunk_mass[c] + min(max(l, 0), chunk_ties[c]) * edge_weight;
      if (v > 0.0) {
        best = c, best_left = l, best_run = before;
        if (!to_end && before + v > want) break;
      }
      before += v, l -= chunk_ties[c];
    }
    chunk = __shfl_sync(0xffffffffu, best, owner & 31);
    left = __shfl_sync(0xffffffffu, best_left, owner & 31);
    run = __shfl_sync(0xffffffffu, best_run, owner & 31);
  }
  // ---- the lane, then the value
  const int i = chunk * 32 + lane;
  const bool there = chunk >= 0 && i < vecs;
  const uint4 w = there ? R.vec(i) : make_uint4(0, 0, 0, 0);
  n = 0;
  if (there)
#pragma unroll
    for (int k = 0; k < kPer; ++k) n += Vec<KIND>::value(w, k) == edge_value;
  n_upto = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, n_upto, d);
    if (lane >= d) n_upto += v;
  }
  left -= n_upto - n;
  double v[kPer];
  m = 0.0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const float x = Vec<KIND>::value(w, k);
    v[k] = !there ? 0.0 : x == edge_value ? (left-- > 0 ? edge_weight : 0.0) : above_edge(x);
    m += v[k];
  }
  double upto = m;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double o = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += o;
  }
  const unsigned beyond = to_end ? 0u : __ballot_sync(0xffffffffu, m > 0.0 && run + upto > want), with = __ballot_sync(0xffffffffu, m > 0.0);
  if (lane == (beyond ? __ffs(beyond) - 1 : 31 - __clz(with))) {
    double taken = 0.0;
    run += upto - m;
    int id = -1;
    bool done = false;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      run += v[k];
      if (v[k] > 0.0 && !done) {
        taken = v[k], id = R.id0 + i * kPer + k;
        done = !to_end && run > want;
      }
    }
    p.ids[r] = id;
    p.logprob[r] = (float)log(taken / all);
  }
}

template <int KIND, int THREADS, bool STAGED>
static int launch_sample(const SampleParams& p, int64_t rows, cudaStream_t stream) {
  static bool configured[64] = {};
  const int64_t smem = (p.chunks * 12 + 15) / 16 * 16 + (STAGED ? p.chunks * 512ll : 0);
  DeviceInfo di;
  int rc;
  if ((rc = device_info(&di))) return rc;
  if (!configured[di.dev]) {
    BLR_CUDA_OK(cudaFuncSetAttribute(sample_kernel<KIND, THREADS, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleDynamic));
    configured[di.dev] = true;
  }
  return q8_launch(sample_kernel<KIND, THREADS, STAGED>, dim3((unsigned)rows), THREADS, (int)smem, stream, p);
}

}  // namespace blr

using namespace blr;

extern "C" {

int blr_sample(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int kind, const float* uniform, const blr_sampling* s, int64_t* ids, float* logprob,
               void* stream) {
  BLR_REQUIRE(kind >= 0 && kind <= 2, BLR_ERR_ARG, "unknown kind of logits %d", kind);
  const int64_t size = kind == 2 ? 4 : 2;
  BLR_REQUIRE(rows >= 0 && rows < (1ll << 31) && vocab > 0 && (rows <= 1 || ld >= vocab), BLR_ERR_ARG, "sample: %lld rows of %lld", (long long)rows, (long long)vocab);
  BLR_REQUIRE(vocab * size <= kSampleMostBytes, BLR_ERR_UNSUPPORTED, "sample takes rows of at most %lld bytes, not %lld", (long long)kSampleMostBytes, (long long)(vocab * size));
  BLR_REQUIRE(s, BLR_ERR_ARG, "null pointer");
  BLR_REQUIRE(s->temperature || s->temperature_all >= 0.f, BLR_ERR_ARG, "sample: the temperature must not be negative");
  BLR_REQUIRE((s->top_p || s->top_p_all == s->top_p_all) && (s->min_p || s->min_p_all == s->min_p_all), BLR_ERR_ARG, "sample: top_p and min_p must be numbers");
  if (rows == 0) return BLR_OK;
  BLR_REQUIRE(logits && uniform && ids && logprob, BLR_ERR_ARG, "null pointer");
  BLR_REQUIRE(reinterpret_cast<uintptr_t>(logits) % size == 0, BLR_ERR_ARG, "sample: logits must be aligned to their size");
  SampleParams p = {};
  p.logits = logits, p.ld = ld, p.uniform = uniform, p.s = *s;
  p.ids = reinterpret_cast<long long*>(ids), p.logprob = logprob;
  const int64_t per = 16 / size, vecs = (vocab + 2 * per - 2) / per;  // (as many vectors as a row can have, however it is aligned)
  p.vocab = (int)vocab, p.chunks = (int)((vecs + 31) / 32);
  for (int i = 0; i < 4; ++i) p.series[i] = (i > 0 ? p.series[i - 1] : 1.0) * (0.69314718055994530942 / 256.0) / (i + 1);
  p.series[4] = 6755399441055744.0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define BLR_SAMPLE(THREADS, STAGED) \
  (kind == 0 ? launch_sample<0, THREADS, STAGED>(p, rows, st) : kind == 1 ? launch_sample<1, THREADS, STAGED>(p, rows, st) : launch_sample<2, THREADS, STAGED>(p, rows, st))
  // Threads, both sides measured (us from a graph, 16-bit logits; k: k = 50 and p = 0.95, nucleus: p = 0.9):
  // rows of up to 512 vectors have 128, eight to an SM (1000 values, k: 4 rows 7.5, with 512 threads 25.9; 600 rows 12 | 69; 600 nuclei 46 | 56);
  // what is kept in shared memory 512, two to an SM, although there is an SM for each (32000 values, 4 rows: k 8.6, with 1024 threads 9.9; the whole row 12.2 | 11.7, nucleus 37 | 36);
  // what is not 1024 where there is an SM for each row (150000 values, 4 rows: k 14.1, with 512 threads 16.6; the whole row 33 | 40).
  // Keeping a row saves what L2 takes to give it again (32000 values, 600 rows: greedy 25.8, read again 27.4; nucleus 112 | 115).  None of these was measured with a k beyond the list.
  if (vecs <= 512) return BLR_SAMPLE(128, true);
  if (p.chunks * 512ll <= kStaged) return BLR_SAMPLE(512, true);
  return rows <= sm_count() ? BLR_SAMPLE(1024, false) : BLR_SAMPLE(512, false);
#undef BLR_SAMPLE
}

}  // extern "C"
