// What the kernels around a key / value cache in pages share: its layout.
#pragma once
#include "q8.cuh"

namespace blr {

// Slot s of a sequence lies in page table[seq][s / page] of the pool, at place s % page; a number that is no page of the pool: nowhere.  Strides count 16-bit values.
struct PagedView {
  uint16_t *k, *v;
  long long k_page, k_head, k_slot, v_page, v_head, v_slot;
  const int* table;
  long long ld_table;
  int kv_heads, pages, page_log2, slots;  // slots of a sequence: those that its row of the table has pages for
};

int paged_view(const blr_paged_cache* cache, PagedView* out);  // checks the cache's description

// ---- attention: what the kernels share
struct PagedAttnParams {
  PagedView c;
  const uint16_t* q;
  uint16_t* out;
  long long ldq, ldo;
  const long long *start, *n_new;
  float* part;       // ns > 1: of each (sequence, kv head, row, split) hd sums, the maximum that they are taken against, the sum of the weights, 2 free
  unsigned* status;  // NULL, or where a wait that gave up is noted
  float scale_log2;
  int T, H, G, rows, q_tiles, ns, n_bh, n_seq;
  int room;  // CTAs that the SMs hold
};

// Slots that a row of token t sees.
__device__ __forceinline__ int paged_seen(long long start, long long count, long long t, int slots) {
  if (t >= count) return 0;
  const long long n = min(start, (long long)slots) + t + 1;
  return n <= 0 ? 0 : n > slots ? slots : (int)n;
}
// The slots that the last of rows [r0, r1) of a kv head sees: 0 where none of them is a token.
__device__ __forceinline__ int paged_seen_by(const PagedAttnParams& p, long long start, long long count, int r0, int r1) {
  r1 = min(r1, p.rows);
  if (r0 >= r1 || r0 / p.G >= count) return 0;
  return paged_seen(start, count, min((long long)((r1 - 1) / p.G), count - 1), p.c.slots);
}

// How the keys of a row tile, `keys` of them, are shared out: its CTAs take this many each, in multiples of `grain`.  As few as let the CTAs that the SMs hold at a time take all row
// tiles of all sequences, none by more than ns; a tile of `light` rows or fewer counts 7/8.  By the sequences' lengths, which the host does not know: every warp works it out for
// itself.
__device__ __forceinline__ int paged_share(const PagedAttnParams& p, int keys, int rows, int per, int light, int grain, int lane) {
  const int n = p.n_seq * p.q_tiles;
  int ctas = p.ns;
  if (n > 1) {
    auto cost = [&](int i) {  // keys of sequence i / q_tiles for its tile i % q_tiles, in eighths of a grain
      const int b = i / p.q_tiles, r0 = (i - b * p.q_tiles) * per;
      const long long count = p.n_new == nullptr ? p.T : min((long long)p.T, p.n_new[b]);
      return (paged_seen_by(p, p.start[b], count, r0, r0 + per) + grain - 1) / grain * (p.rows - r0 <= light ? 7 : 8);
    };
    const int first = lane < n ? cost(lane) : 0;  // (most calls have no more than 32)
    int most = first;                             // in grains
    for (int i = lane + 32; i < n; i += 32) most = max(most, cost(i));
    most = max(1, (__reduce_max_sync(0xffffffffu, most) + 7) / 8);
    int least = (most + p.ns - 1) / p.ns;
    while (least < most) {
      const int s = (least + most) / 2;
      const float part = __frcp_rn(8.f * s) * 0.999999f;  // (an integer division costs ten times as much; one CTA more or less is no harm)
      int sum = (int)ceilf(first * part);
      for (int i = lane + 32; i < n; i += 32) sum += (int)ceilf(cost(i) * part);
      if ((long long)__reduce_add_sync(0xffffffffu, sum) * p.c.kv_heads <= p.room) most = s;
      else least = s + 1;
    }
    ctas = ((keys + grain - 1) / grain * (rows <= light ? 7 : 8) + 8 * most - 1) / (8 * most);
  }
  ctas = max(ctas, 1);
  return max(1, ((keys + grain - 1) / grain + ctas - 1) / ctas) * grain;
}

static constexpr int kPagedPromptRows = 256;  // rows of a CTA of the kernel for many
bool paged_prompt_fits(const blr_paged_cache* cache);
int paged_launch_prompt(const PagedAttnParams& p, const blr_paged_cache* cache, bool bf16, cudaStream_t stream);

}  // namespace blr
