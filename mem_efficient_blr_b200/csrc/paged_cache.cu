// A key / value cache in pages: written as the rotary embedding makes the keys.
//
//   (x_i, x_{i + hd/2}) -> (x_i c_i - x_{i + hd/2} s_i, x_{i + hd/2} c_i + x_i s_i)  for q and k, with the angles of the token's slot; v as it is
// in fp32, one rounding to the values' type.  q goes to rows of its own, k and v to the pages that the sequence's table names.
// Bound by HBM for prompts, by the launch for a step: 2048 tokens, 32 heads of 128: 102 MB in 18.7 us from inputs that come from HBM (5.4 TB/s; 8.6 of 14 stalled warps wait for their
// loads), 16 x 1 tokens 2.2 us from a graph.
#include "../../include/blr_b200.h"
#include "paged.cuh"
#include "tmap.h"

namespace blr {

int paged_view(const blr_paged_cache* c, PagedView* out) {
  BLR_REQUIRE(c != nullptr, BLR_ERR_ARG, "null cache");
  BLR_REQUIRE(c->n_seq >= 0 && c->pages >= 0 && c->kv_heads > 0 && c->pages_per_seq > 0, BLR_ERR_ARG, "a paged cache needs kv_heads and a table of pages");
  BLR_REQUIRE(c->head_dim == 64 || c->head_dim == 128, BLR_ERR_UNSUPPORTED, "paged caches have heads of 64 or 128 values, got %d", c->head_dim);
  BLR_REQUIRE(c->page == 16 || c->page == 32 || c->page == 64 || c->page == 128, BLR_ERR_UNSUPPORTED, "a paged cache has pages of 16, 32, 64 or 128 slots, got %d", c->page);
  BLR_REQUIRE(c->n_seq * c->kv_heads < (1ll << 31) && c->pages < (1ll << 31) && c->pages_per_seq <= (1ll << 30) / c->page, BLR_ERR_SHAPE, "a paged cache of too many pages or sequences");
  BLR_REQUIRE(c->n_seq <= 1 || c->ld_table >= c->pages_per_seq, BLR_ERR_ARG, "the table's rows overlap");
  for (const int64_t* s : {c->k_strides, c->v_strides})
    for (int i = 0; i < 3; ++i) BLR_REQUIRE(s[i] > 0 && s[i] % 8 == 0, BLR_ERR_ARG, "a paged cache's strides are positive multiples of 8 values");
  if (c->n_seq > 0) {
    BLR_REQUIRE(c->table && (c->pages == 0 || (c->k && c->v)), BLR_ERR_ARG, "null pointer");
    BLR_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) == 0 && (reinterpret_cast<uintptr_t>(c->table) & 3) == 0, BLR_ERR_ARG,
                "a paged cache needs 16-byte aligned pages and a 4-byte aligned table");
  }
  out->k = static_cast<uint16_t*>(c->k), out->v = static_cast<uint16_t*>(c->v);
  out->k_page = c->k_strides[0], out->k_head = c->k_strides[1], out->k_slot = c->k_strides[2];
  out->v_page = c->v_strides[0], out->v_head = c->v_strides[1], out->v_slot = c->v_strides[2];
  out->table = c->table, out->ld_table = c->ld_table;
  out->kv_heads = c->kv_heads, out->pages = (int)c->pages;
  out->page_log2 = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
  out->slots = (int)(c->pages_per_seq << out->page_log2);
  return BLR_OK;
}

struct PagedAppendParams {
  PagedView c;
  const uint16_t *q, *k, *v;
  uint16_t* q_out;
  long long ldq, ldk, ldv, ldo;
  const float *cos_t, *sin_t;
  const long long *start, *n_new;
  uint32_t items;  // warps: rows x parts
  int T, H, heads, parts, positions;  // heads: of q, k and v; parts of a row; positions: slots that have angles
};

// 8 lanes share a row of a head: lane e holds E = hd / 16 neighbouring values of each half, the pairs that the rotation turns.
template <int E>
struct Halves {
  uint32_t x[E / 2], y[E / 2];
  __device__ __forceinline__ void load(const uint16_t* row, int e) {
    if constexpr (E == 8) {
      const uint4 p = *reinterpret_cast<const uint4*>(row + e * E), r = *reinterpret_cast<const uint4*>(row + 8 * E + e * E);
      x[0] = p.x, x[1] = p.y, x[2] = p.z, x[3] = p.w, y[0] = r.x, y[1] = r.y, y[2] = r.z, y[3] = r.w;
    } else {
      const uint2 p = *reinterpret_cast<const uint2*>(row + e * E), r = *reinterpret_cast<const uint2*>(row + 8 * E + e * E);
      x[0] = p.x, x[1] = p.y, y[0] = r.x, y[1] = r.y;
    }
  }
  __device__ __forceinline__ void store(uint16_t* row, int e) const {
    if constexpr (E == 8) {
      *reinterpret_cast<uint4*>(row + e * E) = make_uint4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<uint4*>(row + 8 * E + e * E) = make_uint4(y[0], y[1], y[2], y[3]);
    } else {
      *reinterpret_cast<uint2*>(row + e * E) = make_uint2(x[0], x[1]);
      *reinterpret_cast<uint2*>(row + 8 * E + e * E) = make_uint2(y[0], y[1]);
    }
  }
  template <bool BF16>
  __device__ __forceinline__ void rotate(const float (&c)[E], const float (&s)[E]) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 a = q8_up2<BF16>(x[i]), b = q8_up2<BF16>(y[i]);
      x[i] = q8_down2<BF16>(a.x * c[2 * i] - b.x * s[2 * i], a.y * c[2 * i + 1] - b.y * s[2 * i + 1]);
      y[i] = q8_down2<BF16>(b.x * c[2 * i] + a.x * s[2 * i], b.y * c[2 * i + 1] + a.y * s[2 * i + 1]);
    }
  }
};
template <int E>
__device__ __forceinline__ void angles(const float* t, int e, float (&c)[E]) {
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    const float4 f = *reinterpret_cast<const float4*>(t + e * E + 4 * i);
    c[4 * i] = f.x, c[4 * i + 1] = f.y, c[4 * i + 2] = f.z, c[4 * i + 3] = f.w;
  }
}

// A warp has 4 U heads of a token, of those of q, k and v one behind another: it asks for all of them before it turns the first.
static constexpr int kPagedWarps = 8;

template <bool BF16, int E, int U>
__global__ void __launch_bounds__(32 * kPagedWarps) rope_append_paged_kernel(const __grid_constant__ PagedAppendParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int hd = 16 * E;
  const int lane = threadIdx.x & 31, sub = lane >> 3, e = lane & 7;
  const uint32_t item = blockIdx.x * kPagedWarps + (threadIdx.x >> 5), row = item / (uint32_t)p.parts, b = row / (uint32_t)p.T, t = row - b * p.T;
  const int h0 = (int)(item - row * p.parts) * 4 * U + sub, KV = p.c.kv_heads;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (item >= p.items) return;
  const long long slot = min(p.start[b], (long long)p.c.slots) + t;
  bool live = (p.n_new == nullptr || (long long)t < p.n_new[b]) && slot >= 0 && slot < p.c.slots && slot < p.positions;
  int page = live ? p.c.table[(long long)b * p.c.ld_table + (slot >> p.c.page_log2)] : -1;
  live = page >= 0 && page < p.c.pages;
  Halves<E> a[U] = {};
  if (live) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + 4 * u;
      if (h < p.heads)
        a[u].load(h < p.H ? p.q + row * p.ldq + (long long)h * hd : h < p.H + KV ? p.k + row * p.ldk + (long long)(h - p.H) * hd : p.v + row * p.ldv + (long long)(h - p.H - KV) * hd, e);
    }
    float c[E], s[E];
    angles<E>(p.cos_t + slot * (hd / 2), e, c);
    angles<E>(p.sin_t + slot * (hd / 2), e, s);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h0 + 4 * u < p.H + KV) a[u].template rotate<BF16>(c, s);
  }
  const long long in = slot & ((1 << p.c.page_log2) - 1);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + 4 * u;
    if (h < p.H) a[u].store(p.q_out + row * p.ldo + (long long)h * hd, e);
    else if (live && h < p.H + KV) a[u].store(p.c.k + page * p.c.k_page + (h - p.H) * p.c.k_head + in * p.c.k_slot, e);
    else if (live && h < p.heads) a[u].store(p.c.v + page * p.c.v_page + (h - p.H - KV) * p.c.v_head + in * p.c.v_slot, e);
  }
}

}  // namespace blr

using namespace blr;

extern "C" {

int blr_rope_append_paged(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const float* cos_table, const float* sin_table,
                          int64_t positions, const int64_t* start, const int64_t* n_new, int64_t n_tok, int heads, int dtype, const blr_paged_cache* cache,
                          void* q_out, int64_t ldo, void* stream) {
  PagedAppendParams p = {};
  int rc;
  if ((rc = paged_view(cache, &p.c))) return rc;
  BLR_REQUIRE(dtype == BLR_DTYPE_F16 || dtype == BLR_DTYPE_BF16, BLR_ERR_ARG, "unknown dtype %d", dtype);
  BLR_REQUIRE(n_tok >= 0 && n_tok < (1ll << 31) && heads > 0 && heads < (1 << 20) && positions >= 0, BLR_ERR_ARG, "rope_append_paged: n_tok = %lld, heads = %d", (long long)n_tok,
              heads);
  BLR_REQUIRE((ldq | ldk | ldv | ldo) % 8 == 0, BLR_ERR_ARG, "rope_append_paged: row strides must be multiples of 8");
  if (cache->n_seq == 0 || n_tok == 0) return BLR_OK;
  BLR_REQUIRE(q && k && v && cos_table && sin_table && start && q_out, BLR_ERR_ARG, "null pointer");
  BLR_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(q_out) |
                reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) & 15) == 0, BLR_ERR_ARG,
              "rope_append_paged needs 16-byte aligned pointers");
  p.q = static_cast<const uint16_t*>(q), p.k = static_cast<const uint16_t*>(k), p.v = static_cast<const uint16_t*>(v);
  p.q_out = static_cast<uint16_t*>(q_out);
  p.ldq = ldq, p.ldk = ldk, p.ldv = ldv, p.ldo = ldo;
  p.cos_t = cos_table, p.sin_t = sin_table;
  p.start = reinterpret_cast<const long long*>(start), p.n_new = reinterpret_cast<const long long*>(n_new);
  p.T = (int)n_tok, p.H = heads, p.heads = heads + 2 * cache->kv_heads, p.positions = (int)(positions < p.c.slots ? positions : p.c.slots);
  const long long rows = cache->n_seq * n_tok;
  // 16 heads a warp where that leaves the SMs 16 warps each, 4 else: a prompt of 2048 tokens 13.7 us from a graph, by fours 15.4; 5 x 777 tokens of 36 heads of 64 6.2 | 7.9;
  // 16 x 1 tokens by fours 2.2, by sixteens 2.8.
  const bool wide = rows * ((p.heads + 15) / 16) >= 16ll * sm_count();
  const int per = wide ? 16 : 4;
  p.parts = (p.heads + per - 1) / per;
  const long long items = rows * p.parts, ctas = (items + kPagedWarps - 1) / kPagedWarps;
  BLR_REQUIRE(items < (1ll << 31) - kPagedWarps, BLR_ERR_SHAPE, "too many tokens");
  p.items = (uint32_t)items;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel) { return q8_launch(kernel, dim3((unsigned)ctas), 32 * kPagedWarps, 0, st, p); };
  const bool bf = dtype == BLR_DTYPE_BF16;
  if (cache->head_dim == 128)
    return bf ? (wide ? go(rope_append_paged_kernel<true, 8, 4>) : go(rope_append_paged_kernel<true, 8, 1>))
              : (wide ? go(rope_append_paged_kernel<false, 8, 4>) : go(rope_append_paged_kernel<false, 8, 1>));
  return bf ? (wide ? go(rope_append_paged_kernel<true, 4, 4>) : go(rope_append_paged_kernel<true, 4, 1>))
            : (wide ? go(rope_append_paged_kernel<false, 4, 4>) : go(rope_append_paged_kernel<false, 4, 1>));
}

}  // extern "C"
