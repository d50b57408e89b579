// pages.h — moving tokens of a paged cache, all layers in one launch: copies of pages, and the drafted tokens that stay
// closed up behind the tokens before them.
#pragma once

#include "serve.h"

namespace trellis {

constexpr int PAGE_LAYERS = 32;   // layers of one launch (their pointers travel in its arguments)
constexpr int PAGE_AHEAD = 4;     // rows of keys, and of values, that a lane group has in flight

struct Layers {
  void* k[PAGE_LAYERS];
  void* v[PAGE_LAYERS];
  float* scores[PAGE_LAYERS];
  int32_t* pos[PAGE_LAYERS];
};

// 16 bytes of a key's and a value's row a lane, lpr lanes (a power of 2) a row.
struct RowPair {
  u32x4_t k, v;
};
__device__ __forceinline__ RowPair load_rows(const Layers& l, int layer, long long at, int sub) {
  return {*reinterpret_cast<const u32x4_t*>(static_cast<const char*>(l.k[layer]) + 2 * at + 16 * sub),
          *reinterpret_cast<const u32x4_t*>(static_cast<const char*>(l.v[layer]) + 2 * at + 16 * sub)};
}
// NT: nontemporal stores.
template <bool NT = false>
__device__ __forceinline__ void store_rows(const Layers& l, int layer, long long at, int sub, RowPair r) {
  u32x4_t* k = reinterpret_cast<u32x4_t*>(static_cast<char*>(l.k[layer]) + 2 * at + 16 * sub);
  u32x4_t* v = reinterpret_cast<u32x4_t*>(static_cast<char*>(l.v[layer]) + 2 * at + 16 * sub);
  if constexpr (NT) {
    __builtin_nontemporal_store(r.k, k);
    __builtin_nontemporal_store(r.v, v);
  } else {
    *k = r.k;
    *v = r.v;
  }
}

// Page dst[i] takes the first counts[i] tokens of page src[i] (all without counts); a page outside the pool, or onto
// itself: nothing. A workgroup takes PAGE_AHEAD rows a lane group of one (layer, copy, head): `parts` of them a page.
// Bound: memory (12 layers x 40 pages of 64 tokens of 8 heads of 128 with scores and positions, 256 MB moved: 41.8 us, 6.1 TB/s;
// 54.6 with plain stores, 42.2 with nontemporal loads alone, 47.0 with both).
struct CopyArgs {
  Cache c;
  Layers l;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* counts;   // or null
  int n;
};

template <bool NT>
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a, int lpr, int parts) {
  const int part = blockIdx.x % parts;
  const unsigned rest = blockIdx.x / parts;
  const int head = rest % a.c.heads;
  const unsigned unit = rest / a.c.heads;
  const int i = unit % a.n, layer = unit / a.n;
  const int src = load_const(a.src + i), dst = load_const(a.dst + i), page = 1 << a.c.page_shift;
  const int count = a.counts ? min(load_const(a.counts + i), page) : page;
  if (static_cast<unsigned>(src) >= static_cast<unsigned>(a.c.pages) ||
      static_cast<unsigned>(dst) >= static_cast<unsigned>(a.c.pages) || src == dst)
    return;
  const int groups = 256 / lpr, sub = threadIdx.x & (lpr - 1), group = threadIdx.x / lpr;
  const int first = part * groups * PAGE_AHEAD;
  const bool own = sub * 8 < a.c.d;
  RowPair r[PAGE_AHEAD];
#pragma unroll
  for (int u = 0; u < PAGE_AHEAD; ++u) {
    const int slot = first + u * groups + group;
    if (own && slot < count) r[u] = load_rows(a.l, layer, a.c.row_at(src, head, slot), sub);
  }
#pragma unroll
  for (int u = 0; u < PAGE_AHEAD; ++u) {
    const int slot = first + u * groups + group;
    if (own && slot < count) store_rows<NT>(a.l, layer, a.c.row_at(dst, head, slot), sub, r[u]);
  }
  for (int slot = first + threadIdx.x; slot < min(count, first + groups * PAGE_AHEAD); slot += 256) {
    const long long s = a.c.slot_at(src, head, slot), t = a.c.slot_at(dst, head, slot);
    if (a.l.scores[layer]) a.l.scores[layer][t] = a.l.scores[layer][s];
    if (a.l.pos[layer]) a.l.pos[layer][t] = a.l.pos[layer][s];
  }
}

// Of row b's n = starts[b + 1] - starts[b] newest tokens, in the slots from base = lens[b] - n on, those on its path stay:
// token path[b][i] moves to slot base + i. The path ends where an entry is not above the one before it, or not below n.
// In place: an entry is at least its own number, so a slot is read no later than its group of tokens is written (the
// barrier), and groups go upwards. One workgroup a (layer, row, head).
// Bound: the chain length -> path -> page ids -> rows for the few tokens of a step (16 rows of up to 6 tokens, 12 layers of
// 8 heads of 128: 5.5 us), memory beyond (48 rows of up to 90, 30 layers of 3 heads of 64: 17.5 us, 71 MB, 4.1 TB/s).
struct KeepArgs {
  Cache c;
  Layers l;
  const int32_t* starts;
  const int32_t* path;
  long long path_stride;
  int path_width;
  int32_t* new_lens;   // null: not this launch's
};

__global__ __launch_bounds__(256) void keep_kernel(KeepArgs a, int lpr) {
  __shared__ int s_end;
  const int tid = threadIdx.x, lane = tid & 63;
  const int head = blockIdx.x % a.c.heads;
  const unsigned unit = blockIdx.x / a.c.heads;
  const int b = unit % a.c.rows, layer = unit / a.c.rows;
  const int len = load_const(a.c.lens + b);
  const long long fresh = static_cast<long long>(load_const(a.starts + b + 1)) - load_const(a.starts + b);
  const int n = static_cast<int>(max(0ll, min(fresh, 0x7fffffffll)));
  const long long base = static_cast<long long>(len) - n;
  const int32_t* path = a.path + b * a.path_stride;
  if (tid == 0) s_end = a.path_width;
  __syncthreads();
  for (int i0 = 0; i0 < a.path_width; i0 += 256) {
    const int i = i0 + tid;
    const bool ends = i < a.path_width && (path[i] >= n || path[i] <= (i ? path[i - 1] : -1));
    const unsigned long long hit = __ballot(ends);
    if (hit && lane == 0) atomicMin(&s_end, i + __builtin_ctzll(hit));
  }
  __syncthreads();
  const int count = s_end;
  if (a.new_lens && layer == 0 && head == 0 && tid == 0)
    a.new_lens[b] = static_cast<int>(max(0ll, min(base + count, 0x7fffffffll)));
  const long long cap = static_cast<long long>(a.c.width) << a.c.page_shift;
  const int groups = 256 / lpr, sub = tid & (lpr - 1), group = tid / lpr;
  const bool own = sub * 8 < a.c.d;
  for (int i0 = 0; i0 < count; i0 += groups * PAGE_AHEAD) {
    RowPair r[PAGE_AHEAD];
    float score[PAGE_AHEAD];
    int32_t pos[PAGE_AHEAD];
    long long to[PAGE_AHEAD], to_slot[PAGE_AHEAD];
#pragma unroll
    for (int u = 0; u < PAGE_AHEAD; ++u) {
      const int i = i0 + u * groups + group;
      to[u] = -1;
      if (i >= count) continue;
      const long long src = base + path[i], dst = base + i;
      if (src == dst || dst < 0 || src >= cap) continue;
      const int from = a.c.page_of(b, static_cast<int>(src)), page = a.c.page_of(b, static_cast<int>(dst));
      if (from < 0 || page < 0) continue;
      to[u] = a.c.row_at(page, head, static_cast<int>(dst));
      to_slot[u] = a.c.slot_at(page, head, static_cast<int>(dst));
      if (own) r[u] = load_rows(a.l, layer, a.c.row_at(from, head, static_cast<int>(src)), sub);
      const long long s = a.c.slot_at(from, head, static_cast<int>(src));
      if (sub == 0 && a.l.scores[layer]) score[u] = a.l.scores[layer][s];
      if (sub == 0 && a.l.pos[layer]) pos[u] = a.l.pos[layer][s];
    }
    // what the group's tokens leave is in registers before any of it is written over
    wait_vmcnt<0>();
    __syncthreads();
#pragma unroll
    for (int u = 0; u < PAGE_AHEAD; ++u) {
      if (to[u] < 0) continue;
      if (own) store_rows(a.l, layer, to[u], sub, r[u]);
      if (sub == 0 && a.l.scores[layer]) a.l.scores[layer][to_slot[u]] = score[u];
      if (sub == 0 && a.l.pos[layer]) a.l.pos[layer][to_slot[u]] = pos[u];
    }
  }
}

}  // namespace trellis
