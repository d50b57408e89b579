// serve_host.h — what the C entry points of the operators between the packed linears share on the host: checks of
// arguments, a call's cache as its kernels see it, grid limits.
#pragma once

#include <hip/hip_runtime.h>

#include "serve.h"
#include "trellis_amd.h"

namespace trellis {

inline bool known_dtype(int dt) { return dt == TRELLIS_F32 || dt == TRELLIS_F16 || dt == TRELLIS_BF16; }
inline int dtype_size(int dt) { return dt == TRELLIS_F32 ? 4 : 2; }
inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline int launched() { return hipGetLastError() == hipSuccess ? TRELLIS_OK : TRELLIS_ERR_LAUNCH; }
inline int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

// Workgroups of a launch: HIP counts threads in 32 bits per dimension.
inline bool grid_fits(int64_t blocks, int threads) { return blocks * threads < (int64_t(1) << 32) && blocks < (int64_t(1) << 31); }

inline int device_cus() {
  static const int cus = [] {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1)
      return 256;
    return n;
  }();
  return cus;
}

inline size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

// The tokens of a row that a call can see.
inline int longest(const trellis_kv_cache* c) {
  const int64_t cap = static_cast<int64_t>(c->width) * c->page_size;
  return static_cast<int>(c->max_len < cap ? c->max_len : cap);
}

inline int validate_cache(const trellis_kv_cache* c) {
  if (!c || !c->k || !c->v || (c->rows != 0 && (!c->table || !c->lens))) return TRELLIS_ERR_NULL;
  if (c->dtype != TRELLIS_F16 && c->dtype != TRELLIS_BF16) return TRELLIS_ERR_DTYPE;
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8 || c->heads < 1) return TRELLIS_ERR_HEADS;
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)) || c->pages < 1 || c->width < 1)
    return TRELLIS_ERR_PAGE;
  if (c->rows < 0 || c->max_len < 0) return TRELLIS_ERR_BATCH;
  // 16-byte rows, and byte offsets within a page that fit 32 bits
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->page_stride % 8 || c->head_stride % 8 || c->slot_stride % 8 ||
      c->page_stride < 0 || c->head_stride < 0 || c->slot_stride < c->head_dim ||
      c->slot_stride >= (int64_t(1) << 30) / c->page_size || c->table_stride < 0)
    return TRELLIS_ERR_ALIGN;
  // token numbers, and one tile or segment past the last, stay within 32 bits
  if (longest(c) > (1 << 30)) return TRELLIS_ERR_RANGE;
  return TRELLIS_OK;
}

inline Cache cache_of(const trellis_kv_cache* c) {
  Cache r;
  r.k = c->k;
  r.v = c->v;
  r.scores = c->scores;
  r.pos = c->pos;
  r.table = c->table;
  r.lens = c->lens;
  r.page_stride = c->page_stride;
  r.head_stride = c->head_stride;
  r.slot_stride = c->slot_stride;
  r.table_stride = c->table_stride;
  r.pages = c->pages;
  r.heads = c->heads;
  r.page_shift = log2_of(c->page_size);
  r.d = c->head_dim;
  r.rows = c->rows;
  r.width = c->width;
  r.max_len = c->max_len;
  return r;
}

inline int lanes_per_row(int d) { return 1 << log2_of((d + 7) / 8); }

}  // namespace trellis
