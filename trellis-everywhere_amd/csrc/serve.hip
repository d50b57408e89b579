// serve.hip — C ABI of the operators between the packed linears (include/trellis_amd.h): validation,
// launch planning and the dispatch to norm.h, append.h, attend.h and evict.h.
#include <hip/hip_runtime.h>

#include <cstring>

#include "append.h"
#include "attend.h"
#include "evict.h"
#include "norm.h"
#include "serve_host.h"

using namespace trellis;

namespace {

// ---------------------------------------------------------------- residual norm

// The fewest chunks of 8 a thread that 1024 threads cover a row with, and those threads.
int norm_chunks(int width) { return width <= 8192 ? 1 : width <= 16384 ? 2 : 4; }
int norm_threads(int width) {
  const int per = 8 * norm_chunks(width);
  return ((width + per - 1) / per + 63) / 64 * 64;
}

template <class TX, class TR>
void launch_norm(const NormArgs& a, bool vec, int64_t rows, hipStream_t st) {
  const int chunks = norm_chunks(a.width), threads = norm_threads(a.width);
  const dim3 grid(static_cast<unsigned>(rows)), block(threads);
  if (chunks == 1) {
    if (vec) hipLaunchKernelGGL((norm_kernel<TX, TR, true, 1>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((norm_kernel<TX, TR, false, 1>), grid, block, 0, st, a);
  } else if (chunks == 2) {
    if (vec) hipLaunchKernelGGL((norm_kernel<TX, TR, true, 2>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((norm_kernel<TX, TR, false, 2>), grid, block, 0, st, a);
  } else {
    if (vec) hipLaunchKernelGGL((norm_kernel<TX, TR, true, 4>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((norm_kernel<TX, TR, false, 4>), grid, block, 0, st, a);
  }
}

template <class TX>
void launch_norm_r(const NormArgs& a, int r_dtype, bool vec, int64_t rows, hipStream_t st) {
  if (r_dtype == TRELLIS_F32) launch_norm<TX, float>(a, vec, rows, st);
  else if (r_dtype == TRELLIS_F16) launch_norm<TX, _Float16>(a, vec, rows, st);
  else launch_norm<TX, bf16_t>(a, vec, rows, st);
}

// ---------------------------------------------------------------- cache

template <class TX, class TC>
void launch_append(const AppendArgs& a, bool vec, bool nt, int lpr, int rounds, int parts, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.tokens * parts));
  if (!vec) hipLaunchKernelGGL((append_kernel<TX, TC, false, false>), grid, dim3(256), 0, st, a, lpr, rounds, parts);
  else if (nt) hipLaunchKernelGGL((append_kernel<TX, TC, true, true>), grid, dim3(256), 0, st, a, lpr, rounds, parts);
  else hipLaunchKernelGGL((append_kernel<TX, TC, true, false>), grid, dim3(256), 0, st, a, lpr, rounds, parts);
}

// ---------------------------------------------------------------- attention

struct AttendPlan : AttChunks {
  int64_t logit_stride;
  size_t off_ml, off_total, off_logits, ws;
};

AttendPlan attend_plan(const trellis_kv_cache* c, int q_heads, bool accumulate) {
  AttendPlan p;
  const int n = longest(c), group = q_heads / c->heads;
  static_cast<AttChunks&>(p) = att_chunks(c->rows, c->heads, q_heads, c->head_dim, n, device_cus());
  const size_t bh = static_cast<size_t>(c->rows) * q_heads;
  p.logit_stride = (static_cast<int64_t>(n) + 31) / 32 * 32;
  const size_t slots = p.aim ? static_cast<size_t>(p.items) * group : 0;
  p.off_ml = up256(slots * c->head_dim * 4);
  p.off_total = p.off_ml + up256(slots * 8);
  p.off_logits = p.off_total + (accumulate ? up256(bh * 8) : 0);
  p.ws = p.off_logits + (accumulate ? up256(bh * p.logit_stride * 4) : 0);
  return p;
}

// Nontemporal loads where a call of 16 MB and more reads whole 128-byte lines once: keys and values of some tens
// of layers of that size do not stay in the 256 MB last-level cache until their next use (36 layers in turn: 4000
// tokens of 8 heads of 128 11.4 -> 10.3 us, 16000 20.3 -> 19.1; one layer of 131072 101 -> 91 us, 64 rows of 8192
// 379 -> 344). Not below (32 rows up to 512 tokens of 3 heads of 64: 7.6 -> 8.2), for other head dims (96: 81 -> 92) or
// where a second workgroup reads the same lines (more than 16 query heads a head; 64 over 2: 42 -> 51).
bool attend_streams(const trellis_kv_cache* c, const AttendPlan& p) {
  const int64_t bytes = static_cast<int64_t>(c->rows) * longest(c) * c->heads * c->head_dim * 4;
  return bytes >= 16000000 && p.row_blocks == 1 && c->head_dim % 64 == 0;
}

template <class T, int DP, bool FULL, bool EXACT>
void launch_attend_nt(const AttendArgs& a, bool nt, unsigned grid, hipStream_t st) {
  const dim3 block(64 * ATT_WAVES);
  if constexpr (FULL) {
    if (nt) {
      hipLaunchKernelGGL((attend_kernel<T, DP, FULL, EXACT, true>), dim3(grid), block, 0, st, a);
      return;
    }
  }
  hipLaunchKernelGGL((attend_kernel<T, DP, FULL, EXACT, false>), dim3(grid), block, 0, st, a);
}

template <class T, int DP>
void launch_attend(const AttendArgs& a, bool exact, bool nt, unsigned grid, hipStream_t st) {
  if (a.c.d == DP) {
    if (exact) launch_attend_nt<T, DP, true, true>(a, nt, grid, st);
    else launch_attend_nt<T, DP, true, false>(a, nt, grid, st);
  } else {
    if (exact) launch_attend_nt<T, DP, false, true>(a, nt, grid, st);
    else launch_attend_nt<T, DP, false, false>(a, nt, grid, st);
  }
}

template <class T>
void launch_attend_d(const AttendArgs& a, bool exact, bool nt, unsigned grid, hipStream_t st) {
  if (a.c.d <= 64) launch_attend<T, 64>(a, exact, nt, grid, st);
  else if (a.c.d <= 128) launch_attend<T, 128>(a, exact, nt, grid, st);
  else launch_attend<T, 256>(a, exact, nt, grid, st);
}

int validate_attention(const trellis_kv_cache* c, int q_heads, int accumulate) {
  const int v = validate_cache(c);
  if (v) return v;
  if (q_heads < 1 || q_heads % c->heads) return TRELLIS_ERR_HEADS;
  if (accumulate && !c->scores) return TRELLIS_ERR_NULL;
  return TRELLIS_OK;
}

// ---------------------------------------------------------------- eviction

int validate_evict(const trellis_kv_cache* c, int keep, int recent) {
  const int v = validate_cache(c);
  if (v) return v;
  if (!c->scores || !c->pos) return TRELLIS_ERR_NULL;
  if (!aligned(c->scores, 16) || !aligned(c->pos, 16)) return TRELLIS_ERR_ALIGN;
  if (keep < 1 || recent < 0 || recent > keep) return TRELLIS_ERR_KEEP;
  return TRELLIS_OK;
}

template <int THREADS, int G, bool FUSED>
void launch_evict_g(const EvictArgs& a, int lpr, unsigned grid, hipStream_t st) {
  hipLaunchKernelGGL((evict_select_kernel<THREADS, G, FUSED>), dim3(grid), dim3(THREADS), 0, st, a, lpr);
}

// The smallest form whose registers hold the longest row (beyond 32768 tokens the last, in segments).
template <bool FUSED>
void launch_evict_ept(const EvictArgs& a, int n, int lpr, unsigned grid, hipStream_t st) {
  if (n <= 2048) launch_evict_g<512, 1, FUSED>(a, lpr, grid, st);
  else if (n <= 4096) launch_evict_g<1024, 1, FUSED>(a, lpr, grid, st);
  else if (n <= 16384) launch_evict_g<1024, 4, FUSED>(a, lpr, grid, st);
  else launch_evict_g<1024, 8, FUSED>(a, lpr, grid, st);
}

void launch_evict_select(const EvictArgs& a, int n, bool fused, int lpr, unsigned grid, hipStream_t st) {
  if (fused) launch_evict_ept<true>(a, n, lpr, grid, st);
  else launch_evict_ept<false>(a, n, lpr, grid, st);
}

struct EvictPlan {
  int list;       // the most tokens of a row and head that are kept
  int most;       // the most moves it can make
  bool fused;     // few enough for the select kernel: no lists in the workspace
  size_t off_first, off_second, ws;
};

EvictPlan evict_plan(const trellis_kv_cache* c, int keep, bool apart) {
  EvictPlan p;
  const int n = longest(c);
  p.list = keep < n ? keep : n;
  p.most = apart ? p.list : n - keep < keep ? n - keep : keep;
  p.fused = !apart && p.most <= EV_FUSED;
  const size_t bh = static_cast<size_t>(c->rows) * c->heads;
  p.off_first = up256(bh * 4);
  p.off_second = p.off_first + up256(bh * p.list * 4);
  p.ws = p.fused ? 0 : p.off_second + up256(bh * p.list * 4);
  return p;
}

}  // namespace

extern "C" {

int trellis_residual_norm(const void* x, int64_t ldx, int x_dtype, const void* residual, int64_t ldr,
                          int r_dtype, const void* gate, int64_t ldg, int gate_inner,
                          const float* post_weight, const float* weight, float scale, float eps, void* h,
                          int64_t ldh, void* y, int64_t ldy, int y_dtype, int64_t rows, int width,
                          void* stream) {
  if (rows < 0) return TRELLIS_ERR_BATCH;
  if (width < 1 || width > TRELLIS_NORM_MAX_WIDTH) return TRELLIS_ERR_WIDTH;
  if (!known_dtype(x_dtype) || !known_dtype(r_dtype) || !known_dtype(y_dtype)) return TRELLIS_ERR_DTYPE;
  if (rows == 0) return TRELLIS_OK;
  if (!x || !weight || !y) return TRELLIS_ERR_NULL;
  if (!grid_fits(rows, norm_threads(width))) return TRELLIS_ERR_BATCH;
  const int xs = dtype_size(x_dtype), rs = dtype_size(r_dtype), ys = dtype_size(y_dtype);
  if (!aligned(x, xs) || !aligned(y, ys) || (residual && !aligned(residual, rs)) || (h && !aligned(h, rs)) ||
      (gate && !aligned(gate, xs)) || !aligned(weight, 4) || (post_weight && !aligned(post_weight, 4)) ||
      (gate_inner != 0 && gate_inner != 1) || (rows > 1 && (ldy < width || (h && ldh < width))))
    return TRELLIS_ERR_ALIGN;
  // whole 16-byte accesses everywhere, or none
  const auto vec16 = [&](const void* p, int64_t ld, int size) { return !p || (aligned(p, 16) && (rows == 1 || ld * size % 16 == 0)); };
  const bool vec = width % 8 == 0 && vec16(x, ldx, xs) && vec16(residual, ldr, rs) && vec16(h, ldh, rs) &&
                   vec16(y, ldy, ys) && (gate_inner == 0 || vec16(gate, ldg, xs)) && vec16(weight, 0, 4) &&
                   vec16(post_weight, 0, 4);
  NormArgs a;
  a.x = x;
  a.residual = residual;
  a.gate = gate;
  a.post_w = post_weight;
  a.w = weight;
  a.h = h;
  a.y = y;
  a.ldx = ldx;
  a.ldr = ldr;
  a.ldg = ldg;
  a.ldh = ldh;
  a.ldy = ldy;
  a.width = width;
  a.gate_inner = gate_inner;
  a.y_dt = y_dtype;
  a.scale = scale;
  a.eps = eps;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (x_dtype == TRELLIS_F32) launch_norm_r<float>(a, r_dtype, vec, rows, st);
  else if (x_dtype == TRELLIS_F16) launch_norm_r<_Float16>(a, r_dtype, vec, rows, st);
  else launch_norm_r<bf16_t>(a, r_dtype, vec, rows, st);
  return launched();
}

int trellis_kv_append(const trellis_kv_cache* cache, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                      const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                      int64_t v_token_stride, int64_t v_head_stride, int x_dtype, int tokens, int q_heads,
                      const int32_t* starts, const int32_t* positions, const float* q_weight, const float* k_weight,
                      float eps, const float* cos, const float* sin, int rot, int n_positions, void* q_out,
                      int q_dtype, void* stream) {
  const int bad = validate_cache(cache);
  if (bad) return bad;
  if (!known_dtype(x_dtype) || !known_dtype(q_dtype)) return TRELLIS_ERR_DTYPE;
  if (q_heads < 1 || q_heads % cache->heads) return TRELLIS_ERR_HEADS;
  if (tokens < 0 || (!starts && tokens != cache->rows)) return TRELLIS_ERR_BATCH;
  if ((cos != nullptr) != (sin != nullptr) || (q_weight != nullptr) != (k_weight != nullptr)) return TRELLIS_ERR_NULL;
  if (cos && (rot < 16 || rot % 16 || rot > cache->head_dim)) return TRELLIS_ERR_HEADS;
  if (cos && n_positions < 1) return TRELLIS_ERR_RANGE;
  if (tokens == 0) return TRELLIS_OK;
  if (!q || !k || !v || !q_out) return TRELLIS_ERR_NULL;
  if (cache->rows < 1) return TRELLIS_ERR_BATCH;
  const int xs = dtype_size(x_dtype);
  if (!aligned(q, xs) || !aligned(k, xs) || !aligned(v, xs) || !aligned(q_out, 16) ||
      !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(cos, 16) || !aligned(sin, 16))
    return TRELLIS_ERR_ALIGN;
  AppendArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_t = q_token_stride;
  a.q_h = q_head_stride;
  a.k_t = k_token_stride;
  a.k_h = k_head_stride;
  a.v_t = v_token_stride;
  a.v_h = v_head_stride;
  a.q_out = q_out;
  a.q_w = q_weight;
  a.k_w = k_weight;
  a.cos = cos;
  a.sin = sin;
  a.starts = starts;
  a.positions = positions;
  a.tokens = tokens;
  a.hq = q_heads;
  a.q_dt = q_dtype;
  a.rot = rot;
  a.n_positions = n_positions;
  a.eps = eps;
  a.c = cache_of(cache);
  const int per = 16 / xs;
  const bool vec = aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && q_token_stride % per == 0 &&
                   q_head_stride % per == 0 && k_token_stride % per == 0 && k_head_stride % per == 0 &&
                   v_token_stride % per == 0 && v_head_stride % per == 0;
  const int lpr = lanes_per_row(cache->head_dim);
  // a workgroup per token; while those do not fill the CUs, the token's heads over several
  const int64_t heads = q_heads + 2 * static_cast<int64_t>(cache->heads), groups = 256 / lpr;
  const int64_t all = (heads + groups - 1) / groups;
  const int64_t parts = tokens * all <= 2 * device_cus() ? all : 1;
  if (!grid_fits(tokens * parts, 256)) return TRELLIS_ERR_BATCH;
  const int rounds = static_cast<int>((all + parts - 1) / parts);
  // prompts of 16 MB and more: what is written is not read again from the caches (6007 tokens of 48 heads of 128
  // 38.5 -> 30.5 us)
  const bool nt = tokens * heads * cache->head_dim * 2 >= 16000000;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool f16 = cache->dtype == TRELLIS_F16;
  if (x_dtype == TRELLIS_F32) {
    if (f16) launch_append<float, _Float16>(a, vec, nt, lpr, rounds, static_cast<int>(parts), st);
    else launch_append<float, bf16_t>(a, vec, nt, lpr, rounds, static_cast<int>(parts), st);
  } else if (x_dtype == TRELLIS_F16) {
    if (f16) launch_append<_Float16, _Float16>(a, vec, nt, lpr, rounds, static_cast<int>(parts), st);
    else launch_append<_Float16, bf16_t>(a, vec, nt, lpr, rounds, static_cast<int>(parts), st);
  } else {
    if (f16) launch_append<bf16_t, _Float16>(a, vec, nt, lpr, rounds, static_cast<int>(parts), st);
    else launch_append<bf16_t, bf16_t>(a, vec, nt, lpr, rounds, static_cast<int>(parts), st);
  }
  return launched();
}

int trellis_attention_workspace_bytes(const trellis_kv_cache* cache, int q_heads, int accumulate, size_t* bytes) {
  if (!bytes) return TRELLIS_ERR_NULL;
  const int v = validate_attention(cache, q_heads, accumulate);
  if (v) return v;
  *bytes = attend_plan(cache, q_heads, accumulate != 0).ws;
  return TRELLIS_OK;
}

int trellis_paged_attention(const trellis_kv_cache* cache, const void* q, int64_t q_row_stride, int64_t q_head_stride,
                            int q_dtype, int q_heads, float scale, int accumulate, void* out, int out_dtype,
                            void* workspace, size_t ws_bytes, void* stream) {
  const int v = validate_attention(cache, q_heads, accumulate);
  if (v) return v;
  if (!known_dtype(q_dtype) || !known_dtype(out_dtype)) return TRELLIS_ERR_DTYPE;
  if (cache->rows == 0) return TRELLIS_OK;
  if (!q || !out) return TRELLIS_ERR_NULL;
  const int qs = dtype_size(q_dtype);
  if (!aligned(q, qs) || !aligned(out, 16)) return TRELLIS_ERR_ALIGN;
  const AttendPlan p = attend_plan(cache, q_heads, accumulate != 0);
  if (p.ws && (!workspace || ws_bytes < p.ws)) return TRELLIS_ERR_WORKSPACE;
  if (p.ws && !aligned(workspace, 256)) return TRELLIS_ERR_ALIGN;
  char* ws = static_cast<char*>(workspace);
  AttendArgs a;
  a.q = q;
  a.q_b = q_row_stride;
  a.q_h = q_head_stride;
  a.q_dt = q_dtype;
  a.q_vec = aligned(q, 16) && q_row_stride * qs % 16 == 0 && q_head_stride * qs % 16 == 0;
  a.out = out;
  a.out_dt = out_dtype;
  a.hq = q_heads;
  a.group = q_heads / cache->heads;
  a.row_blocks = p.row_blocks;
  a.aim = p.aim;
  a.chunk = p.chunk;
  a.items = static_cast<int>(p.items);
  a.scale = scale * 1.44269504088896340736f;
  a.part = reinterpret_cast<float*>(ws);
  a.ml = reinterpret_cast<float*>(ws + p.off_ml);
  a.total = accumulate ? reinterpret_cast<float*>(ws + p.off_total) : nullptr;
  a.logits = accumulate ? reinterpret_cast<float*>(ws + p.off_logits) : nullptr;
  a.logit_stride = p.logit_stride;
  a.c = cache_of(cache);
  const int64_t one = static_cast<int64_t>(cache->rows) * cache->heads, bh = static_cast<int64_t>(cache->rows) * q_heads;
  const int64_t blocks = (p.items + 7) / 8 * 8 * p.row_blocks;
  const int64_t joins = p.aim ? bh : 0;
  const int64_t finish = joins + (accumulate ? one * ((longest(cache) + 255) / 256) : 0);
  // (chunks count the units of all rows and heads in 32 bits)
  if (!grid_fits(blocks, 64 * ATT_WAVES) || !grid_fits(finish, 256) ||
      one * ((longest(cache) + ATT_UNIT - 1) / ATT_UNIT) >= (int64_t(1) << 31))
    return TRELLIS_ERR_BATCH;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool exact = q_dtype != cache->dtype || out_dtype == TRELLIS_F32;
  const bool nt = attend_streams(cache, p);
  if (cache->dtype == TRELLIS_F16) launch_attend_d<_Float16>(a, exact, nt, static_cast<unsigned>(blocks), st);
  else launch_attend_d<bf16_t>(a, exact, nt, static_cast<unsigned>(blocks), st);
  if (finish > 0)
    hipLaunchKernelGGL(attend_finish_kernel, dim3(static_cast<unsigned>(finish)), dim3(256), 0, st, a, static_cast<int>(joins));
  return launched();
}

int trellis_evict_workspace_bytes(const trellis_kv_cache* cache, int keep, int apart, size_t* bytes) {
  if (!bytes) return TRELLIS_ERR_NULL;
  const int v = validate_evict(cache, keep, 0);
  if (v) return v;
  *bytes = evict_plan(cache, keep, apart != 0).ws;
  return TRELLIS_OK;
}

int trellis_kv_evict(const trellis_kv_cache* cache, int keep, int recent, const int32_t* next_pos,
                     const int32_t* out_table, int64_t out_table_stride, int out_width, int32_t* new_lens,
                     void* workspace, size_t ws_bytes, void* stream) {
  const int v = validate_evict(cache, keep, recent);
  if (v) return v;
  if (out_table && (out_width < 1 || out_table_stride < 0)) return TRELLIS_ERR_PAGE;
  if (cache->rows == 0) return TRELLIS_OK;
  if (!new_lens) return TRELLIS_ERR_NULL;
  if (new_lens == cache->lens) return TRELLIS_ERR_RANGE;
  const EvictPlan p = evict_plan(cache, keep, out_table != nullptr);
  if (p.ws && (!workspace || ws_bytes < p.ws)) return TRELLIS_ERR_WORKSPACE;
  if (p.ws && !aligned(workspace, 256)) return TRELLIS_ERR_ALIGN;
  char* ws = static_cast<char*>(workspace);
  EvictArgs a;
  a.c = cache_of(cache);
  a.next_pos = next_pos;
  a.out_table = out_table;
  a.out_stride = out_table_stride;
  a.out_width = out_width;
  a.keep = keep;
  a.recent = recent;
  a.new_lens = new_lens;
  a.list = p.list;
  a.count = reinterpret_cast<int32_t*>(ws);
  a.first = reinterpret_cast<int32_t*>(ws + p.off_first);
  a.second = reinterpret_cast<int32_t*>(ws + p.off_second);
  const int64_t bh = static_cast<int64_t>(cache->rows) * cache->heads;
  // the moves in groups of the rows one workgroup moves, up to 64 workgroups a row and head
  const int lpr = lanes_per_row(cache->head_dim);
  int blocks = p.most > 0 ? (p.most + 256 / lpr - 1) / (256 / lpr) : 0;
  if (blocks > 64) blocks = 64;
  if (!grid_fits(bh, 1024) || !grid_fits(bh * blocks, 256)) return TRELLIS_ERR_BATCH;
  hipStream_t st = static_cast<hipStream_t>(stream);
  launch_evict_select(a, longest(cache), p.fused, lpr, static_cast<unsigned>(bh), st);
  if (blocks > 0 && !p.fused)
    hipLaunchKernelGGL(evict_move_kernel, dim3(static_cast<unsigned>(bh * blocks)), dim3(256), 0, st, a, lpr, blocks);
  return launched();
}

}  // extern "C"
