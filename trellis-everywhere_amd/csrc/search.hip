// search.hip — C ABI of the operators that carry several hypotheses over a paged cache (include/trellis_amd.h):
// validation, launch planning and the dispatch to tree.h, beam.h and pages.h.
#include <hip/hip_runtime.h>

#include "beam.h"
#include "pages.h"
#include "serve_host.h"
#include "tree.h"
#include "tree_join.h"

using namespace trellis;

namespace {

// ---------------------------------------------------------------- attention of several new tokens

int validate_tree(const trellis_kv_cache* c, int q_heads, int tokens, int q_dtype, int out_dtype) {
  const int v = validate_cache(c);
  if (v) return v;
  if (q_heads < 1 || q_heads % c->heads) return TRELLIS_ERR_HEADS;
  if (!known_dtype(q_dtype) || !known_dtype(out_dtype)) return TRELLIS_ERR_DTYPE;
  if (tokens < 0 || (tokens > 0 && c->rows < 1)) return TRELLIS_ERR_BATCH;
  // (queries are counted in 32 bits)
  if (static_cast<int64_t>(tokens) * q_heads >= (int64_t(1) << 31)) return TRELLIS_ERR_BATCH;
  return TRELLIS_OK;
}

// Types that take the exact form: q or out of another type than the cache's.
bool tree_exact(const trellis_kv_cache* c, int q_dtype, int out_dtype) { return q_dtype != c->dtype || out_dtype != c->dtype; }

struct TreePlan : TreeChunks {
  int qr;
  size_t off_ml, off_done, ws;
};

TreePlan tree_plan(const trellis_kv_cache* c, int q_heads, int tokens, bool exact) {
  TreePlan p;
  static_cast<TreeChunks&>(p) = tree_chunks(c->rows, c->heads, q_heads, c->head_dim, tokens, longest(c), exact, device_cus());
  p.qr = 32 * tree_waves(exact);
  const size_t slots = p.aim ? static_cast<size_t>(p.items) * p.qr : 0;
  p.off_ml = up256(slots * c->head_dim * 4);
  p.off_done = p.off_ml + up256(slots * 8);
  p.ws = p.off_done + (p.aim ? up256((static_cast<size_t>(p.blocks) / c->heads + 1) * sizeof(TreeBlock)) : 0);
  return p;
}

// ---------------------------------------------------------------- beams

int validate_beam(int batch, int beams, int vocab, int k) {
  if (batch < 0) return TRELLIS_ERR_BATCH;
  if (beams < 1 || beams > BEAM_MOST || k < 1 || k > BEAM_MOST || vocab < 1) return TRELLIS_ERR_BEAMS;
  return TRELLIS_OK;
}

struct BeamPlan {
  int rounds;         // of 512 logits a wave holds: 2, 4, 8 or 16
  int runs, per;      // waves a beam, pieces of 8 logits of each
  size_t off_best, ws;
};

// The longest runs that leave waves enough, 8 a CU, for the logits to be on their way; a beam has up to 64, each of
// several rounds then.
BeamPlan beam_plan(int batch, int beams, int vocab, int k) {
  const int64_t rows = static_cast<int64_t>(batch) * beams, pieces = (static_cast<int64_t>(vocab) + 7) / 8;
  // (a workgroup's four waves share a beam)
  const auto runs = [&](int rounds) { return (pieces + 256 * rounds - 1) / (256 * rounds) * 4; };
  BeamPlan p;
  p.rounds = 16;
  while (p.rounds > 2 && rows * runs(p.rounds) < 8 * device_cus() && runs(p.rounds / 2) <= BEAM_MOST) p.rounds /= 2;
  p.runs = static_cast<int>(runs(p.rounds) < BEAM_MOST ? runs(p.rounds) : BEAM_MOST);
  p.per = static_cast<int>((pieces + p.runs - 1) / p.runs);
  p.off_best = up256(static_cast<size_t>(rows) * p.runs * 16);
  p.ws = p.off_best + up256(static_cast<size_t>(rows) * (p.runs / 4) * k * 8);
  return p;
}

template <class T>
void launch_beam_part(const BeamArgs& a, int rounds, unsigned grid, hipStream_t st) {
  const dim3 block(256);
  if (rounds == 2) hipLaunchKernelGGL((beam_part_kernel<T, 2>), dim3(grid), block, 0, st, a);
  else if (rounds == 4) hipLaunchKernelGGL((beam_part_kernel<T, 4>), dim3(grid), block, 0, st, a);
  else if (rounds == 8) hipLaunchKernelGGL((beam_part_kernel<T, 8>), dim3(grid), block, 0, st, a);
  else hipLaunchKernelGGL((beam_part_kernel<T, 16>), dim3(grid), block, 0, st, a);
}

// ---------------------------------------------------------------- pages

// Layers of one pool geometry; the pointers of `count` of them.
int validate_layers(const trellis_kv_cache* c, int layers) {
  if (layers < 1) return TRELLIS_ERR_LAYERS;
  if (!c) return TRELLIS_ERR_NULL;
  for (int i = 0; i < layers; ++i) {
    const int v = validate_cache(c + i);
    if (v) return v;
    if (c[i].page_stride != c->page_stride || c[i].head_stride != c->head_stride || c[i].slot_stride != c->slot_stride ||
        c[i].pages != c->pages || c[i].heads != c->heads || c[i].page_size != c->page_size || c[i].head_dim != c->head_dim ||
        c[i].dtype != c->dtype)
      return TRELLIS_ERR_LAYERS;
    if (!aligned(c[i].scores, 4) || !aligned(c[i].pos, 4)) return TRELLIS_ERR_ALIGN;
  }
  return TRELLIS_OK;
}

Layers layers_of(const trellis_kv_cache* c, int count) {
  Layers l = {};
  for (int i = 0; i < count; ++i) {
    l.k[i] = c[i].k;
    l.v[i] = c[i].v;
    l.scores[i] = c[i].scores;
    l.pos[i] = c[i].pos;
  }
  return l;
}

}  // namespace

extern "C" {

int trellis_tree_attention_workspace_bytes(const trellis_kv_cache* cache, int tokens, int q_heads, int q_dtype, int out_dtype,
                                           size_t* bytes) {
  if (!bytes) return TRELLIS_ERR_NULL;
  const int v = validate_tree(cache, q_heads, tokens, q_dtype, out_dtype);
  if (v) return v;
  *bytes = tree_plan(cache, q_heads, tokens, tree_exact(cache, q_dtype, out_dtype)).ws;
  return TRELLIS_OK;
}

int trellis_tree_attention(const trellis_kv_cache* cache, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                           int q_dtype, int tokens, int q_heads, const int32_t* starts, const int32_t* parents, float scale,
                           void* out, int out_dtype, void* workspace, size_t ws_bytes, void* stream) {
  const int v = validate_tree(cache, q_heads, tokens, q_dtype, out_dtype);
  if (v) return v;
  if (!starts && cache->rows > 0 && tokens % cache->rows) return TRELLIS_ERR_BATCH;
  if (tokens == 0) return TRELLIS_OK;
  if (!q || !out) return TRELLIS_ERR_NULL;
  const int qs = dtype_size(q_dtype);
  if (!aligned(q, qs) || !aligned(out, 16)) return TRELLIS_ERR_ALIGN;
  const bool exact = tree_exact(cache, q_dtype, out_dtype);
  const TreePlan p = tree_plan(cache, q_heads, tokens, exact);
  if (p.ws && (!workspace || ws_bytes < p.ws)) return TRELLIS_ERR_WORKSPACE;
  if (p.ws && !aligned(workspace, 256)) return TRELLIS_ERR_ALIGN;
  char* ws = static_cast<char*>(workspace);
  TreeLaunch l;
  TreeArgs& a = l.a;
  a.q = q;
  a.q_t = q_token_stride;
  a.q_h = q_head_stride;
  a.q_dt = q_dtype;
  a.q_vec = aligned(q, 16) && q_token_stride * qs % 16 == 0 && q_head_stride * qs % 16 == 0;
  a.out_dt = out_dtype;
  a.tokens = tokens;
  a.hq = q_heads;
  a.group = q_heads / cache->heads;
  a.starts = starts;
  a.each = starts ? 0 : tokens / cache->rows;
  a.parents = parents;
  a.out = out;
  a.aim = p.aim;
  a.items = static_cast<int>(p.items);
  a.scale = scale * 1.44269504088896340736f;
  a.part = reinterpret_cast<float*>(ws);
  a.ml = reinterpret_cast<float*>(ws + p.off_ml);
  a.done = reinterpret_cast<TreeBlock*>(ws + p.off_done);
  a.c = cache_of(cache);
  // the chunks, then those that see to tokens of no row
  const int64_t blocks = p.items + (starts ? (static_cast<int64_t>(tokens) + 63) / 64 : 0);
  // (a block has about its share of the chunks)
  const int64_t parts = p.aim ? p.items / p.blocks : 1;
  const int shares = parts >= 16 && cache->head_dim <= 128 ? 4 : parts >= 8 ? 2 : 1;
  const int rows = tree_join_rows(cache->head_dim, shares), subs = (p.qr + rows - 1) / rows;
  const int64_t joins = p.aim ? p.blocks * subs : 0;
  // (chunks count the units of all blocks in 32 bits)
  if (!grid_fits(blocks, 256) || !grid_fits(joins, 256) ||
      (p.aim && p.blocks * tree_units(longest(cache)) >= (int64_t(1) << 31)))
    return TRELLIS_ERR_BATCH;
  l.exact = exact;
  l.grid = static_cast<unsigned>(blocks);
  l.stream = static_cast<hipStream_t>(stream);
  if (cache->dtype == TRELLIS_F16) launch_tree_f16(l);
  else launch_tree_bf16(l);
  if (joins > 0) hipLaunchKernelGGL(tree_join_kernel, dim3(static_cast<unsigned>(joins)), dim3(256), 0, l.stream, a, p.qr, subs, shares);
  return launched();
}

int trellis_beam_workspace_bytes(int batch, int beams, int vocab, int k, size_t* bytes) {
  if (!bytes) return TRELLIS_ERR_NULL;
  const int v = validate_beam(batch, beams, vocab, k);
  if (v) return v;
  *bytes = beam_plan(batch, beams, vocab, k).ws;
  return TRELLIS_OK;
}

int trellis_beam_select(const void* logits, int64_t batch_stride, int64_t beam_stride, int dtype, int batch, int beams,
                        int vocab, const float* scores, const uint8_t* ended, int end_token, int k, float* new_scores,
                        int32_t* new_beams, int32_t* new_tokens, void* workspace, size_t ws_bytes, void* stream) {
  const int v = validate_beam(batch, beams, vocab, k);
  if (v) return v;
  if (!known_dtype(dtype)) return TRELLIS_ERR_DTYPE;
  if (end_token < 0 || end_token >= vocab) return TRELLIS_ERR_RANGE;
  if (batch == 0) return TRELLIS_OK;
  if (!logits || !scores || !new_scores || !new_beams || !new_tokens) return TRELLIS_ERR_NULL;
  if (!aligned(logits, dtype_size(dtype)) || !aligned(scores, 4) || !aligned(new_scores, 4) || !aligned(new_beams, 4) ||
      !aligned(new_tokens, 4))
    return TRELLIS_ERR_ALIGN;
  const BeamPlan p = beam_plan(batch, beams, vocab, k);
  if (!workspace || ws_bytes < p.ws) return TRELLIS_ERR_WORKSPACE;
  if (!aligned(workspace, 256)) return TRELLIS_ERR_ALIGN;
  const int64_t blocks = static_cast<int64_t>(batch) * beams * (p.runs / 4);
  if (!grid_fits(blocks, 256) || static_cast<int64_t>(batch) * beams > INT32_MAX) return TRELLIS_ERR_BATCH;
  BeamArgs a;
  a.x = logits;
  a.x_b = batch_stride;
  a.x_j = beam_stride;
  a.batch = batch;
  a.beams = beams;
  a.vocab = vocab;
  a.k = k;
  a.end_token = end_token;
  a.scores = scores;
  a.ended = ended;
  a.out_scores = new_scores;
  a.out_beams = new_beams;
  a.out_tokens = new_tokens;
  char* ws = static_cast<char*>(workspace);
  a.runs = p.runs;
  a.per = p.per;
  a.sums = reinterpret_cast<double*>(ws);
  a.best = reinterpret_cast<unsigned long long*>(ws + p.off_best);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(blocks);
  if (dtype == TRELLIS_F32) launch_beam_part<float>(a, p.rounds, grid, st);
  else if (dtype == TRELLIS_F16) launch_beam_part<_Float16>(a, p.rounds, grid, st);
  else launch_beam_part<bf16_t>(a, p.rounds, grid, st);
  hipLaunchKernelGGL(beam_join_kernel, dim3(batch), dim3(64 * (beams < 16 ? beams : 16)), 0, st, a);
  return launched();
}

int trellis_kv_copy_pages(const trellis_kv_cache* layers, int n_layers, const int32_t* src, const int32_t* dst,
                          const int32_t* counts, int n, void* stream) {
  const int v = validate_layers(layers, n_layers);
  if (v) return v;
  if (n < 0) return TRELLIS_ERR_BATCH;
  if (n == 0) return TRELLIS_OK;
  if (!src || !dst) return TRELLIS_ERR_NULL;
  CopyArgs a;
  a.c = cache_of(layers);
  a.src = src;
  a.dst = dst;
  a.counts = counts;
  a.n = n;
  const int lpr = lanes_per_row(layers->head_dim), rows = 256 / lpr * PAGE_AHEAD, parts = (layers->page_size + rows - 1) / rows;
  const int64_t one = static_cast<int64_t>(n) * layers->heads * parts;
  const int most = n_layers < PAGE_LAYERS ? n_layers : PAGE_LAYERS;
  if (one > INT32_MAX || !grid_fits(one * most, 256)) return TRELLIS_ERR_BATCH;
  // From 16 MB on a copy of what no cache holds is faster so (plain / nontemporal: 16 MB 9.8 / 8.7 us, 31 16.9 / 13.3, 63
  // 28.2 / 25.6, 126 51.6 / 47.0, 252 100.7 / 95.8; 9 MB 8.2 / 8.1). What is read again at once then comes from memory: with
  // a gather of the keys right behind, 16 MB 21.1 / 22.0, 31 35.6 / 35.3, 63 59.0 / 69.8, 126 112 / 132, 252 261 / 262.
  const bool nt = static_cast<int64_t>(n) * n_layers * layers->heads * layers->page_size * layers->head_dim * 4 >= 16000000;
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (int at = 0; at < n_layers; at += PAGE_LAYERS) {
    const int some = n_layers - at < PAGE_LAYERS ? n_layers - at : PAGE_LAYERS;
    a.l = layers_of(layers + at, some);
    const dim3 grid(static_cast<unsigned>(one * some));
    if (nt) hipLaunchKernelGGL(copy_pages_kernel<true>, grid, dim3(256), 0, st, a, lpr, parts);
    else hipLaunchKernelGGL(copy_pages_kernel<false>, grid, dim3(256), 0, st, a, lpr, parts);
  }
  return launched();
}

int trellis_kv_keep(const trellis_kv_cache* layers, int n_layers, const int32_t* starts, const int32_t* path,
                    int64_t path_stride, int path_width, int32_t* new_lens, void* stream) {
  const int v = validate_layers(layers, n_layers);
  if (v) return v;
  if (path_width < 0 || path_stride < 0) return TRELLIS_ERR_RANGE;
  if (layers->rows == 0) return TRELLIS_OK;
  if (!starts || (path_width > 0 && !path) || !new_lens) return TRELLIS_ERR_NULL;
  if (new_lens == layers->lens) return TRELLIS_ERR_RANGE;
  KeepArgs a;
  a.c = cache_of(layers);
  a.starts = starts;
  a.path = path;
  a.path_stride = path_stride;
  a.path_width = path_width;
  const int lpr = lanes_per_row(layers->head_dim);
  const int64_t one = static_cast<int64_t>(layers->rows) * layers->heads;
  const int most = n_layers < PAGE_LAYERS ? n_layers : PAGE_LAYERS;
  if (!grid_fits(one * most, 256)) return TRELLIS_ERR_BATCH;
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (int at = 0; at < n_layers; at += PAGE_LAYERS) {
    const int some = n_layers - at < PAGE_LAYERS ? n_layers - at : PAGE_LAYERS;
    a.l = layers_of(layers + at, some);
    a.new_lens = at == 0 ? new_lens : nullptr;
    hipLaunchKernelGGL(keep_kernel, dim3(static_cast<unsigned>(one * some)), dim3(256), 0, st, a, lpr);
  }
  return launched();
}

}  // extern "C"
