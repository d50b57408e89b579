// evict.h — eviction from a paged cache by accumulated attention weight. Per row b and key-value head, of
// the n = length tokens (n > keep):
//   kept: those with pos >= next_pos - recent, then the largest scores, `keep` in all; equal scores by
//         the lowest slot (a NaN score counts as the largest);
//   moved: a kept token below slot `keep` stays in its slot, and the slots that are not kept (holes) take
//         the kept tokens from above `keep`, both in ascending order. Sources and holes are disjoint, so
//         the moves of one head have no order among them.
// In place only the moves are made; with an out table every kept token goes to its slot there.
//
// evict_select_kernel, one workgroup per (row, head): the keep-th largest key by 8-bit digits of the keys'
// range (LDS histograms), then one pass in slot order that ranks holes and sources by ballots.
// evict_move_kernel copies.
#pragma once

#include "serve.h"

namespace trellis {

constexpr int EV_THREADS = 1024;
constexpr int EV_WAVES = EV_THREADS / 64;
constexpr uint32_t EV_RECENT = 0xFFFFFFFFu;   // key of a token kept for its position

struct EvictArgs {
  Cache c;
  const int32_t* next_pos;    // [rows], or null: the lengths
  const int32_t* out_table;   // or null: in place
  long long out_stride;
  int out_width;
  int keep, recent;
  int32_t* new_lens;          // [rows]
  int32_t* count;             // workspace: [rows][heads] list lengths
  int32_t* first;             // workspace: [rows][heads][keep]
  int32_t* second;            // workspace: [rows][heads][keep]
};
// In place, entry r of the lists is the move second[r] -> first[r]. With an out table, entry j of `first` is
// the source of slot j, or -1 - r: second[r].

// Order-preserving: a larger score has a larger key; NaN above infinity, below EV_RECENT.
__device__ __forceinline__ uint32_t ev_key(float score) {
  if (score != score) return EV_RECENT - 1;
  const uint32_t u = __builtin_bit_cast(uint32_t, score + 0.0f);   // -0 counts as 0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t ev_token_key(const EvictArgs& a, int b, int head, int j, int from) {
  const int page = a.c.page_of(b, j);
  if (page < 0) return 0;
  const long long p = a.c.slot_at(page, head, j);
  return a.c.pos[p] >= from ? EV_RECENT : ev_key(a.c.scores[p]);
}

// Exclusive rank of `flag` over the workgroup in thread order, and the total.
__device__ __forceinline__ int block_rank(bool flag, int* totals, int& total) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const unsigned long long vote = __ballot(flag);
  if (lane == 0) totals[wave] = __popcll(vote);
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < EV_WAVES; ++w) {
    const int t = totals[w];
    before += w < wave ? t : 0;
    total += t;
  }
  __syncthreads();
  return before + __popcll(vote & ((1ull << lane) - 1));
}

__global__ __launch_bounds__(EV_THREADS) void evict_select_kernel(EvictArgs a) {
  __shared__ int hist[256], totals[EV_WAVES], s_digit, s_left;
  const int tid = threadIdx.x;
  const int head = blockIdx.x % a.c.heads, b = blockIdx.x / a.c.heads;
  const int n = a.c.length(b);
  const long long bh = blockIdx.x;
  if (tid == 0 && head == 0) a.new_lens[b] = min(n, a.keep);
  int32_t* first = a.first + bh * a.keep;
  int32_t* second = a.second + bh * a.keep;
  if (n <= a.keep) {
    // everything stays: nothing moves in place, all slots are copied to an out table
    if (a.out_table)
      for (int j = tid; j < n; j += EV_THREADS) first[j] = j;
    if (tid == 0) a.count[bh] = a.out_table ? n : 0;
    return;
  }
  const int next = a.next_pos ? a.next_pos[b] : n;
  const int from = next - a.recent;

  // ---- the key of the keep-th largest, digit by digit, and how many of its equals are kept
  uint32_t prefix = 0;
  int left = a.keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += EV_THREADS) {
      const uint32_t key = ev_token_key(a, b, head, j, from);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int digit = 255, rest = left;
      while (digit > 0 && hist[digit] < rest) rest -= hist[digit--];
      s_digit = digit;
      s_left = rest;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(s_digit) << shift;
    left = s_left;
    __syncthreads();
  }

  // ---- in slot order: what is kept, the holes below `keep`, the sources above
  int equals = 0, holes = 0, sources = 0;
  for (int j0 = 0; j0 < n; j0 += EV_THREADS) {
    const int j = j0 + tid;
    const uint32_t key = j < n ? ev_token_key(a, b, head, j, from) : 0;
    int total;
    const bool equal = j < n && key == prefix;
    const int er = equals + block_rank(equal, totals, total);
    equals += total;
    const bool kept = j < n && (key > prefix || (equal && er < left));
    const bool hole = j < a.keep && !kept;
    const int hr = holes + block_rank(hole, totals, total);
    holes += total;
    const bool source = j >= a.keep && kept;
    const int sr = sources + block_rank(source, totals, total);
    sources += total;
    if (source) second[sr] = j;
    if (a.out_table) {
      if (j < a.keep) first[j] = kept ? j : -1 - hr;
    } else if (hole) {
      first[hr] = j;
    }
  }
  if (tid == 0) a.count[bh] = a.out_table ? a.keep : holes;
}

// One move per group of lpr lanes (16 bytes of k and v a lane).
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a, int lpr, int blocks) {
  const long long bh = blockIdx.x / blocks;
  const int head = bh % a.c.heads, b = bh / a.c.heads;
  const int per = 256 / lpr, sub = threadIdx.x & (lpr - 1);
  const int count = a.count[bh];
  const int32_t* first = a.first + bh * a.keep;
  const int32_t* second = a.second + bh * a.keep;
  for (int r = (blockIdx.x % blocks) * per + threadIdx.x / lpr; r < count; r += blocks * per) {
    int src, dst, to;
    if (a.out_table) {
      dst = r;
      src = first[r];
      if (src < 0) src = second[-1 - src];
      to = (dst >> a.c.page_shift) < a.out_width ? a.out_table[b * a.out_stride + (dst >> a.c.page_shift)] : -1;
      if (static_cast<unsigned>(to) >= static_cast<unsigned>(a.c.pages)) to = -1;
    } else {
      dst = first[r];
      src = second[r];
      to = a.c.page_of(b, dst);
    }
    const int page = a.c.page_of(b, src);
    if (page < 0 || to < 0) continue;
    const long long s = a.c.row_at(page, head, src), t = a.c.row_at(to, head, dst);
    if (sub * 8 < a.c.d) {
      const u32x4_t k = *reinterpret_cast<const u32x4_t*>(static_cast<const char*>(a.c.k) + 2 * s + 16 * sub);
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(static_cast<const char*>(a.c.v) + 2 * s + 16 * sub);
      *reinterpret_cast<u32x4_t*>(static_cast<char*>(a.c.k) + 2 * t + 16 * sub) = k;
      *reinterpret_cast<u32x4_t*>(static_cast<char*>(a.c.v) + 2 * t + 16 * sub) = v;
    }
    if (sub == 0) {
      const long long p = a.c.slot_at(page, head, src), q = a.c.slot_at(to, head, dst);
      a.c.scores[q] = a.c.scores[p];
      a.c.pos[q] = a.c.pos[p];
    }
  }
}

}  // namespace trellis
