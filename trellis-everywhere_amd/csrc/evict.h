// evict.h — eviction from a paged cache by accumulated attention weight. Per row b and key-value head, of
// the n = length tokens, with `top` slots below which the kept ones end up:
//   kept: those with pos >= next_pos - recent, then the largest scores, `top` in all; equal scores by
//         the lowest slot (a NaN score counts as the largest);
//   moved: a kept token below slot `top` stays in its slot, and the slots that are not kept (holes) take
//         the kept tokens from above `top`, both in ascending order. Sources and holes are disjoint, so
//         the moves of one head have no order among them.
// In place only the moves are made, and top = keep (rows of up to keep tokens stay); with an out table every kept
// token goes to its slot there, and top = min(keep, n, the table's slots).
// A token on a page that does not exist is none: in place its slot is no hole, and as many tokens are kept as there
// are slots below top; with an out table n counts the others alone, which close up.
//
// evict_select_kernel, one workgroup per (row, head): the smallest kept key by 11-bit digits of the keys'
// range (LDS histograms), then one scan in slot order over the holes below `top` and the kept tokens above it, which
// numbers both: holes first, so a source's rank less their count is the hole that it fills.
// evict_move_kernel copies; a call whose rows can move EV_FUSED tokens at most copies in the first kernel.
// Bound: the first kernel by its chain of dependent steps, the second by memory. 16 rows of 8 heads of 1025 tokens
// 8.5 us (loads 1.6, three digits of 1.1 each, ranks 1.2, the move 0.8-1.1), with an out table 4 of up to 16000 14.5
// (loads 3.4, a digit of all keys 2.3, of few 1.5, ranks 3.5) and the copies 8.7 (34 MB, 3.9 TB/s); in place 4 of 16000
// cut to 2048 17.5 and 11.6. A row of 32000, with 32 keys a thread, 28.0 and 6.3; of 100000, read again in segments for
// each step, 122 and 9.5. With 8-bit digits found by one thread and every step's keys read again the first two took 47.8
// and 92.7.
#pragma once

#include "serve.h"

namespace trellis {

constexpr uint32_t EV_RECENT = 0xFFFFFFFFu;   // key of a token kept for its position

struct EvictArgs {
  Cache c;
  const int32_t* next_pos;    // [rows], or null: the lengths
  const int32_t* out_table;   // or null: in place
  long long out_stride;
  int out_width;
  int keep, recent;
  int32_t* new_lens;          // [rows]
  int list;                   // entries of a row and head's lists: min(keep, longest row)
  int32_t* count;             // workspace: [rows][heads] list lengths
  int32_t* first;             // workspace: [rows][heads][list]
  int32_t* second;            // workspace: [rows][heads][list]
};
// In place, entry r of the lists is the move second[r] -> first[r]. With an out table, entry j of `first` is
// the source of slot j, or -1 - r: second[r].

// Order-preserving: a larger score has a larger key; NaN above infinity, below EV_RECENT.
__device__ __forceinline__ uint32_t ev_key(float score) {
  if (score != score) return EV_RECENT - 1;
  const uint32_t u = __builtin_bit_cast(uint32_t, score + 0.0f);   // -0 counts as 0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ void ev_move(const EvictArgs& a, int b, int head, int from, int from_page, int to, int to_page,
                                        int sub) {
  if (from_page < 0 || to_page < 0) return;
  const long long s = a.c.row_at(from_page, head, from), t = a.c.row_at(to_page, head, to);
  if (sub * 8 < a.c.d) {
    const u32x4_t k = *reinterpret_cast<const u32x4_t*>(static_cast<const char*>(a.c.k) + 2 * s + 16 * sub);
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(static_cast<const char*>(a.c.v) + 2 * s + 16 * sub);
    *reinterpret_cast<u32x4_t*>(static_cast<char*>(a.c.k) + 2 * t + 16 * sub) = k;
    *reinterpret_cast<u32x4_t*>(static_cast<char*>(a.c.v) + 2 * t + 16 * sub) = v;
  }
  if (sub == 0) {
    const long long p = a.c.slot_at(from_page, head, from), q = a.c.slot_at(to_page, head, to);
    a.c.scores[q] = a.c.scores[p];
    a.c.pos[q] = a.c.pos[p];
  }
}

constexpr int EV_BINS = 2048;
constexpr int EV_FUSED = 64;    // most moves of a row and head that the select kernel makes itself

// A thread's keys stay in registers: G groups of 4 consecutive tokens (a page id, 16 bytes of positions and of
// scores each), group i of a thread at token segment + 4 (i * THREADS + tid). Rows longer than a segment of
// 4 G THREADS tokens go through in segments, read again for each step.
template <int THREADS, int G, bool FUSED>
__global__ __launch_bounds__(THREADS) void evict_select_kernel(EvictArgs a, int lpr) {
  constexpr int WAVES = THREADS / 64, SEG = 4 * G * THREADS;
  constexpr int BPT = EV_BINS / THREADS;
  __shared__ int hist[2][EV_BINS], totals[WAVES], counts[2][G * WAVES];
  __shared__ int s_digit, s_left, s_equals, s_first[EV_FUSED], s_second[EV_FUSED];
  __shared__ uint32_t s_lo[WAVES], s_hi[WAVES];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int head = blockIdx.x % a.c.heads, b = blockIdx.x / a.c.heads;
  const bool apart = !FUSED && a.out_table;
  const int n = a.c.length(b);
  const int keep = apart ? min(static_cast<long long>(a.keep), static_cast<long long>(a.out_width) << a.c.page_shift) : a.keep;
  const long long bh = blockIdx.x;
  int32_t* first = a.first + bh * a.list;
  int32_t* second = a.second + bh * a.list;
  const auto finish = [&](int len, int moves) {
    if (tid != 0) return;
    if (head == 0) a.new_lens[b] = len;
    if constexpr (!FUSED) a.count[bh] = moves;
  };
  if (n <= keep) {
    // everything stays: nothing moves in place, all slots are copied to an out table (if all exist)
    bool gap = false;
    if (apart) {
      for (int j = tid << a.c.page_shift; j < n; j += THREADS << a.c.page_shift) gap |= a.c.page_of(b, j) < 0;
      gap = __syncthreads_or(gap);
    }
    if (!gap) {
      if (apart)
        for (int j = tid; j < n; j += THREADS) first[j] = j;
      return finish(n, apart ? n : 0);
    }
  }
  const int from = (a.next_pos ? a.next_pos[b] : n) - a.recent;
  const int segs = (n + SEG - 1) / SEG;

  // the segment's keys: loads without branches (of the row's last group past its end, of page 0 for a missing
  // page), so that a step's are all in flight together
  uint32_t key[G][4];
  const auto token = [&](int seg, int i) { return seg * SEG + 4 * (i * THREADS + tid); };
  const auto load = [&](int seg) {
    int page[G];
    u32x4_t at[G];
#pragma unroll
    for (int i = 0; i < G; ++i) page[i] = a.c.page_of(b, min(token(seg, i), (n - 1) & ~3));
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const long long p = a.c.slot_at(max(page[i], 0), head, min(token(seg, i), (n - 1) & ~3));
      at[i] = *reinterpret_cast<const u32x4_t*>(a.c.pos + p);
      const u32x4_t s = *reinterpret_cast<const u32x4_t*>(a.c.scores + p);
#pragma unroll
      for (int q = 0; q < 4; ++q) key[i][q] = s[q];
    }
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        key[i][q] = page[i] < 0 ? 0u : static_cast<int>(at[i][q]) >= from ? EV_RECENT : ev_key(__builtin_bit_cast(float, key[i][q]));
  };
  // f(number among the thread's keys, token, key) for every token of the segment
  const auto each = [&](int seg, auto f) {
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (token(seg, i) + q < n) f(4 * i + q, token(seg, i) + q, key[i][q]);
  };

  // ---- the keys' range
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
  for (int seg = 0; seg < segs; ++seg) {
    load(seg);
    each(seg, [&](int, int, uint32_t k) {
      lo = min(lo, k);
      hi = max(hi, k);
    });
  }
#pragma unroll
  for (int h = 32; h > 0; h >>= 1) {
    lo = min(lo, static_cast<uint32_t>(__shfl_xor(static_cast<int>(lo), h)));
    hi = max(hi, static_cast<uint32_t>(__shfl_xor(static_cast<int>(hi), h)));
  }
  if (lane == 0) {
    s_lo[wave] = lo;
    s_hi[wave] = hi;
  }
  for (int i = tid; i < EV_BINS; i += THREADS) hist[0][i] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    lo = min(lo, s_lo[w]);
    hi = max(hi, s_hi[w]);
  }

  // ---- the slots that kept tokens end up in lie below `top`; `stay` of the tokens are kept. (Only a token without a
  // page has a key of 0.)
  int top = keep, stay = keep;
  if (lo == 0) {
    int there = 0;
    for (int seg = 0; seg < segs; ++seg) {
      if (segs > 1) load(seg);
      each(seg, [&](int, int j, uint32_t k) { there += k != 0 && (apart || j < keep); });
    }
    there = wave_scan(there);
    if (lane == 63) totals[wave] = there;
    __syncthreads();
    stay = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) stay += totals[w];
    if (apart) top = stay = min(stay, keep);
    if (stay == 0) return finish(apart ? 0 : keep, 0);
  }

  // ---- the smallest kept key less lo, digit by digit; `left` of the tokens equal to it are kept
  uint32_t prefix = 0;
  int left = stay, equals = n, bits = hi > lo ? 32 - __builtin_clz(hi - lo) : 0;
  for (int now = 0; bits > 0 && left < equals; now ^= 1) {
    const int shift = max(bits - 11, 0);
    for (int seg = 0; seg < segs; ++seg) {
      if (segs > 1) load(seg);
      each(seg, [&](int, int, uint32_t k) {
        const uint32_t u = k - lo;
        // (the smallest key, which many tokens may share, such as no weight at all, is what is left of the count: adds
        // to one address go one by one)
        if (u != 0 && (bits >= 32 || (u >> bits) == (prefix >> bits)))
          atomicAdd(&hist[now][(u >> shift) & ((1u << (bits - shift)) - 1)], 1);
      });
    }
    __syncthreads();
    // a thread's bins from the top: the one in which the count from above reaches `left`
    int h[BPT], sum = 0;
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      h[i] = hist[now][EV_BINS - 1 - BPT * tid - i];
      sum += h[i];
      hist[now ^ 1][BPT * tid + i] = 0;
    }
    const int scan = wave_scan(sum);
    if (lane == 63) totals[wave] = scan;
    __syncthreads();
    int before = scan - sum, counted = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      before += w < wave ? totals[w] : 0;
      counted += totals[w];
    }
    if (tid == THREADS - 1) {
      h[BPT - 1] += equals - counted;
      sum += equals - counted;
    }
    if (before < left && before + sum >= left) {
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        if (before < left && before + h[i] >= left) {
          s_digit = EV_BINS - 1 - BPT * tid - i;
          s_left = left - before;
          s_equals = h[i];
        }
        before += h[i];
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(s_digit) << shift;
    left = s_left;
    equals = s_equals;
    bits = shift;
  }
  // kept: u >> bits above prefix >> bits, and of those equal there the first `left`

  // ---- exclusive ranks of a flag in slot order: of a group's first token. (Every wave scans the counts of all
  // by itself; two count buffers in turn, as a wave may be a call ahead of another.)
  int turn = 0;
  const auto ranks = [&](uint32_t flags, int (&rank)[G], int& before) {
    int* count = counts[turn];
    turn ^= 1;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int c = __builtin_popcount((flags >> (4 * i)) & 15u);
      const int scan = wave_scan(c);
      rank[i] = scan - c;
      if (lane == 63) count[i * WAVES + wave] = scan;
    }
    __syncthreads();
    constexpr int PER = (G * WAVES + 63) / 64;   // one count a lane, or two
    int c[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] = lane * PER + i < G * WAVES ? count[lane * PER + i] : 0;
      sum += c[i];
    }
    const int run = before + wave_scan(sum) - sum;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int at = i * WAVES + wave, l = at / PER;
      rank[i] += __builtin_amdgcn_readlane(run, l) + (PER == 2 && at % PER ? __builtin_amdgcn_readlane(c[0], l) : 0);
    }
    before = __builtin_amdgcn_readlane(run + sum, 63);
  };
  // tokens of a thread's group below the group's q-th
  const auto lower = [](uint32_t flags, int number) {
    return __builtin_popcount((flags >> (number & ~3)) & ((1u << (number & 3)) - 1));
  };

  int seen = 0, before = 0, holes = -1;
  for (int seg = 0; seg < segs; ++seg) {
    if (segs > 1) load(seg);
    uint32_t kept = 0, equal = 0;
    each(seg, [&](int number, int, uint32_t k) {
      const uint32_t u = bits < 32 ? (k - lo) >> bits : 0, p = bits < 32 ? prefix >> bits : 0;
      if (u > p) kept |= 1u << number;
      if (u == p) equal |= 1u << number;
    });
    int rank[G];
    if (left < equals) {
      // some of the equals only: the lowest slots
      ranks(equal, rank, seen);
      uint32_t some = 0;
      each(seg, [&](int number, int, uint32_t) {
        if (rank[number >> 2] + lower(equal, number) < left) some |= (equal >> number & 1u) << number;
      });
      equal = some;
    }
    kept |= equal;
    // holes below `top`, kept tokens from there on: a group's tokens below `top` flip
    uint32_t moved = kept;
#pragma unroll
    for (int i = 0; i < G; ++i) moved ^= ((1u << min(max(top - token(seg, i), 0), 4)) - 1) << (4 * i);
    if (lo == 0 && !apart)
      each(seg, [&](int number, int j, uint32_t k) {
        if (k == 0 && j < top) moved &= ~(1u << number);
      });
    ranks(moved, rank, before);
    if (holes < 0 && top < (seg + 1) * SEG) {
      // (top < n: the token of slot `top` is in this segment)
#pragma unroll
      for (int i = 0; i < G; ++i)
        if (token(seg, i) == (top & ~3)) s_left = rank[i] + lower(moved, 4 * i + (top & 3));
      __syncthreads();
      holes = s_left;
    }
    each(seg, [&](int number, int j, uint32_t) {
      const bool is = (moved >> number) & 1u;
      const int r = rank[number >> 2] + lower(moved, number);
      if (j < top) {
        if constexpr (FUSED) {
          if (is) s_first[r] = j;
        } else if (apart) {
          first[j] = is ? -1 - r : j;
        } else if (is) {
          first[r] = j;
        }
      } else if (is) {
        if constexpr (FUSED) s_second[r - holes] = j;
        else second[r - holes] = j;
      }
    });
  }
  finish(top, apart ? top : holes);
  if constexpr (FUSED) {
    __syncthreads();
    const int sub = tid & (lpr - 1);
    for (int r = tid / lpr; r < holes; r += THREADS / lpr) {
      const int src = s_second[r], dst = s_first[r];
      ev_move(a, b, head, src, a.c.page_of(b, src), dst, a.c.page_of(b, dst), sub);
    }
  }
}

// One move per group of lpr lanes (16 bytes of k and v a lane).
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a, int lpr, int blocks) {
  const long long bh = blockIdx.x / blocks;
  const int head = bh % a.c.heads, b = bh / a.c.heads;
  const int per = 256 / lpr, sub = threadIdx.x & (lpr - 1);
  const int count = a.count[bh];
  const int32_t* first = a.first + bh * a.list;
  const int32_t* second = a.second + bh * a.list;
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
    ev_move(a, b, head, src, a.c.page_of(b, src), dst, to, sub);
  }
}

}  // namespace trellis
