// tree_rows.h — the attention of several new tokens: its arguments, and where a chunk or a token lies among the rows.
#pragma once

#include "serve.h"
#include "tree_plan.h"

namespace trellis {

struct TreeArgs {
  const void* q;
  long long q_t, q_h;        // strides of q in elements
  int q_dt, q_vec, out_dt, tokens, hq, group;
  const int32_t* starts;     // [rows + 1], or null: `each` tokens a row
  int each;
  const int32_t* parents;    // [tokens], or null
  void* out;                 // [tokens][hq][d]
  int aim;                   // chunks wanted of the whole work; 0: one a block
  int items;                 // workgroups that can have a chunk
  float scale;               // times log2(e)
  float* part;               // [items][queries of a block][d] unnormalised sums of blocks of several chunks
  float* ml;                 // [items][queries of a block][2] their maximum and sum
  struct TreeBlock* done;    // [blocks of one head + 1] what the join needs of each, their number first
  Cache c;
};

// A row's new tokens [first, first + n), the slot of the first, and how many tokens a call sees of it.
struct TreeRow {
  int first, n, base, len;
};

__device__ __forceinline__ TreeRow tree_row(const TreeArgs& a, int row) {
  const int b = min(row, a.c.rows - 1);
  TreeRow r;
  if (a.starts) {
    r.first = max(0, min(load_const(a.starts + b), a.tokens));
    r.n = max(0, min(load_const(a.starts + b + 1), a.tokens) - r.first);
  } else {
    r.first = b * a.each;
    r.n = a.each;
  }
  r.len = a.c.length(b);
  r.base = max(0, load_const(a.c.lens + b)) - r.n;
  if (row >= a.c.rows) r.n = 0;
  return r;
}

// A block of queries of several chunks, as the join finds it.
struct __attribute__((aligned(32))) TreeBlock {
  int live;                  // its chunks
  int first, step;           // the first one's place in one head's line, and from one to the next
  int token, queries, block; // the row's first token and its queries, and which of the row's blocks it is
};

// A row's place in the line of chunks: rows slowest, then its chunks, then its blocks from the last to the first, then
// heads.
struct TreePlace {
  int b, blocks, chunks;   // b < 0: no such row
  int before, skipped;     // chunks and blocks of one head of the rows below
  int all;                 // blocks of all rows (where they are cut into chunks)
  int units;               // of a chunk of the row
};

// The row of chunk `pos` of one head's line. By a whole wave.
__device__ __forceinline__ TreePlace tree_find(const TreeArgs& a, int qr, int pos, int lane) {
  constexpr int AHEAD = TREE_ROWS / 64;
  int units = 0, before = 0, skipped = 0, all = 0;
  for (int s = 0; s < a.c.rows; s += TREE_ROWS) {
    int blocks[AHEAD], own[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      blocks[i] = own[i] = 0;
      if (s + 64 * i >= a.c.rows) continue;
      const TreeRow r = tree_row(a, s + 64 * i + lane);
      blocks[i] = tree_blocks(static_cast<int64_t>(r.n) * a.group, qr);
      own[i] = max(1, tree_units(r.len));
    }
    if (a.aim) {   // (then there are no more rows than these)
      int work = 0, count = 0, most = 0;
      bool falls = false;      // starts in no order: no row then, as their tokens could be more than there are
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (a.starts && s + 64 * i + lane < a.c.rows)
          falls = falls || a.starts[s + 64 * i + lane + 1] < a.starts[s + 64 * i + lane];
        work += blocks[i] * own[i];
        count += blocks[i];
        most = max(most, blocks[i] ? own[i] : 0);
      }
      work = __builtin_amdgcn_readlane(wave_scan(work), 63);
      all = __builtin_amdgcn_readlane(wave_scan(count), 63);
      most = uniform(static_cast<int>(wave_max(static_cast<float>(most), lane)));   // (units: below 2^24)
      units = tree_chunk_units(work, all, most, a.c.heads, a.aim);
      if (__any(falls)) break;
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (s + 64 * i >= a.c.rows) continue;
      const int chunks = a.aim ? (own[i] + units - 1) / units : 1, mine = blocks[i] * chunks, scan = wave_scan(mine);
      const int scan_b = a.aim ? wave_scan(blocks[i]) : scan;
      const unsigned long long hit = __ballot(before + scan > pos);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        return {s + 64 * i + l, __builtin_amdgcn_readlane(blocks[i], l),
                __builtin_amdgcn_readlane(chunks, l), before + __builtin_amdgcn_readlane(scan - mine, l),
                skipped + __builtin_amdgcn_readlane(scan_b - blocks[i], l), all,
                __builtin_amdgcn_readlane((own[i] + chunks - 1) / chunks, l)};   // (its chunks alike)
      }
      before += __builtin_amdgcn_readlane(scan, 63);
      skipped += __builtin_amdgcn_readlane(scan_b, 63);
    }
  }
  return {-1, 0, 0, 0, 0, 0, 0};
}

// The end of the keys that a block of queries can see.
__device__ __forceinline__ int tree_end(const TreeRow& r, int block, int qr, int group) {
  const int last = min(r.n - 1, (block * qr + qr - 1) / group);
  return max(0, min(r.len, r.base + last + 1));
}

}  // namespace trellis
