// tree_plan.h — the arithmetic on sizes of the attention of several new tokens, as plain functions that the host and the
// kernels share.
#pragma once

#include <cstdint>

namespace trellis {

constexpr int TREE_UNIT = 128;                        // tokens that chunks are counted in
constexpr int TREE_LEAST = 1;                         // units of the shortest chunk
constexpr int TREE_WHOLE = 256;                       // tokens up to which a row is not cut
constexpr int TREE_ROWS = 512;                        // the most rows that are cut into chunks

constexpr int tree_units(int n) { return (n + TREE_UNIT - 1) / TREE_UNIT; }

// A row's queries of one key-value head, token by token, are cut into blocks of `qr` = 32 x waves.
constexpr int tree_blocks(int64_t queries, int qr) { return static_cast<int>((queries + qr - 1) / qr); }

// The most units of a chunk: an even share of the work (`units` of `blocks` blocks, the longest `most`) for each of `aim`
// workgroups, two thirds of one where rows are uneven, so that they end together (32 rows of up to 8192 tokens 133 -> 110 us;
// rows of one length 32.9 -> 37.4).
constexpr int tree_chunk_units(int units, int blocks, int most, int heads, int aim) {
  const int64_t work = static_cast<int64_t>(units) * heads;
  const int shares = 2 * static_cast<int64_t>(most) * blocks > 3 * static_cast<int64_t>(units) ? aim + aim / 2 : aim;
  const int64_t even = (work + shares - 1) / shares;
  return static_cast<int>(even > TREE_LEAST ? even : TREE_LEAST);
}

// Waves of a workgroup's four that have queries of their own; the others share a wave's queries and take other keys. All four
// for 16-bit types; two where q's and the weights' terms make the products two to six times as many (fp32 queries: 32 rows
// of 8192 tokens, 1 / 16 / 32 new ones each, two waves 209 / 241 / 419 us, four 332 / 361 / 390, one 205 / 312 / 538).
constexpr int tree_waves(bool exact) { return exact ? 2 : 4; }

struct TreeChunks {
  int aim;         // chunks wanted of the whole work; 0: a block's keys are one chunk
  int64_t blocks;  // the most blocks of all rows and heads
  int64_t items;   // the most chunks that can be made
};

// `tokens` new tokens of `rows` rows up to n long, some `tokens` / rows each.
constexpr TreeChunks tree_chunks(int rows, int heads, int q_heads, int head_dim, int tokens, int n, bool exact, int cus) {
  const int group = q_heads / heads, qr = 32 * tree_waves(exact);
  TreeChunks p = {0, 0, 0};
  if (rows < 1) return p;
  // every row has one block that is not full, and (where a block holds a token's queries) no more blocks than tokens
  const int64_t queries = static_cast<int64_t>(tokens) * group;
  int64_t blocks = queries / qr + rows;
  if (group <= qr && blocks > tokens) blocks = tokens;
  p.blocks = p.items = blocks * heads;
  // A share for each CU; two where the products bound the call and a CU's registers hold two workgroups (one or two shares:
  // a row of 9216 tokens, 1024 new 211 / 180 us, 64 new of 32768 65.1 / 67.6, 24 new 40.7 / 46.0; 8 rows of 4096, 24 new
  // 39.7 / 42.0, 48 new 62.6 / 54.2; 32 rows of 1024, 8 new 32.9 / 37.4).
  const bool twice = !exact && head_dim <= 128 && queries > static_cast<int64_t>(rows) * qr;
  const int64_t want = static_cast<int64_t>(cus) * (twice ? 2 : 1);
  // Two blocks a CU and more stay whole, whatever their lengths (whole / cut: 64 rows of 8 heads, 26 new, uneven up to 8192
  // 221 / 221 us, 96 345 / 359; 64 rows of 4096, 8 new, 186 / 194, of 1024 54.9 / 62.1; 200 uneven up to 2048 180 / 194; a
  // prompt's parts, 16 of 8192 tokens in all, 116 / 129): workgroups that wait leave memory to the others.
  if (n <= TREE_WHOLE || rows > TREE_ROWS || p.items >= 2 * static_cast<int64_t>(cus)) return p;
  p.aim = static_cast<int>(want);
  // (those that the work is cut into, and every block one that is not full)
  const int64_t most = p.blocks * tree_units(n) / TREE_LEAST;
  p.items += most < want + want / 2 ? most : want + want / 2;
  return p;
}

}  // namespace trellis
