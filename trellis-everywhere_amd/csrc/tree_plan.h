// tree_plan.h — the arithmetic on sizes of the attention of several new tokens, as plain functions that the host and the
// kernels share.
#pragma once

#include <cstdint>

namespace trellis {

constexpr int TREE_UNIT = 128;                        // tokens that chunks are counted in
constexpr int TREE_LEAST = 2;                         // units of the shortest chunk
constexpr int TREE_ROWS = 512;                        // the most rows that are cut into chunks

constexpr int tree_units(int n) { return (n + TREE_UNIT - 1) / TREE_UNIT; }

// A row's queries of one key-value head, token by token, are cut into blocks of `qr` = 32 x waves.
constexpr int tree_blocks(int64_t queries, int qr) { return static_cast<int>((queries + qr - 1) / qr); }

// Units of a chunk.
constexpr int tree_chunk_units(int units, int aim) {
  const int even = (units + aim - 1) / aim;
  return even > TREE_LEAST ? even : TREE_LEAST;
}

struct TreeChunks {
  int waves;       // of 32 queries each in a block: 1, 2 or 4 (of a workgroup's four; the others share their keys)
  int aim;         // chunks wanted of the whole work; 0: a block's keys are one chunk
  int64_t items;   // the most chunks that can be made
};

// `tokens` new tokens of `rows` rows up to n long, some `tokens` / rows each.
constexpr TreeChunks tree_chunks(int rows, int heads, int q_heads, int head_dim, int tokens, int n, int cus) {
  const int group = q_heads / heads;
  TreeChunks p = {4, 0, 0};
  if (rows < 1) return p;
  const int64_t queries = static_cast<int64_t>(tokens) * group, each = (queries + rows - 1) / rows;
  p.waves = each <= 32 && head_dim <= 128 ? 1 : each <= 64 ? 2 : 4;
  const int qr = 32 * p.waves;
  // every row has one block that is not full, and (where a block holds a token's queries) no more blocks than tokens
  int64_t blocks = queries / qr + rows;
  if (group <= qr && blocks > tokens) blocks = tokens;
  p.items = blocks * heads;
  const int64_t want = static_cast<int64_t>(cus) * (p.waves == 4 && head_dim <= 128 ? 2 : 1);
  if (n <= TREE_LEAST * TREE_UNIT || rows > TREE_ROWS || p.items >= want) return p;
  p.aim = static_cast<int>(want);
  p.items += p.aim;
  return p;
}

}  // namespace trellis
