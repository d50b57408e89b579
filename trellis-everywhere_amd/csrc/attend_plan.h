// attend_plan.h — the attention's arithmetic on sizes, as plain functions that the host and the kernels share.
#pragma once

#include <cstdint>

namespace trellis {

constexpr int ATT_WAVES = 4;
constexpr int ATT_TILE = 32;                          // tokens per tile
constexpr int ATT_UNIT = ATT_TILE * ATT_WAVES;        // tokens per unit: a tile per wave
constexpr int ATT_PARTS = 1024;                       // the most chunks of a row
constexpr int ATT_LONG = 8;                           // units of a chunk above which more chunks are preferred

constexpr int att_units(int n) { return (n + ATT_UNIT - 1) / ATT_UNIT; }

// ---- chunks. The lengths are on the GPU, so that is where the chunks of several rows are made: all of the same
// number of units, ceil(units / aim) up to ATT_LONG, above that so many that there are up to 4 aim of them (rows of
// uneven lengths then end together), at least 2. The chunks of all rows lie in a line, rows slowest, heads fastest; a
// workgroup's number is its chunk's place in the line, and the place of its partial sums. Against chunks of one size
// planned for the longest row: 16 rows up to 4099 tokens of 8 heads 39.3 -> 32.4 us, 64 up to 8192 228 -> 203, 4 up to
// 8192 24.9 -> 18.7. (aim, 2 aim, 4 aim chunks of 32 rows up to 8192: 120, 103, 98 us; of 24 up to 4096, 7 units each for
// aim: 43, 45, 45; ATT_LONG of 6, 8, 10: those 24 rows 49.6, 43.0, 42.6, 48 rows up to 4096 85, 86, 90, 12 up to 8192 56,
// 48, 48.)
constexpr int att_chunk_units(int units, int aim) {
  const int even = (units - 1) / aim + 1, many = (units - 1) / (4 * aim) + 1;
  return even <= ATT_LONG ? (even > 2 ? even : 2) : (many > ATT_LONG ? many : ATT_LONG);
}

struct AttChunks {
  int row_blocks;   // workgroups that share a chunk: 16 query heads each
  int aim;          // chunks wanted of the whole work; 0: a row is one chunk
  int chunk;        // one row: its chunks' tokens
  int64_t items;    // the most chunks that can be made
};

// One chunk a row up to 512 tokens (400 of 8 heads: 8.4 us either way, and a launch less), and beyond 512 rows, where
// rows alone fill the CUs and every workgroup would look through all lengths (512 rows in chunks / 513 whole: of 1024
// tokens of 8 heads 386 / 339 us, of up to 4096 tokens of 2 heads 213 / 226, one of 8192 among rows of 64 118 / 121).
// Otherwise chunks for two workgroups per CU, one where the head dim's registers leave room for no more (16 rows up
// to 4096 tokens of 2 heads of 256: 30.6 -> 26.5 us): a row's own are planned here (4000 tokens of 8 heads in
// chunks of 128 / 256 / 512: 11.4 / 13.7 / 14.4 us; 32717: 35.6 / 32.9 / 31.1, and 38.9 in 2048), those of several
// on the GPU (att_chunk_units).
constexpr AttChunks att_chunks(int rows, int heads, int q_heads, int head_dim, int n, int cus) {
  AttChunks p = {(q_heads / heads + 15) / 16, 0, 0, static_cast<int64_t>(rows) * heads};
  const int64_t one = p.items;
  if (n <= 512 || rows > 512 || one == 0) return p;
  const int64_t units = one * att_units(n);
  // no row may have more than ATT_PARTS chunks; a group of more row blocks than there are workgroups to aim at still
  // has one
  const int64_t cap = static_cast<int64_t>(ATT_PARTS - 1) * heads / (rows == 1 ? 1 : 4);
  const int64_t want = (head_dim > 128 ? 1 : 2) * cus / p.row_blocks;
  p.aim = static_cast<int>(want > cap ? cap : want);
  if (p.aim < 1) p.aim = 1;
  if (rows == 1) {
    const int64_t size = (units + p.aim - 1) / p.aim;
    p.chunk = static_cast<int>(size < att_units(n) ? size : att_units(n)) * ATT_UNIT;
    p.items = static_cast<int64_t>((n + p.chunk - 1) / p.chunk) * heads;
  } else {
    const int64_t many = units / ATT_LONG < 4 * static_cast<int64_t>(p.aim) ? units / ATT_LONG : 4 * static_cast<int64_t>(p.aim);
    // (and every row and head one that is not full)
    p.items = (many > p.aim ? many : p.aim) + one;
    if (p.items > units) p.items = units;
  }
  return p;
}

// The dim at which a lane begins to load 8 dims of a query head for k-step j: 32 j + 8 g, or the row's last 8 where it
// has none there (head dims that do not fill the last step's lane groups g; the values then count as zeros).
constexpr int att_q_dim(int j, int g, int d) { return 32 * j + 8 * g < d ? 32 * j + 8 * g : d - 8; }

}  // namespace trellis
