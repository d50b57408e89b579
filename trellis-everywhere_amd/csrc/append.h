// append.h — new tokens into a paged key-value cache. Per token and head:
//   q' = rot(norm(q)),  cache key = rot(norm(k)),  cache value = v
//   norm(x) = x * rsqrt(mean(x^2) + eps) * w  (or x),
//   rot: pairs (x_i, x_{i + r/2}), i < r/2, turned by the angle of (position, i):
//        (x_i cos - x_{i+r/2} sin, x_{i+r/2} cos + x_i sin); the dims past r stay (or no rot)
// fp32 from the loads to one rounding per output.
#pragma once

#include "serve.h"

namespace trellis {

struct AppendArgs {
  const void* q;
  const void* k;
  const void* v;
  long long q_t, q_h, k_t, k_h, v_t, v_h;   // strides in elements
  void* q_out;                              // [tokens][hq][d]
  const float* q_w;
  const float* k_w;                         // norm weights [d], or null
  const float* cos;
  const float* sin;                         // [positions][rot / 2], or null
  const int32_t* starts;                    // [rows + 1], or null: token t is row t's
  const int32_t* positions;                 // [tokens], or null: the slot
  int tokens, hq, q_dt, rot, n_positions;
  float eps;
  Cache c;
};

// A workgroup takes one token and `rounds` times 256 / lpr of its heads (q, k, v in that order), lpr lanes (a
// power of 2) a head, so the token's row, slot, page and angles are found once. A lane holds 8 dims of its
// head: the rotary dims as 4 of the first half and their 4 partners of the second (nothing to exchange), the
// others 8 in a row. VEC: every row of q, k and v is 16-byte aligned.
// NT: nontemporal stores.
// Bound: memory for prompts (6007 tokens of 32 + 8 + 8 heads of 128, f16: 29 us, 5.2 TB/s; 38.5 with plain stores, and
// 90 with a lane group per (token, head) that looked up its token's row, slot and angles by itself), the chain length ->
// page id -> store for single tokens (one 3.0 us, 48 of 15 heads of 64 3.5).
template <class TX, class TC, bool VEC, bool NT>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a, int lpr, int rounds, int parts) {
  const int lane = threadIdx.x & 63, sub = threadIdx.x & (lpr - 1), group = threadIdx.x / lpr, groups = 256 / lpr;
  const int heads = a.hq + 2 * a.c.heads, d = a.c.d;
  const int t = blockIdx.x / parts, part = blockIdx.x - t * parts;

  // the token's row b and slot: lens counts the call's tokens already
  int b = t, slot = -1;
  bool live = true;
  if (a.starts) {
    // the row is the number of rows that end at or before t
    b = 0;
    for (int i = 0; i < a.c.rows; i += 64) b += __popcll(__ballot(i + lane < a.c.rows && a.starts[i + lane + 1] <= t));
    live = b < a.c.rows && a.starts[0] <= t;
    if (live) slot = a.c.lens[b] - (a.starts[b + 1] - t);
  } else {
    slot = a.c.lens[b] - 1;
  }
  live = live && slot >= 0 && slot < (static_cast<long long>(a.c.width) << a.c.page_shift);
  const int page = live ? a.c.page_of(b, slot) : -1;
  live = live && page >= 0;
  const int position = a.positions ? a.positions[t] : slot;

  // the lane's dims: d0 .. d0 + 3 and d1 .. d1 + 3
  const int turned = a.cos ? a.rot / 8 : 0;
  const bool turn = sub < turned, own = sub * 8 < d;
  const int d0 = turn ? 4 * sub : 8 * sub, d1 = turn ? a.rot / 2 + 4 * sub : 8 * sub + 4;
  float4_t c = float4_t{1.f, 1.f, 1.f, 1.f}, s = float4_t{0.f, 0.f, 0.f, 0.f};
  if (turn) {
    if (position >= 0 && position < a.n_positions) {
      const long long at = static_cast<long long>(position) * (a.rot / 2) + d0;
      c = *reinterpret_cast<const float4_t*>(a.cos + at);
      s = *reinterpret_cast<const float4_t*>(a.sin + at);
    } else {
      // a position that the table does not hold has no angle
      const float nan = __builtin_nanf("");
      c = s = float4_t{nan, nan, nan, nan};
    }
  }
  for (int r = 0; r < rounds; ++r) {
    const int hh = (part * rounds + r) * groups + group;
    const bool in = hh < heads;
    const int kind = hh < a.hq ? 0 : hh < a.hq + a.c.heads ? 1 : 2;   // q, k, v
    const int head = kind == 0 ? hh : kind == 1 ? hh - a.hq : hh - a.hq - a.c.heads;
    float4_t x = float4_t{0.f, 0.f, 0.f, 0.f}, y = x;
    if (in && own) {
      const TX* src = kind == 0 ? static_cast<const TX*>(a.q) + t * a.q_t + head * a.q_h
                      : kind == 1 ? static_cast<const TX*>(a.k) + t * a.k_t + head * a.k_h
                                  : static_cast<const TX*>(a.v) + t * a.v_t + head * a.v_h;
      x = load4<TX, VEC>(src + d0);
      y = load4<TX, VEC>(src + d1);
    }
    const float* w = kind == 0 ? a.q_w : a.k_w;
    if (w) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss = __builtin_fmaf(x[i], x[i], __builtin_fmaf(y[i], y[i], ss));
      ss = group_sum(ss, lpr, lane);
      if (kind != 2 && own) {
        const float f = 1.0f / __builtin_sqrtf(ss * (1.0f / static_cast<float>(d)) + a.eps);
        x = x * f * *reinterpret_cast<const float4_t*>(w + d0);
        y = y * f * *reinterpret_cast<const float4_t*>(w + d1);
      }
    }
    if (turn && kind != 2) {
      const float4_t u = x * c - y * s;
      y = y * c + x * s;
      x = u;
    }
    if (!in || !own) continue;
    if (kind == 0) {
      // a token without a slot (padding) gets zeros
      if (!live) x = y = float4_t{0.f, 0.f, 0.f, 0.f};
      const long long at = (static_cast<long long>(t) * a.hq + head) * d;
      store4_dt<NT>(a.q_out, at + d0, a.q_dt, x);
      store4_dt<NT>(a.q_out, at + d1, a.q_dt, y);
    } else if (live) {
      TC* dst = static_cast<TC*>(kind == 1 ? a.c.k : a.c.v) + a.c.row_at(page, head, slot);
      store4<NT>(dst + d0, x);
      store4<NT>(dst + d1, y);
      if (kind == 1 && sub == 0) {
        const long long p = a.c.slot_at(page, head, slot);
        if (a.c.scores) a.c.scores[p] = 0.f;
        if (a.c.pos) a.c.pos[p] = position;
      }
    }
  }
}

}  // namespace trellis
