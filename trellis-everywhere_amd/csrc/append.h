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

// LPR lanes (a power of 2, 8 dims each) per (token, head) row; heads in the order q, k, v.
// VEC: every row of q, k and v is 16-byte aligned.
template <class TX, class TC, bool VEC>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a, int lpr) {
  const int lane = threadIdx.x & 63, sub = threadIdx.x & (lpr - 1);
  const int heads = a.hq + 2 * a.c.heads, d = a.c.d;
  const long long item = static_cast<long long>(blockIdx.x) * (256 / lpr) + threadIdx.x / lpr;
  // rows past the last go through the lane exchanges with the others
  const bool in = item < static_cast<long long>(a.tokens) * heads;
  const int t = in ? static_cast<int>(item / heads) : 0, hh = in ? static_cast<int>(item - static_cast<long long>(t) * heads) : 0;
  const int kind = hh < a.hq ? 0 : hh < a.hq + a.c.heads ? 1 : 2;   // q, k, v
  const int head = kind == 0 ? hh : kind == 1 ? hh - a.hq : hh - a.hq - a.c.heads;

  // the token's row b and slot: lens counts the call's tokens already
  int b = t, slot;
  bool live = in;
  if (a.starts) {
    int lo = 0, hi = a.c.rows;   // the last row whose first token is at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.starts[mid] <= t) lo = mid;
      else hi = mid;
    }
    b = lo;
    const int first = a.starts[b], end = a.starts[b + 1];
    live = live && t >= first && t < end;
    slot = a.c.lens[b] - (end - t);
  } else {
    slot = a.c.lens[b] - 1;
  }
  live = live && slot >= 0 && slot < (static_cast<long long>(a.c.width) << a.c.page_shift);
  const int page = live ? a.c.page_of(b, slot) : -1;
  live = live && page >= 0;

  const bool own = in && sub * 8 < d;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const TX* src = kind == 0 ? static_cast<const TX*>(a.q) + t * a.q_t + head * a.q_h
                  : kind == 1 ? static_cast<const TX*>(a.k) + t * a.k_t + head * a.k_h
                              : static_cast<const TX*>(a.v) + t * a.v_t + head * a.v_h;
  if (own) load8<TX, VEC>(src + sub * 8, x);
  const float* w = kind == 0 ? a.q_w : a.k_w;
  const bool normed = kind != 2 && w;
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
  ss = group_sum(ss, lpr, lane);
  if (normed && own) {
    const float f = 1.0f / __builtin_sqrtf(ss * (1.0f / static_cast<float>(d)) + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * f * w[sub * 8 + i];
  }
  const int position = a.positions ? (in ? a.positions[t] : 0) : slot;
  if (a.cos) {
    // the partner dims sit rot / 16 lanes up (first half) or down (second half)
    const int hl = a.rot / 16;
    const bool first = sub < hl, turn = sub < 2 * hl && kind != 2;
    const int from = (lane & ~(lpr - 1)) + (first ? sub + hl : turn ? sub - hl : sub);
    const int i0 = (first ? sub : sub - hl) * 8;
    const bool known = position >= 0 && position < a.n_positions;
    const long long row = static_cast<long long>(known ? position : 0) * (a.rot / 2) + i0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl(x[i], from);
      if (turn && own) {
        // a position that the table does not hold has no angle: NaN
        const float c = known ? a.cos[row + i] : __builtin_nanf(""), s = known ? a.sin[row + i] : __builtin_nanf("");
        x[i] = first ? x[i] * c - other * s : x[i] * c + other * s;
      }
    }
  }
  if (!own) return;
  if (kind == 0) {
    // a token without a slot (padding) gets zeros
    if (!live)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    store8_dt<true>(a.q_out, (static_cast<long long>(t) * a.hq + head) * d + sub * 8, a.q_dt, x);
    return;
  }
  if (!live) return;
  TC* dst = static_cast<TC*>(kind == 1 ? a.c.k : a.c.v) + a.c.row_at(page, head, slot) + sub * 8;
  store8<TC, true>(dst, x);
  if (kind == 1 && sub == 0) {
    const long long p = a.c.slot_at(page, head, slot);
    if (a.c.scores) a.c.scores[p] = 0.f;
    if (a.c.pos) a.c.pos[p] = position;
  }
}

}  // namespace trellis
