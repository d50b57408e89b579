// tree_join.h — the attention of several new tokens: the chunks' results joined (tree.h).
#pragma once

#include "tree_rows.h"

namespace trellis {

// out = sum_i f_i part_i / sum_i f_i sum_i over a block's chunks i, f_i = 2^(m_i - max). A workgroup's threads are (share of
// the chunks, query, 4 dims): `subs` workgroups a block. The maximum runs along with the sums, so that no load waits for
// another one. Bound: the partial sums' bytes (one row of 32717 tokens, 63 new: 33.5 MB in 8.8 us), and a launch behind the
// chunks' (1.5 to 2 us).
constexpr int tree_join_rows(int d, int shares) { return 256 / (d / 4) / shares; }

__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a, int qr, int subs, int shares) {
  __shared__ float4_t s_acc[256];
  __shared__ float2 s_ml[256];
  const int tid = threadIdx.x, d = a.c.d, quads = d / 4;
  const unsigned unit = uniform(blockIdx.x / subs);
  const int sub = blockIdx.x - unit * subs, pos = uniform(unit / a.c.heads), head = unit - pos * a.c.heads;
  const int all = a.done->live;          // (written by the chunks' kernel: no load_const)
  const TreeBlock block = a.done[1 + pos];
  if (pos >= all || block.live < 2) return;
  const int rows = tree_join_rows(d, shares), slot = tid / quads, quad = tid - slot * quads, share = slot / rows;
  const int nth = sub * rows + slot - share * rows, qi = block.block * qr + nth, live = block.live;
  const bool is = share < shares && nth < qr && qi < block.queries;
  // chunk i of the block
  const long long first = (static_cast<long long>(block.first) * a.c.heads + head) * qr + nth;
  const long long step = static_cast<long long>(block.step) * a.c.heads * qr;
  float m = ATT_LOW, sum = 0.f;
  float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
  if (is) {
#pragma unroll 8
    for (int i = share; i < live; i += shares) {
      const float2 v = *reinterpret_cast<const float2*>(a.ml + 2 * (first + i * step));
      const float4_t p = *reinterpret_cast<const float4_t*>(a.part + (first + i * step) * d + 4 * quad);
      const float to = fmaxf(m, v.x), old = exp2f(m - to), f = exp2f(v.x - to);
      m = to;
      sum = sum * old + v.y * f;
      acc = acc * old + p * f;
    }
  }
  if (shares > 1) {
    s_acc[tid] = acc;
    s_ml[tid] = make_float2(m, sum);
    __syncthreads();
    if (share == 0) {
      for (int i = 1; i < shares; ++i) {
        const float2 v = s_ml[tid + i * rows * quads];
        const float to = fmaxf(m, v.x), old = exp2f(m - to), f = exp2f(v.x - to);
        m = to;
        sum = sum * old + v.y * f;
        acc = acc * old + s_acc[tid + i * rows * quads] * f;
      }
    }
  }
  if (!is || share > 0) return;
  const int token = qi / a.group;
  const long long to = (static_cast<long long>(block.token + token) * a.hq + head * a.group + qi - token * a.group) * d;
  store4_dt(a.out, to + 4 * quad, a.out_dt, acc * (sum == 0.f ? 0.f : 1.0f / sum));
}

}  // namespace trellis
