// tree_join.h — the attention of several new tokens: the chunks' results joined (tree.h).
#pragma once

#include "tree_rows.h"

namespace trellis {

// The parts of a (token, key-value head)'s queries joined: out = sum_i f_i part_i / sum_i f_i sum_i, f_i = 2^(m_i - max).
// Threads are (share of the parts, query, 4 dims).
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a, int qr) {
  __shared__ float4_t s_acc[256];
  __shared__ float s_sum[256];
  const int tid = threadIdx.x, lane = tid & 63, d = a.c.d;
  const int t = uniform(blockIdx.x / a.c.heads), head = blockIdx.x - t * a.c.heads;
  const TreePlace at = tree_find(a, qr, -1, t, lane);
  const int b = uniform(at.b);
  if (b < 0 || at.chunks < 2) return;
  const TreeRow row = tree_row(a, b);
  const int size = at.units * TREE_UNIT, token = t - row.first;
  const int quads = d / 4, most = 256 / quads, some = min(a.group, most), shares = most / some;
  const int quad = tid % quads, slot = tid / quads, mine = slot % some, share = slot / some;
  for (int g0 = 0; g0 < a.group; g0 += some) {
    const int g = g0 + mine, qi = token * a.group + g, block = qi / qr;
    const int live = g < a.group && share < shares ? (tree_end(row, block, qr, a.group) + size - 1) / size : 0;
    float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
    if (live > 1) {
      // chunk i of the block
      const auto place = [&](int i) {
        const long long item = static_cast<long long>(at.before + i * at.blocks + at.blocks - 1 - block) * a.c.heads + head;
        return item * qr + (qi - block * qr);
      };
      float mx = ATT_LOW;
#pragma unroll 8
      for (int i = 0; i < live; ++i) mx = fmaxf(mx, a.ml[2 * place(i)]);
#pragma unroll 4
      for (int i = share; i < live; i += shares) {
        const float2 v = *reinterpret_cast<const float2*>(a.ml + 2 * place(i));
        const float f = exp2f(v.x - mx);
        sum = __builtin_fmaf(v.y, f, sum);
        acc += *reinterpret_cast<const float4_t*>(a.part + place(i) * d + 4 * quad) * f;
      }
    }
    s_acc[tid] = acc;
    s_sum[tid] = sum;
    __syncthreads();
    if (live > 1 && share == 0) {
      for (int i = 1; i < shares; ++i) {
        acc += s_acc[tid + i * some * quads];
        sum += s_sum[tid + i * some * quads];
      }
      store4_dt(a.out, (static_cast<long long>(t) * a.hq + head * a.group + g) * d + 4 * quad, a.out_dt, acc * (sum == 0.f ? 0.f : 1.0f / sum));
    }
    __syncthreads();
  }
}

}  // namespace trellis
