// tree.h — attention of several new tokens per row over a paged key-value cache. Row b's n newest tokens lie in its last n
// slots, base = length - n; the i-th of them sees the slots below base, itself and its ancestors:
//   out_i = sum_j p_ij v_j,  p_i = softmax over the j it sees of scale q_i . k_j,
// its parent being parents[i] (a token before it; anything else: none), or (no parents) the token before it, so that it
// sees all up to itself: a prompt, or part of one. A token that sees nothing gives zeros.
#pragma once

#include "serve.h"

namespace trellis {

struct TreeArgs {
  const void* q;
  long long q_t, q_h;        // strides of q in elements
  int q_dt, out_dt, tokens, hq, group;
  const int32_t* starts;     // [rows + 1], or null: `each` tokens a row
  int each;
  const int32_t* parents;    // [tokens], or null
  void* out;                 // [tokens][hq][d]
  float scale;
  Cache c;
};

__device__ __forceinline__ float load_dt(const void* p, long long i, int dt) {
  if (dt == DT_F32) return static_cast<const float*>(p)[i];
  if (dt == DT_F16) return static_cast<const _Float16*>(p)[i];
  return static_cast<const bf16_t*>(p)[i];
}

// One wave a (token, query head): a key a lane for the logits, four dims a lane for the sums.
template <class T>
__global__ __launch_bounds__(64) void tree_kernel(TreeArgs a) {
  __shared__ float s_q[256];
  const int lane = threadIdx.x, t = blockIdx.x / a.hq, qh = blockIdx.x - t * a.hq, head = qh / a.group, d = a.c.d;
  int b = t / max(a.each, 1), first = b * a.each, n = a.each;
  if (a.starts) {
    b = 0;
    for (int i = 0; i < a.c.rows; i += 64) b += __popcll(__ballot(i + lane < a.c.rows && a.starts[i + lane + 1] <= t));
    first = b < a.c.rows ? min(max(a.starts[b], 0), a.tokens) : 0;
    n = b < a.c.rows && first <= t ? min(a.starts[b + 1], a.tokens) - first : 0;
  }
  float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
  float m = -3.0e38f, l = 0.f;
  const int len = n > 0 ? a.c.length(b) : 0, i = t - first;
  const long long base = n > 0 ? static_cast<long long>(a.c.lens[b]) - n : 0;
  if (n > 0 && base + i >= 0 && base + i < len) {
    for (int j = lane; j < d; j += 64) s_q[j] = load_dt(a.q, t * a.q_t + qh * a.q_h + j, a.q_dt);
    __syncthreads();
    const int end = static_cast<int>(base + i) + 1;
    for (int j0 = 0; j0 < end; j0 += 64) {
      const int j = j0 + lane;
      bool sees = j < end;
      if (sees && a.parents && j >= base) {
        const int want = static_cast<int>(j - base);
        int at = i;
        while (at > want) {
          const int p = a.parents[first + at];
          at = p >= 0 && p < at ? p : -1;
        }
        sees = at == want;
      }
      const int page = sees ? a.c.page_of(b, j) : -1;
      sees = page >= 0;
      const long long row = sees ? a.c.row_at(page, head, j) : 0;
      float s = 0.f;
      if (sees) {
        const T* k = static_cast<const T*>(a.c.k) + row;
        for (int e = 0; e < d; e += 8) {
          float f[8];
          load8<T, true>(k + e, f);
#pragma unroll
          for (int u = 0; u < 8; ++u) s = __builtin_fmaf(f[u], s_q[e + u], s);
        }
        s *= a.scale;
      }
      const float top = fmaxf(m, wave_max(sees ? s : -3.0e38f, lane));
      const float f = exp2f((m - top) * 1.44269504f), p = sees ? exp2f((s - top) * 1.44269504f) : 0.f;
      m = top;
      l = l * f + wave_sum(p, lane);
      acc *= f;
      for (int u = 0; u < 64; ++u) {
        const float w = __shfl(p, u);
        const long long r = __shfl(row, u);
        if (!__shfl(static_cast<int>(sees), u)) continue;
        if (4 * lane < d) acc += load4<T, true>(static_cast<const T*>(a.c.v) + r + 4 * lane) * w;
      }
    }
  }
  if (4 * lane < d) store4_dt(a.out, (static_cast<long long>(t) * a.hq + qh) * d + 4 * lane, a.out_dt, acc * (l == 0.f ? 0.f : 1.0f / l));
}

}  // namespace trellis
