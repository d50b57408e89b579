// norm.h — the norms around a block with its residual, one pass over the data:
//   b = x, or x * rsqrt(mean(x^2) + eps) * post_w      (the norm after the block)
//   h = residual + scale * gate * b                    (the residual stream)
//   y = h * rsqrt(mean(h^2) + eps) * w                 (the norm before the next block)
// Everything is fp32 from the loads to one rounding per output; y is formed from h before h is
// rounded to the residual's type.
#pragma once

#include "serve.h"

namespace trellis {

struct NormArgs {
  const void* x;
  const void* residual;   // or null: h = scale * gate * b
  const void* gate;       // x's type, or null
  const float* post_w;    // or null
  const float* w;
  void* h;                // residual's type, or null
  void* y;
  long long ldx, ldr, ldg, ldh, ldy;
  int width, gate_inner, y_dt;
  float scale, eps;
};

// The sum over the workgroup, in every thread; one LDS slot per wave, its own for each of a kernel's sums.
__device__ __forceinline__ float block_sum(float v, float* slots) {
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  v = wave_sum(v, lane);
  if (waves == 1) return v;
  if (lane == 0) slots[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lane < waves ? slots[lane] : 0.f;
  return wave_sum(v, lane);
}

// One workgroup per row, the row in registers: C chunks of 8 elements per thread. VEC: a thread's chunk is
// 8 consecutive elements, loaded 16 bytes at a time; otherwise (odd widths, strides or addresses) its
// elements are blockDim apart. Loads past the row's end take its last elements instead, without a branch, and
// everything a thread needs (C = 1; with more the weights of the last product come late) is in flight before
// the first sum.
// Bound: memory from some hundred rows on (8192 rows of 4096, f16 x and f32 residual 70 us, 5.7 TB/s; of 4095 79 us,
// 5.1; 2048 of 12288 56 us, 5.4; 1000 of 32768 with both norms and a gate 113 us, 4.0), below the chain of its steps
// (one row of 4096 2.2 us, 37 gated rows of 1531 with both norms 4.4).
template <class TX, class TR, bool VEC, int C>
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs a) {
  __shared__ float slots[2][16];
  const int tid = threadIdx.x, nt = blockDim.x, width = a.width;
  const long long row = blockIdx.x;
  const TX* x = static_cast<const TX*>(a.x) + row * a.ldx;
  const TX* gate = a.gate ? static_cast<const TX*>(a.gate) + row * a.ldg : nullptr;
  const TR* res = a.residual ? static_cast<const TR*>(a.residual) + row * a.ldr : nullptr;
  const auto at = [&](int c, int i) { return VEC ? (tid + c * nt) * 8 + i : tid + (c * 8 + i) * nt; };
  typedef float v8[8];
  const auto fetch = [&](const auto* p, v8& v, int c) {
    if constexpr (VEC) {
      load8<std::remove_cv_t<std::remove_pointer_t<decltype(p)>>, true>(p + min(at(c, 0), width - 8), v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(p[min(at(c, i), width - 1)]);
    }
  };

  const auto in = [&](int c, int i) { return at(c, VEC ? 0 : i) < width; };   // (VEC: a multiple of 8)
  const auto fetch_gate = [&](v8& v, int c) {
    if (a.gate_inner != 0) return fetch(gate, v, c);
    const float g0 = static_cast<float>(gate[0]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = g0;
  };

  float b[C][8], r[C][8], p[8], g[8], w[8];
#pragma unroll
  for (int c = 0; c < C; ++c) fetch(x, b[c], c);
  if (res)
#pragma unroll
    for (int c = 0; c < C; ++c) fetch(res, r[c], c);
  if constexpr (C == 1) {
    if (a.post_w) fetch(a.post_w, p, 0);
    if (gate) fetch_gate(g, 0);
    fetch(a.w, w, 0);
  }
  const float inv = 1.0f / static_cast<float>(width);
  if (a.post_w) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (in(c, i)) ss = __builtin_fmaf(b[c][i], b[c][i], ss);
    const float f = 1.0f / __builtin_sqrtf(block_sum(ss, slots[0]) * inv + a.eps);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if constexpr (C > 1) fetch(a.post_w, p, c);
#pragma unroll
      for (int i = 0; i < 8; ++i) b[c][i] = b[c][i] * f * p[i];
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (gate) {
      if constexpr (C > 1) fetch_gate(g, c);
#pragma unroll
      for (int i = 0; i < 8; ++i) b[c][i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      b[c][i] = res ? __builtin_fmaf(a.scale, b[c][i], r[c][i]) : a.scale * b[c][i];
      if (in(c, i)) ss = __builtin_fmaf(b[c][i], b[c][i], ss);
    }
  }
  const float f = 1.0f / __builtin_sqrtf(block_sum(ss, slots[1]) * inv + a.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float y[8];
    if constexpr (C > 1) fetch(a.w, w, c);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = b[c][i] * f * w[i];
    if constexpr (VEC) {
      if (in(c, 0)) {
        if (a.h) store8<TR, true>(static_cast<TR*>(a.h) + row * a.ldh + at(c, 0), b[c]);
        store8_dt<true>(a.y, row * a.ldy + at(c, 0), a.y_dt, y);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (in(c, i)) {
          if (a.h) static_cast<TR*>(a.h)[row * a.ldh + at(c, i)] = static_cast<TR>(b[c][i]);
          store_dt(a.y, row * a.ldy + at(c, i), a.y_dt, y[i]);
        }
    }
  }
}

}  // namespace trellis
