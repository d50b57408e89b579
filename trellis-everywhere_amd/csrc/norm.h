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
// elements are blockDim apart.
template <class TX, class TR, bool VEC, int C>
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs a) {
  __shared__ float slots[2][16];
  const int tid = threadIdx.x, nt = blockDim.x, width = a.width;
  const long long row = blockIdx.x;
  const TX* x = static_cast<const TX*>(a.x) + row * a.ldx;
  const TX* gate = a.gate ? static_cast<const TX*>(a.gate) + row * a.ldg : nullptr;
  const TR* res = a.residual ? static_cast<const TR*>(a.residual) + row * a.ldr : nullptr;
  const auto at = [&](int c, int i) { return VEC ? (tid + c * nt) * 8 + i : tid + (c * 8 + i) * nt; };

  float b[C][8], r[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) b[c][i] = r[c][i] = 0.f;
  const auto fetch = [&](const auto* p, float (&v)[8], int c) {
    if constexpr (VEC) {
      if (at(c, 0) < width) load8<std::remove_cv_t<std::remove_pointer_t<decltype(p)>>, true>(p + at(c, 0), v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at(c, i) < width) v[i] = static_cast<float>(p[at(c, i)]);
    }
  };
#pragma unroll
  for (int c = 0; c < C; ++c) fetch(x, b[c], c);
  if (res)
#pragma unroll
    for (int c = 0; c < C; ++c) fetch(res, r[c], c);
  const float inv = 1.0f / static_cast<float>(width);
  if (a.post_w) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(b[c][i], b[c][i], ss);
    const float f = 1.0f / __builtin_sqrtf(block_sum(ss, slots[0]) * inv + a.eps);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float p[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      fetch(a.post_w, p, c);
#pragma unroll
      for (int i = 0; i < 8; ++i) b[c][i] = b[c][i] * f * p[i];
    }
  }
  if (gate) {
    if (a.gate_inner == 0) {
      const float g0 = static_cast<float>(gate[0]);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) b[c][i] *= g0;
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float g[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        fetch(gate, g, c);
#pragma unroll
        for (int i = 0; i < 8; ++i) b[c][i] *= g[i];
      }
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      b[c][i] = __builtin_fmaf(a.scale, b[c][i], r[c][i]);
      // (elements past the width are 0 in b and r, and stay 0 unless scale is not finite)
      if (at(c, i) < width) ss = __builtin_fmaf(b[c][i], b[c][i], ss);
    }
  const float f = 1.0f / __builtin_sqrtf(block_sum(ss, slots[1]) * inv + a.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, y[8];
    fetch(a.w, w, c);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = b[c][i] * f * w[i];
    if constexpr (VEC) {
      if (at(c, 0) < width) {
        if (a.h) store8<TR, true>(static_cast<TR*>(a.h) + row * a.ldh + at(c, 0), b[c]);
        store8_dt<true>(a.y, row * a.ldy + at(c, 0), a.y_dt, y);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at(c, i) < width) {
          if (a.h) static_cast<TR*>(a.h)[row * a.ldh + at(c, i)] = static_cast<TR>(b[c][i]);
          store_dt(a.y, row * a.ldy + at(c, i), a.y_dt, y[i]);
        }
    }
  }
}

}  // namespace trellis
