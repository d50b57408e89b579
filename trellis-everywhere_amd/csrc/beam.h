// beam.h — beam search's selection over beams and vocabulary. Per batch element, of the candidates
//   c(j, v) = score_j + x_jv - lse_j,  lse_j = log sum_v exp(x_jv)
// of beam j's logits x_j (an ended beam offers (j, end token) alone, at score_j), the k largest, equal ones by the
// lower beam, then the lower token. A candidate that is -inf or not a number is none.
// Within a beam the order is that of its logits, so the sums meet only where beams do, in 64 bits there: candidates of two
// beams may be nearer to each other than a rounding to 32 bits.
#pragma once

#include "serve.h"

namespace trellis {

constexpr int BEAM_MOST = 64;   // beams, and candidates kept of each (TRELLIS_BEAM_MAX)

struct BeamArgs {
  const void* x;
  long long x_b, x_j;           // strides of batch and beam in elements
  int batch, beams, vocab, k, end_token;
  const float* scores;          // [batch][beams]
  const uint8_t* ended;         // [batch][beams] or null
  float* out_scores;            // [batch][k]
  int32_t* out_beams;
  int32_t* out_tokens;
  double* lse;                  // workspace: [batch][beams]
  uint2* best;                  // workspace: [batch][beams][k] (key, token)
};

// Order-preserving, 0 for what is no candidate: -inf, not a number.
__device__ __forceinline__ uint32_t beam_key(float x) {
  if (!(x > -__builtin_inff())) return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);   // -0 counts as 0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float beam_value(uint32_t key) {
  return __builtin_bit_cast(float, (key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// One workgroup a beam: maximum and sum, then k times the largest below the last.
template <class T>
__global__ __launch_bounds__(256) void beam_row_kernel(BeamArgs a) {
  __shared__ float s_f[4];
  __shared__ double s_d[4];
  __shared__ unsigned long long s_u[4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int row = blockIdx.x, b = row / a.beams, j = row - b * a.beams;
  const T* x = static_cast<const T*>(a.x) + b * a.x_b + j * a.x_j;
  float top = -__builtin_inff();
  for (int i = tid; i < a.vocab; i += 256) {
    const float v = static_cast<float>(x[i]);
    top = v > top ? v : top;
  }
  top = wave_max(top, lane);
  if (lane == 0) s_f[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_f[0], s_f[1]), fmaxf(s_f[2], s_f[3]));
  double sum = 0.0;
  for (int i = tid; i < a.vocab; i += 256) {
    const float v = static_cast<float>(x[i]);
    if (v > -__builtin_inff()) sum += expf(v - top);
  }
  for (int h = 32; h > 0; h >>= 1) sum += __shfl_xor(sum, h);
  if (lane == 0) s_d[wave] = sum;
  __syncthreads();
  if (tid == 0) a.lse[row] = top + log((s_d[0] + s_d[1]) + (s_d[2] + s_d[3]));
  unsigned long long last = ~0ull;
  for (int n = 0; n < a.k; ++n) {
    unsigned long long best = 0;
    for (int i = tid; i < a.vocab; i += 256) {
      const uint32_t key = beam_key(static_cast<float>(x[i]));
      const unsigned long long c = key ? static_cast<unsigned long long>(key) << 32 | ~static_cast<uint32_t>(i) : 0;
      if (c < last && c > best) best = c;
    }
    for (int h = 32; h > 0; h >>= 1) {
      const unsigned long long o = __shfl_xor(best, h);
      best = o > best ? o : best;
    }
    __syncthreads();
    if (lane == 0) s_u[wave] = best;
    __syncthreads();
    for (int w = 0; w < 4; ++w) best = s_u[w] > best ? s_u[w] : best;
    last = best;
    if (tid == 0) a.best[static_cast<long long>(row) * a.k + n] = make_uint2(best >> 32, ~static_cast<uint32_t>(best));
  }
}

// One wave a batch element: a beam a lane, its candidates in order; k times the largest of the lanes' first ones.
__global__ __launch_bounds__(64) void beam_join_kernel(BeamArgs a) {
  const int lane = threadIdx.x, b = blockIdx.x;
  const long long row = static_cast<long long>(b) * a.beams + min(lane, a.beams - 1);
  const double none = -static_cast<double>(__builtin_inff());
  const bool ended = a.ended && a.ended[row];
  const double score = a.scores[row], lse = ended ? 0.0 : a.lse[row];
  int at = 0, token = a.end_token;
  double value = none;
  const auto next = [&]() {
    value = none;
    if (lane >= a.beams) return;
    if (ended) {
      if (at == 0) value = score;
    } else if (at < a.k) {
      const uint2 c = a.best[row * a.k + at];
      token = c.y;
      if (c.x) value = score + (static_cast<double>(beam_value(c.x)) - lse);
    }
    if (!(value > none)) value = none;
    ++at;
  };
  next();
  for (int n = 0; n < a.k; ++n) {
    double best = value;
    int from = lane;
    for (int h = 1; h < 64; h <<= 1) {
      const double o = __shfl_xor(best, h);
      const int f = __shfl_xor(from, h);
      if (o > best || (o == best && f < from)) {
        best = o;
        from = f;
      }
    }
    const int picked = __shfl(token, from);
    if (lane == 0) {
      const long long o = static_cast<long long>(b) * a.k + n;
      const bool is = best > none;
      a.out_scores[o] = static_cast<float>(best);
      a.out_beams[o] = is ? from : 0;
      a.out_tokens[o] = is ? picked : a.end_token;
    }
    if (lane == from) next();
  }
}

}  // namespace trellis
