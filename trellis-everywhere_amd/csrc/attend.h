// attend.h — attention of one new token per row over a paged key-value cache, split over the length.
//
//   s_j = scale * q . k_j  (j < length),  p = softmax(s),  out = sum_j p_j v_j,
// for each query head over its key-value head (G = query heads / key-value heads share one), and
// optionally score_j += sum over those G heads of p_j. A row of length 0 gives zeros.
//
// Bound: every key and value is read once, 4 d bytes a token and key-value head against 4 G d flops.
//
// A workgroup takes a chunk of one (row, key-value head)'s tokens; its four waves take tiles of 32 tokens
// in turn, each on its own with no LDS and no barrier in the loop:
//   * S^T = K Q^T by v_mfma_f32_16x16x32: the A operand's lane (token l % 16, dims 8 (l / 16) ..) is a
//     16-byte load of a key's row, straight from memory; the B operand holds up to 16 query heads;
//   * the result has lane (head l % 16, tokens 4 (l / 16) + r) of each 16-token half, which is the B
//     operand P^T of out^T = V^T P^T if lane group g = l / 16 counts the tokens {4g + r, 16 + 4g + r} as
//     its k-slots: no lane exchange between the two products;
//   * V^T, the A operand, wants 8 tokens of one dim per lane. Each lane loads d / 16 consecutive dims of its
//     group's 8 tokens (whole rows per 16 lanes) and transposes in its own registers (v_perm_b32);
//   * both products leave the head on l % 16, so the running maximum and the sum are per-lane values.
//     The maximum that the weights are taken against moves only when a logit passes it by 2^4 (the weights
//     stay below 2^15), checked by one ballot, so a tile costs no exchange between lane groups.
// Precision: the weights enter their product as two terms of the cache's type (f16: 22 bits, their scale
// keeping them out of its subnormals; bf16: 16 bits, three terms where q or out is fp32), the sums are fp32.
// q of another type than the cache's is scaled by a power of 2 and split the same way.
//
// The chunks' results (maximum, sum, unnormalised out) meet in attend_join_kernel, in a fixed order.
#pragma once

#include "serve.h"

namespace trellis {

constexpr int ATT_WAVES = 4;
constexpr int ATT_TILE = 32;                          // tokens per tile
constexpr int ATT_CHUNK_MIN = ATT_TILE * ATT_WAVES;   // the shortest chunk: a tile per wave
constexpr int ATT_SPLITS = 1024;                      // the most chunks of a row
constexpr float ATT_LOW = -3.0e38f;                   // below every logit that counts
constexpr float ATT_TOP = 11.f;                       // log2 of the weight at the maximum when it is set
constexpr float ATT_SLACK = 4.f;                      // how far (log2) a logit may pass it

struct AttendArgs {
  const void* q;
  long long q_b, q_h;     // strides of q in elements
  int q_dt, q_vec;        // q_vec: q's rows are 16-byte aligned
  void* out;              // [rows][hq][d]
  int out_dt, hq, group, row_blocks, splits;
  float scale;            // times log2(e)
  float* part;            // splits > 1: [rows][kv heads][splits][hq of the kv head][d] unnormalised sums
  float* ml;              // [rows][hq][splits][2] maximum and sum
  float* total;           // with scores: [rows][hq][2] maximum and 1 / sum
  float* logits;          // with scores: [rows][hq][logit_stride]
  long long logit_stride;
  Cache c;
};

// The chunk of a row of n tokens: at least ATT_CHUNK_MIN, so that short rows use fewer workgroups.
__device__ __forceinline__ int att_chunk(int n, int splits) {
  const int per = (n + splits - 1) / splits;
  return max((per + ATT_CHUNK_MIN - 1) / ATT_CHUNK_MIN, 1) * ATT_CHUNK_MIN;
}

template <class T> struct AttType;
template <> struct AttType<_Float16> {
  typedef _Float16 vec8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float4_t mfma(vec8 a, vec8 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct AttType<bf16_t> {
  typedef __bf16 vec8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float4_t mfma(vec8 a, vec8 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

__device__ __forceinline__ float max_groups(float v, int lane) {   // over the four lanes of a head
  v = fmaxf(v, lane_xor<16>(v, lane));
  return fmaxf(v, lane_xor<32>(v, lane));
}
__device__ __forceinline__ float sum_groups(float v, int lane) {
  v += lane_xor<16>(v, lane);
  return v + lane_xor<32>(v, lane);
}

// T: the cache's type. DP: head dims padded to 64, 128 or 256; FULL: d == DP. EXACT: q or out is of another
// type than the cache's.
template <class T, int DP, bool FULL, bool EXACT>
__global__ __launch_bounds__(64 * ATT_WAVES) void attend_kernel(AttendArgs a) {
  typedef AttType<T> AT;
  typedef typename AT::vec8 vec8;
  constexpr bool BF = sizeof(T) == 2 && !std::is_same<T, _Float16>::value;
  constexpr int NQ = EXACT ? (BF ? 3 : 2) : 1;      // terms of q
  constexpr int NP = EXACT && BF ? 3 : 2;           // terms of the weights
  constexpr int KS = DP / 32;                       // k-steps of the first product
  constexpr int DL = DP / 16;                       // dims per lane of V
  constexpr int VC = DL / 4;                        // 8-byte pieces of them
  __shared__ float s_m[ATT_WAVES][16], s_l[ATT_WAVES][16];
  __shared__ __align__(16) float s_o[ATT_WAVES][16][DP + 4];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r16 = lane & 15, g = lane >> 4;
  int id = blockIdx.x;
  const int split = id % a.splits; id /= a.splits;
  const int rb = id % a.row_blocks; id /= a.row_blocks;
  const int head = id % a.c.heads, b = id / a.c.heads;
  const int n = __builtin_amdgcn_readfirstlane(a.c.length(b));
  const int chunk = att_chunk(n, a.splits);
  const int begin = split * chunk, end = min(n, begin + chunk);
  if (begin >= n && split > 0) return;              // (a row of length 0 still writes its zeros)
  const int rows = min(16, a.group - rb * 16);      // query heads of this workgroup
  const int h0 = head * a.group + rb * 16;          // the first of them
  const int d = a.c.d;

  // ---- q: lane (head r16, dims 32 j + 8 g ..), in NQ terms of T
  vec8 q[NQ][KS];
  float fold = a.scale;
  {
    float f[KS][8];
#pragma unroll
    for (int j = 0; j < KS; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[j][i] = 0.f;
      const int dim = 32 * j + 8 * g;
      if (r16 < rows && dim < d) {
        const long long at = b * a.q_b + (h0 + r16) * a.q_h + dim;
        if (a.q_dt == DT_F32) {
          if (a.q_vec) load8<float, true>(static_cast<const float*>(a.q) + at, f[j]);
          else load8<float, false>(static_cast<const float*>(a.q) + at, f[j]);
        } else if (a.q_dt == DT_F16) {
          if (a.q_vec) load8<_Float16, true>(static_cast<const _Float16*>(a.q) + at, f[j]);
          else load8<_Float16, false>(static_cast<const _Float16*>(a.q) + at, f[j]);
        } else {
          if (a.q_vec) load8<bf16_t, true>(static_cast<const bf16_t*>(a.q) + at, f[j]);
          else load8<bf16_t, false>(static_cast<const bf16_t*>(a.q) + at, f[j]);
        }
      }
    }
    if constexpr (EXACT) {
      // the row's largest element to [0.5, 1), so that no term leaves the type's range
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[j][i]));
      top = max_groups(top, lane);
      const int e = top > 0.f && top < __builtin_inff() ? __builtin_amdgcn_frexp_expf(top) : 0;
      fold = __builtin_ldexpf(fold, e);
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float rest = __builtin_ldexpf(f[j][i], -e);
#pragma unroll
          for (int t = 0; t < NQ; ++t) {
            const T part = static_cast<T>(rest);
            q[t][j][i] = part;
            rest -= static_cast<float>(part);
          }
        }
    } else {
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) q[0][j][i] = static_cast<T>(f[j][i]);
    }
  }

  // ---- the wave's tiles: begin / 32 + wave, + 4, ..
  float4_t o[DL];
#pragma unroll
  for (int e = 0; e < DL; ++e) o[e] = float4_t{0.f, 0.f, 0.f, 0.f};
  float m = ATT_LOW, l = 0.f;

  u32x4_t kf[2][KS];
  uint2 vf[8][VC];
  const int sstr = static_cast<int>(a.c.slot_stride) * 2;      // bytes
  // the lane's byte offsets within a 16-token half
  const int koff = r16 * sstr + g * 16;
  const int voff = 4 * g * sstr + r16 * DL * 2;
  int pg[2];                                                   // pages of the tile's halves
  long long at[2];                                             // their element offsets
  const auto locate = [&](int t0) {
    // (a half that begins past the row's end may lie past the table: it is masked, any row serves)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int j = t0 + 16 * hf < n ? t0 + 16 * hf : t0;
      pg[hf] = a.c.page_of(b, j);
      at[hf] = a.c.row_at(max(pg[hf], 0), head, j);
    }
  };
  const auto load_k = [&]() {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const char* p = static_cast<const char*>(a.c.k) + 2 * at[hf];
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        if (FULL || 32 * j + 8 * g < d) kf[hf][j] = *reinterpret_cast<const u32x4_t*>(p + koff + 64 * j);
        else kf[hf][j] = u32x4_t{0, 0, 0, 0};
      }
    }
  };
  const auto load_v = [&]() {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const char* p = static_cast<const char*>(a.c.v) + 2 * at[i >> 2];
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        if (FULL || r16 * DL + 4 * c < d) vf[i][c] = *reinterpret_cast<const uint2*>(p + voff + (i & 3) * sstr + 8 * c);
        else vf[i][c] = make_uint2(0, 0);
      }
    }
  };

  const int step = ATT_TILE * ATT_WAVES;
  int t0 = begin + wave * ATT_TILE;
  bool have = t0 < end;
  if (have) {
    locate(t0);
    load_k();
    load_v();
  }
  while (have) {
    const int cur = t0;
    const bool whole = cur + ATT_TILE <= n && pg[0] >= 0 && pg[1] >= 0;
    const bool ok0 = pg[0] >= 0, ok1 = pg[1] >= 0;
    // ---- S^T = K Q^T
    float s[8];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int t = 0; t < NQ; ++t) acc = AT::mfma(__builtin_bit_cast(vec8, kf[hf][j]), q[t][j], acc);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[4 * hf + r] = acc[r] * fold;
    }
    if (!whole) {
      // tokens past the end and on missing pages: no weight, and nothing of what their memory holds
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = cur + 16 * (i >> 2) + 4 * g + (i & 3);
        if (!(j < n && (i < 4 ? ok0 : ok1))) {
          s[i] = -__builtin_inff();
#pragma unroll
          for (int c = 0; c < VC; ++c) vf[i][c] = make_uint2(0, 0);
        }
      }
    }
    if (a.logits && r16 < rows) {
      float* p = a.logits + (static_cast<long long>(b) * a.hq + h0 + r16) * a.logit_stride + cur + 4 * g;
      *reinterpret_cast<float4_t*>(p) = float4_t{s[0], s[1], s[2], s[3]};
      *reinterpret_cast<float4_t*>(p + 16) = float4_t{s[4], s[5], s[6], s[7]};
    }
    // ---- weights against the running maximum
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i]);
    if (__any(top > m + (ATT_TOP + ATT_SLACK))) {
      const float to = fmaxf(m, max_groups(top, lane) - ATT_TOP);
      const float f = exp2f(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int e = 0; e < DL; ++e) o[e] *= f;
    }
    vec8 p[NP];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float w = __builtin_amdgcn_exp2f(s[i] - m);
      l += w;
#pragma unroll
      for (int t = 0; t < NP; ++t) {
        const T part = static_cast<T>(w);
        p[t][i] = part;
        w -= static_cast<float>(part);
      }
    }
    // ---- out^T += V^T P^T, a dim pair (one 32-bit word of the 8 tokens' rows) at a time
#pragma unroll
    for (int e = 0; e < DL; e += 2) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = (e & 2) ? vf[i][e / 4].y : vf[i][e / 4].x;
      u32x4_t lo, hi;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100u);
        hi[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302u);
      }
#pragma unroll
      for (int t = 0; t < NP; ++t) {
        o[e] = AT::mfma(__builtin_bit_cast(vec8, lo), p[t], o[e]);
        o[e + 1] = AT::mfma(__builtin_bit_cast(vec8, hi), p[t], o[e + 1]);
      }
    }
    t0 += step;
    have = t0 < end;
    if (have) {
      locate(t0);
      load_k();
      load_v();
    }
  }
  l = sum_groups(l, lane);

  // ---- the waves' results meet
  if (g == 0) {
    s_m[wave][r16] = m;
    s_l[wave][r16] = l;
  }
  if (r16 < rows) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < DL; e += 4)
        *reinterpret_cast<float4_t*>(&s_o[wave][r16][DL * (4 * g + r) + e]) = float4_t{o[e][r], o[e + 1][r], o[e + 2][r], o[e + 3][r]};
  }
  __syncthreads();
  const long long bh = static_cast<long long>(b) * a.hq + h0;
  for (int it = threadIdx.x; it < rows * (DP / 4); it += 64 * ATT_WAVES) {
    const int row = it / (DP / 4), dim = (it % (DP / 4)) * 4;
    float mx = s_m[0][row];
#pragma unroll
    for (int w = 1; w < ATT_WAVES; ++w) mx = fmaxf(mx, s_m[w][row]);
    float sum = 0.f;
    float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < ATT_WAVES; ++w) {
      const float f = exp2f(s_m[w][row] - mx);
      sum = __builtin_fmaf(s_l[w][row], f, sum);
      acc += *reinterpret_cast<const float4_t*>(&s_o[w][row][dim]) * f;
    }
    if (a.splits == 1) {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;   // no token (or none on a page that exists)
      if (dim < d) {
        const long long o0 = (bh + row) * d + dim;
#pragma unroll
        for (int i = 0; i < 4; ++i) store_dt(a.out, o0 + i, a.out_dt, acc[i] * inv);
      }
      if (a.total && dim == 0) {
        a.total[2 * (bh + row)] = mx;
        a.total[2 * (bh + row) + 1] = inv;
      }
    } else {
      if (dim < d) *reinterpret_cast<float4_t*>(a.part + ((bh + row) * a.splits + split) * d + dim) = acc;
      if (dim == 0) {
        float* p = a.ml + 2 * ((bh + row) * a.splits + split);
        p[0] = mx;
        p[1] = sum;
      }
    }
  }
}

// The chunks of one (row, query head) joined: out = sum_c f_c part_c / sum_c f_c sum_c, f_c = 2^(m_c - max).
// A workgroup's threads take the chunks' maxima and sums side by side, then the partial sums as (chunk group,
// 4 dims), so that all of a round's loads are in flight together; one thread per dim that walked the chunks
// one after another took 48 us for 64 chunks of 32 heads, this takes 4.
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a) {
  __shared__ float s_f[ATT_SPLITS], s_red[2][4];
  __shared__ float4_t s_acc[256];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const long long bh = blockIdx.x;
  const int b = static_cast<int>(bh / a.hq), d = a.c.d;
  const int n = a.c.length(b), chunk = att_chunk(n, a.splits);
  const int used = max((n + chunk - 1) / chunk, 1);
  const float2* ml = reinterpret_cast<const float2*>(a.ml) + bh * a.splits;
  float m[ATT_SPLITS / 256], l[ATT_SPLITS / 256], mx = ATT_LOW;
#pragma unroll
  for (int i = 0; i < ATT_SPLITS / 256; ++i) {
    const int c = tid + 256 * i;
    const float2 v = c < used ? ml[c] : make_float2(ATT_LOW, 0.f);
    m[i] = v.x;
    l[i] = v.y;
    mx = fmaxf(mx, v.x);
  }
  mx = wave_max(mx, lane);
  if (lane == 0) s_red[0][wave] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < ATT_SPLITS / 256; ++i) {
    const float f = exp2f(m[i] - mx);
    if (tid + 256 * i < used) s_f[tid + 256 * i] = f;
    sum = __builtin_fmaf(l[i], f, sum);
  }
  sum = wave_sum(sum, lane);
  if (lane == 0) s_red[1][wave] = sum;
  __syncthreads();
  sum = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;   // no token (or none on a page that exists)
  const int quads = d / 4, groups = 256 / quads;
  const int grp = tid / quads, dim = (tid - grp * quads) * 4;
  float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
  if (grp < groups) {
#pragma unroll 8
    for (int c = grp; c < used; c += groups)
      acc += *reinterpret_cast<const float4_t*>(a.part + (bh * a.splits + c) * d + dim) * s_f[c];
  }
  s_acc[tid] = acc;
  __syncthreads();
  if (grp == 0) {
    for (int i = 1; i < groups; ++i) acc += s_acc[i * quads + tid];
#pragma unroll
    for (int i = 0; i < 4; ++i) store_dt(a.out, bh * d + dim + i, a.out_dt, acc[i] * inv);
  }
  if (a.total && tid == 0) {
    a.total[2 * bh] = mx;
    a.total[2 * bh + 1] = inv;
  }
}

// score_j += sum over the key-value head's query heads of p_j.
__global__ __launch_bounds__(256) void attend_score_kernel(AttendArgs a) {
  int id = blockIdx.x;
  const int per = (a.c.max_len + 255) / 256;
  const int j = (id % per) * 256 + threadIdx.x; id /= per;
  const int head = id % a.c.heads, b = id / a.c.heads;
  if (j >= a.c.length(b)) return;
  const int page = a.c.page_of(b, j);
  if (page < 0) return;
  float sum = 0.f;
  for (int i = 0; i < a.group; ++i) {
    const long long bh = static_cast<long long>(b) * a.hq + head * a.group + i;
    sum += exp2f(a.logits[bh * a.logit_stride + j] - a.total[2 * bh]) * a.total[2 * bh + 1];
  }
  a.c.scores[a.c.slot_at(page, head, j)] += sum;
}

}  // namespace trellis
