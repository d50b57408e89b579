// attend.h — attention of one new token per row over a paged key-value cache, split over the length.
//
//   s_j = scale * q . k_j  (j < length),  p = softmax(s),  out = sum_j p_j v_j,
// for each query head over its key-value head (G = query heads / key-value heads share one), and
// optionally score_j += sum over those G heads of p_j. A row of length 0 gives zeros.
//
// Bound: HBM. Every key and value is read once (counters: 1.00 times their bytes), 4 d bytes a token and key-value head
// against 4 G d flops. 8 heads of 128 for 32 query heads: 64 rows of 8192 tokens 341 us (6.3 TB/s), 64 of uneven lengths
// up to 8192 183 (5.9), one of 131072 91 (5.9), of 32717 27.6 (4.9, of which 4 the join), of 1000 8.7, one of 149
// tokens of a small model 5.1: there the chain length -> page ids -> keys -> weights -> values.
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
//     are at most 2^15, of bf16 2^4), checked by one ballot, so a tile costs no exchange between lane groups.
// Precision: the weights enter their product as two terms of the cache's type (f16: 22 bits, their scale
// keeping them out of its subnormals; bf16: 16 bits, of which a 16-bit out keeps 8 or 11, and three terms, 24 bits,
// where q is of another type or out is fp32), the sums are fp32.
// q of another type than the cache's (or with an fp32 out) is scaled by a power of 2 and split the same way: into an
// f16 cache 22 bits of each element down to 2^-17 of its row's largest, 2^-39 of that below.
//
// The chunks' results (maximum, sum, unnormalised out) meet in attend_finish_kernel, in a fixed order; with scores
// its other workgroups turn the logits that this kernel left into weights.
#pragma once

#include "attend_plan.h"
#include "serve.h"

namespace trellis {

constexpr float ATT_LOW = -3.0e38f;                   // below every logit that counts
constexpr float ATT_TOP = 11.f;                       // f16: log2 of the weight at the maximum when it is set
constexpr float ATT_SLACK = 4.f;                      // how far (log2) a logit may pass it

struct AttendArgs {
  const void* q;
  long long q_b, q_h;     // strides of q in elements
  int q_dt, q_vec;        // q_vec: q's rows are 16-byte aligned
  void* out;              // [rows][hq][d]
  int out_dt, hq, group, row_blocks;
  int aim;                // chunks wanted of the whole work; 0: a row is one chunk
  int chunk;              // one row: its chunks' tokens
  int items;              // workgroups (of one row block) that can have a chunk
  float scale;            // times log2(e)
  float* part;            // [items][group][d] unnormalised sums of rows of several chunks
  float* ml;              // [items][group][2] their maximum and sum
  float* total;           // with scores: [rows][hq][2] maximum and 1 / sum of rows of one chunk
  float* logits;          // with scores: [rows][hq][logit_stride]
  long long logit_stride;
  Cache c;
};

// A value that is the same in every lane, into a scalar register (a division leaves it in a vector register, and
// addresses made from it in two a lane).
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Lengths of rows r0 .. r0 + 63, one a lane.
__device__ __forceinline__ int att_lengths(const Cache& c, int r0, int lane) {
  const int b = r0 + lane, n = c.length(min(b, c.rows - 1));
  return b < c.rows ? n : 0;
}

// Units of a chunk of several rows (by a whole wave); `len0`: att_lengths of rows 0 .. 63.
__device__ __forceinline__ int att_chunk(const AttendArgs& a, int len0, int lane) {
  int units = 0;
  for (int r0 = 0; r0 < a.c.rows; r0 += 64)
    units += __builtin_amdgcn_readlane(wave_scan(att_units(r0 ? att_lengths(a.c, r0, lane) : len0)), 63);
  units *= a.c.heads;
  return uniform(att_chunk_units(units, a.aim));
}

struct Place {
  int b, n;       // a row and its length
  int chunks;     // of one head of it
  int before;     // chunks of one head of all rows below it
};

// The row with chunk `pos` of the line, or (pos < 0) row `b`; chunks 0 where the line ends below pos.
__device__ __forceinline__ Place att_find(const AttendArgs& a, int chunk, int pos, int b, int len0, int lane) {
  int before = 0;
  for (int r0 = 0; r0 < a.c.rows; r0 += 64) {
    const int len = r0 ? att_lengths(a.c, r0, lane) : len0, mine = (att_units(len) + chunk - 1) / chunk, scan = wave_scan(mine);
    const unsigned long long hit = pos < 0 ? (b < r0 + 64 ? 1ull << (b - r0) : 0) : __ballot((before + scan) * a.c.heads > pos);
    if (hit) {
      const int l = __builtin_ctzll(hit), chunks = __builtin_amdgcn_readlane(mine, l);
      return {r0 + l, __builtin_amdgcn_readlane(len, l), chunks, before + __builtin_amdgcn_readlane(scan, l) - chunks};
    }
    before += __builtin_amdgcn_readlane(scan, 63);
  }
  return {0, 0, 0, before};
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

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// NT: nontemporal, for what is read once and not again soon.
template <bool NT, class V>
__device__ __forceinline__ V load_once(const V* p) {
  return NT ? __builtin_nontemporal_load(p) : *p;
}

// T: the cache's type. DP: head dims padded to 64, 128 or 256; FULL: d == DP. EXACT: q or out is of another
// type than the cache's. NT: keys and values by nontemporal loads.
template <class T, int DP, bool FULL, bool EXACT, bool NT>
__global__ __launch_bounds__(64 * ATT_WAVES) void attend_kernel(AttendArgs a) {
  typedef AttType<T> AT;
  typedef typename AT::vec8 vec8;
  constexpr bool BF = sizeof(T) == 2 && !std::is_same<T, _Float16>::value;
  constexpr int NQ = EXACT ? (BF ? 3 : 2) : 1;      // terms of q
  constexpr int NP = EXACT && BF ? 3 : 2;           // terms of the weights
  constexpr int UP = BF ? 0 : 15;                   // log2 that q's largest element stays below
  constexpr float TOP = BF ? 0.f : ATT_TOP;         // (bf16 has no subnormals to keep out of, and values up to 2^128)
  constexpr int KS = DP / 32;                       // k-steps of the first product
  constexpr int DL = DP / 16;                       // dims per lane of V
  constexpr int VC = DL / 4;                        // 8-byte pieces of them
  __shared__ float s_m[ATT_WAVES][16], s_l[ATT_WAVES][16];
  __shared__ __align__(16) float s_o[ATT_WAVES][16][DP + 4];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r16 = lane & 15, g = lane >> 4;
  // The row blocks of an item are 8 workgroups apart, on one XCD (workgroups go to the 8 XCDs in turn), where the
  // second finds keys and values in its L2.
  const unsigned bid = blockIdx.x, octet = bid / (8 * a.row_blocks), in8 = bid - octet * 8 * a.row_blocks;
  const int rb = uniform(in8 >> 3), item = uniform(octet * 8 + (in8 & 7));
  if (item >= a.items) return;
  int b, head, n, begin, size;
  if (a.aim == 0) {
    b = uniform(item / a.c.heads);
    head = item - b * a.c.heads;
    begin = 0;
    n = size = a.c.length(b);
  } else if (a.chunk) {
    b = 0;
    const int nth = uniform(item / a.c.heads);
    head = item - nth * a.c.heads;
    size = a.chunk;
    begin = nth * size;
    n = a.c.length(0);
  } else {
    const int len0 = att_lengths(a.c, 0, lane), units = att_chunk(a, len0, lane);
    const Place at = att_find(a, units, item, 0, len0, lane);
    if (at.chunks == 0) return;
    const int off = item - at.before * a.c.heads, nth = uniform(off / a.c.heads);
    b = at.b;
    n = at.n;
    head = off - nth * a.c.heads;
    size = units * ATT_UNIT;
    begin = nth * size;
  }
  b = uniform(b);
  head = uniform(head);
  begin = uniform(begin);
  size = uniform(size);
  const int rows = min(16, a.group - rb * 16);      // query heads of this workgroup
  const int h0 = head * a.group + rb * 16;          // the first of them
  const int d = a.c.d;
  int t0 = begin + wave * ATT_TILE;
  // the first tile's pages beside the length (of the table's last page where it has no such: that tile is not taken)
  int pg[2];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf)
    pg[hf] = load_const(a.c.table + b * a.c.table_stride + min((t0 + 16 * hf) >> a.c.page_shift, a.c.width - 1));
  n = uniform(n);
  if (begin >= n && begin > 0) return;              // (a row of length 0 is one chunk where rows are, and gets its zeros)
  const int end = min(n, begin + size);
  const bool whole = end - begin == n;             // the row is one chunk

  // ---- q: lane (head r16, dims 32 j + 8 g ..), in NQ terms of T; zeros for heads and dims that are none
  vec8 q[NQ][KS];
  float fold = a.scale;
  const long long q_at = b * a.q_b + (h0 + (r16 < rows ? r16 : 0)) * a.q_h;
  const auto is_q = [&](int j) { return r16 < rows && (FULL || 32 * j + 8 * g < d); };
  const auto load_q = [&](const auto* p, auto vec) {
    float f[KS][8];
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      const int off = FULL ? 32 * j + 8 * g : att_q_dim(j, g, d);
      load8<std::remove_cv_t<std::remove_pointer_t<decltype(p)>>, decltype(vec)::value>(p + q_at + off, f[j]);
    }
    if constexpr (EXACT) {
      // the row's largest element to just below 2^UP, so that no term leaves the type's range: for f16 as high as it
      // goes, as what the second term holds of the row's small elements lies near its subnormals
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!is_q(j)) f[j][i] = 0.f;
          top = fmaxf(top, fabsf(f[j][i]));
        }
      top = max_groups(top, lane);
      const int e = top > 0.f && top < __builtin_inff() ? __builtin_amdgcn_frexp_expf(top) - UP : 0;
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
        for (int i = 0; i < 8; ++i) q[0][j][i] = is_q(j) ? static_cast<T>(f[j][i]) : static_cast<T>(0.f);
    }
  };
  const auto load_q_as = [&](const auto* p) {
    if (a.q_vec) load_q(p, std::true_type{});
    else load_q(p, std::false_type{});
  };

  // ---- the wave's tiles: every fourth of the run
  float4_t o[DL];
#pragma unroll
  for (int e = 0; e < DL; ++e) o[e] = float4_t{0.f, 0.f, 0.f, 0.f};
  float m = ATT_LOW, l = 0.f;

  u32x4_t kf[2][KS];
  u32x2_t vf[8][VC];
  const int sstr = static_cast<int>(a.c.slot_stride) * 2;      // bytes
  // the lane's byte offsets within a 16-token half
  const unsigned koff = r16 * sstr + g * 16;
  const unsigned voff = 4 * g * sstr + r16 * DL * 2;
  struct Where {
    int t0;             // the tile's first token
    bool ok[2];         // its halves' pages exist
    long long at[2];    // the halves' element offsets
  };
  // page ids of a tile's halves (a half that begins past the row's end may lie past the table: it is masked, the
  // other half's page serves)
  const auto pages_of = [&](int t0, int (&pg)[2]) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int j = t0 + 16 * hf < n ? t0 + 16 * hf : t0;
      pg[hf] = load_const(a.c.table + b * a.c.table_stride + (j >> a.c.page_shift));
    }
  };
  const auto locate = [&](int t0, const int (&pg)[2]) {
    Where w;
    w.t0 = t0;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int id = __builtin_amdgcn_readfirstlane(pg[hf]);
      w.ok[hf] = static_cast<unsigned>(id) < static_cast<unsigned>(a.c.pages);
      w.at[hf] = a.c.row_at(w.ok[hf] ? id : 0, head, t0 + 16 * hf < n ? t0 + 16 * hf : t0);
    }
    return w;
  };
  const auto load_k = [&](const Where& w) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const char* p = static_cast<const char*>(a.c.k) + 2 * w.at[hf];
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        if (FULL || 32 * j + 8 * g < d) kf[hf][j] = load_once<NT>(reinterpret_cast<const u32x4_t*>(p + koff + 64 * j));
        else kf[hf][j] = u32x4_t{0, 0, 0, 0};
      }
    }
  };
  const auto load_v = [&](const Where& w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const char* p = static_cast<const char*>(a.c.v) + 2 * w.at[i >> 2];
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        if (FULL || r16 * DL + 4 * c < d) vf[i][c] = load_once<NT>(reinterpret_cast<const u32x2_t*>(p + voff + (i & 3) * sstr + 8 * c));
        else vf[i][c] = u32x2_t{0, 0};
      }
    }
  };
  float s[8];
  // S^T = K Q^T
  const auto logits = [&]() {
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
  };
  // the weights against the running maximum, and out^T += V^T P^T
  const auto accumulate = [&](const Where& w) {
    if (w.t0 + ATT_TILE > n || !w.ok[0] || !w.ok[1]) {
      // tokens past the end and on missing pages: no weight, and nothing of what their memory holds
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = w.t0 + 16 * (i >> 2) + 4 * g + (i & 3);
        if (!(j < n && w.ok[i >> 2])) {
          s[i] = -__builtin_inff();
#pragma unroll
          for (int c = 0; c < VC; ++c) vf[i][c] = u32x2_t{0, 0};
        }
      }
    }
    if (a.logits && r16 < rows) {
      float* p = a.logits + (static_cast<long long>(b) * a.hq + h0 + r16) * a.logit_stride + w.t0 + 4 * g;
      *reinterpret_cast<float4_t*>(p) = float4_t{s[0], s[1], s[2], s[3]};
      *reinterpret_cast<float4_t*>(p + 16) = float4_t{s[4], s[5], s[6], s[7]};
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i]);
    if (__any(top - m > TOP + ATT_SLACK)) {
      const float most = max_groups(top, lane);
      float to = fmaxf(m, most - TOP);
      if (most - to > TOP + ATT_SLACK) to = most;   // (of 2^27 and more that difference is rounded, up to 16)
      const float f = exp2f(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int e = 0; e < DL; ++e) o[e] *= f;
    }
    vec8 p[NP];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = __builtin_amdgcn_exp2f(s[i] - m);
      l += x;
#pragma unroll
      for (int t = 0; t < NP; ++t) {
        const T part = static_cast<T>(x);
        p[t][i] = part;
        x -= static_cast<float>(part);
      }
    }
    // a dim pair (one 32-bit word of the 8 tokens' rows) at a time
#pragma unroll
    for (int e = 0; e < DL; e += 2) {
      uint32_t x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (e & 2) ? vf[i][e / 4].y : vf[i][e / 4].x;
      u32x4_t lo, hi;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x05040100u);
        hi[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302u);
      }
#pragma unroll
      for (int t = 0; t < NP; ++t) {
        o[e] = AT::mfma(__builtin_bit_cast(vec8, lo), p[t], o[e]);
        o[e + 1] = AT::mfma(__builtin_bit_cast(vec8, hi), p[t], o[e + 1]);
      }
    }
  };

  // q's loads and the first tile's go out together: q in the cache's type first, as it needs no conversion
  if (t0 + 16 >= n) pg[1] = pg[0];
  if (!EXACT) load_q_as(static_cast<const T*>(a.q));
  if (t0 < end) {
    Where w = locate(t0, pg);
    load_k(w);
    load_v(w);
    if (EXACT) {
      if (a.q_dt == DT_F32) load_q_as(static_cast<const float*>(a.q));
      else if (a.q_dt == DT_F16) load_q_as(static_cast<const _Float16*>(a.q));
      else load_q_as(static_cast<const bf16_t*>(a.q));
    }
    while (true) {
      const int next = t0 + ATT_TILE * ATT_WAVES;
      const bool more = next < end;
      pages_of(more ? next : t0, pg);
      logits();
      accumulate(w);
      if (!more) break;
      t0 = next;
      w = locate(t0, pg);
      load_k(w);
      load_v(w);
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
    if (whole) {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;   // no token (or none on a page that exists)
      if (dim < d) store4_dt(a.out, (bh + row) * d + dim, a.out_dt, acc * inv);
      if (a.total && dim == 0) *reinterpret_cast<float2*>(a.total + 2 * (bh + row)) = make_float2(mx, inv);
    } else {
      const long long at = static_cast<long long>(item) * a.group + rb * 16 + row;
      if (dim < d) *reinterpret_cast<float4_t*>(a.part + at * d + dim) = acc;
      if (dim == 0) *reinterpret_cast<float2*>(a.ml + 2 * at) = make_float2(mx, sum);
    }
  }
}

// The chunks of a (row, key-value head): `used` of them, the i-th at place first + i * heads of the line.
struct Parts {
  int n, used, first, heads;
  __device__ __forceinline__ long long at(int i) const { return first + static_cast<long long>(i) * heads; }
};

__device__ __forceinline__ Parts att_parts(const AttendArgs& a, int b, int head, int lane) {
  if (a.aim == 0) return {a.c.length(b), 1, 0, 0};
  if (a.chunk) {
    const int n = a.c.length(0);
    return {n, (n + a.chunk - 1) / a.chunk, head, a.c.heads};
  }
  const int len0 = att_lengths(a.c, 0, lane);
  const Place at = att_find(a, att_chunk(a, len0, lane), -1, b, len0, lane);
  return {at.n, at.chunks, at.before * a.c.heads + head, a.c.heads};
}

// The parts of one (row, query head) joined: out = sum_i f_i part_i / sum_i f_i sum_i, f_i = 2^(m_i - max).
// A workgroup's threads take the parts' maxima and sums side by side, and the partial sums as (part group, 4
// dims), the first ATT_AHEAD of a thread loaded before the maxima are known. (One thread per dim that walked the
// parts one after another took 48 us for 64 parts of 32 heads; this takes 4.0, and 7.1 for the 2
// to 4 parts each of 64 rows' 32 heads.)
constexpr int ATT_AHEAD = 8;

__device__ __forceinline__ void attend_join(const AttendArgs& a, long long bh) {
  __shared__ float s_f[ATT_PARTS], s_red[2][4];
  __shared__ float4_t s_acc[256];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int b = static_cast<int>(bh / a.hq), qh = static_cast<int>(bh - static_cast<long long>(b) * a.hq), d = a.c.d;
  const int head = qh / a.group, in_group = qh - head * a.group;
  const Parts parts = att_parts(a, b, head, lane);
  const int quads = d / 4, groups = 256 / quads;
  const int grp = tid / quads, dim = (tid - grp * quads) * 4;
  if (parts.used < 2) {
    if (parts.used == 0 && grp == 0) store4_dt(a.out, bh * d + dim, a.out_dt, float4_t{0.f, 0.f, 0.f, 0.f});
    return;
  }
  const int used = parts.used;
  const bool mine = grp < groups;
  const auto part = [&](int i) {
    return *reinterpret_cast<const float4_t*>(a.part + (parts.at(i) * a.group + in_group) * d + dim);
  };
  float4_t ahead[ATT_AHEAD];
#pragma unroll
  for (int i = 0; i < ATT_AHEAD; ++i)
    if (i * groups < used) ahead[i] = part(min(mine ? grp + i * groups : 0, used - 1));
  float m[ATT_PARTS / 256], l[ATT_PARTS / 256], mx = ATT_LOW;
#pragma unroll
  for (int i = 0; i < ATT_PARTS / 256; ++i) {
    const int p = tid + 256 * i;
    m[i] = ATT_LOW;
    l[i] = 0.f;
    if (256 * i >= used) continue;
    float2 v = make_float2(ATT_LOW, 0.f);
    if (p < used) v = reinterpret_cast<const float2*>(a.ml)[parts.at(p) * a.group + in_group];
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
  for (int i = 0; i < ATT_PARTS / 256; ++i) {
    const float f = exp2f(m[i] - mx);
    if (tid + 256 * i < used) s_f[tid + 256 * i] = f;
    sum = __builtin_fmaf(l[i], f, sum);
  }
  sum = wave_sum(sum, lane);
  if (lane == 0) s_red[1][wave] = sum;
  __syncthreads();
  sum = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;   // no token on a page that exists
  float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
  if (mine) {
#pragma unroll
    for (int i = 0; i < ATT_AHEAD; ++i)
      if (grp + i * groups < used) acc += ahead[i] * s_f[grp + i * groups];
    for (int i = grp + ATT_AHEAD * groups; i < used; i += groups) acc += part(i) * s_f[i];
  }
  s_acc[tid] = acc;
  __syncthreads();
  if (grp == 0) {
    for (int i = 1; i < groups; ++i) acc += s_acc[i * quads + tid];
    store4_dt(a.out, bh * d + dim, a.out_dt, acc * inv);
  }
}

// score_j += sum over the key-value head's query heads of p_j, for 256 tokens of a (row, head): each wave first
// joins the maxima and sums of its share of the query heads.
__device__ __forceinline__ void attend_score(const AttendArgs& a, int id) {
  __shared__ float s_m[64], s_inv[64];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int per = a.c.rows * a.c.heads, block = id / per, at = id - block * per;
  const int b = at / a.c.heads, head = at - b * a.c.heads;
  const Parts parts = att_parts(a, b, head, lane);
  const int n = parts.n, j = block * 256 + tid;
  if (block * 256 >= n) return;
  const long long bh0 = static_cast<long long>(b) * a.hq + head * a.group;
  const float* logits = a.logits + bh0 * a.logit_stride + j;
  float sum = 0.f;
  for (int g0 = 0; g0 < a.group; g0 += 64) {
    const int some = min(64, a.group - g0);
    for (int i = wave; i < some; i += 4) {
      float mx = ATT_LOW, inv;
      if (parts.used == 1) {
        const float2 v = reinterpret_cast<const float2*>(a.total)[bh0 + g0 + i];
        mx = v.x;
        inv = v.y;
      } else {
        const auto ml = [&](int p) { return reinterpret_cast<const float2*>(a.ml)[parts.at(p) * a.group + g0 + i]; };
        for (int p = lane; p < parts.used; p += 64) mx = fmaxf(mx, ml(p).x);
        mx = wave_max(mx, lane);
        float total = 0.f;
        for (int p = lane; p < parts.used; p += 64) {
          const float2 v = ml(p);
          total = __builtin_fmaf(v.y, exp2f(v.x - mx), total);
        }
        total = wave_sum(total, lane);
        inv = total == 0.f ? 0.f : 1.0f / total;
      }
      if (lane == 0) {
        s_m[i] = mx;
        s_inv[i] = inv;
      }
    }
    __syncthreads();
    if (j < n)
#pragma unroll 4
      for (int i = 0; i < some; ++i) sum += exp2f(logits[(g0 + i) * a.logit_stride] - s_m[i]) * s_inv[i];
    __syncthreads();
  }
  if (j >= n) return;
  const int page = a.c.page_of(b, j);
  if (page >= 0) a.c.scores[a.c.slot_at(page, head, j)] += sum;
}

// The workgroups of the join, then those of the scores.
__global__ __launch_bounds__(256) void attend_finish_kernel(AttendArgs a, int joins) {
  if (static_cast<int>(blockIdx.x) < joins) attend_join(a, blockIdx.x);
  else attend_score(a, blockIdx.x - joins);
}

}  // namespace trellis
