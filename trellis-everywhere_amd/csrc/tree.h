// tree.h — attention of several new tokens per row over a paged key-value cache. Row b's n newest tokens lie in its last n
// slots, base = length - n; the i-th of them sees the slots below base, itself and its ancestors:
//   out_i = sum_j p_ij v_j,  p_i = softmax over the j it sees of scale q_i . k_j,
// its parent being parents[i] (a token before it; anything else: none), or (no parents) the token before it, so that it
// sees all up to itself: a prompt, or part of one. A token that sees nothing gives zeros.
//
// A workgroup takes a chunk of one (row, key-value head)'s keys and a block of its queries (token by token, a token's
// query heads side by side): WR of its four waves take 32 queries each, and 4 / WR share their keys. Keys and values
// come tile by tile into LDS (16-byte loads straight there, the next tile's under way while one is used), rows of 16-byte
// pieces in an order that keeps the reads apart:
//   * S^T = K Q^T by v_mfma_f32_32x32x16: the A operand's lane (token l % 32, dims 8 (l / 32) ..) is 16 bytes of a key's row;
//     the B operand, 32 queries, stays in registers;
//   * the result has lane (query l % 32, tokens 8 (r / 4) + 4 (l / 32) + r % 4), which is the B operand P^T of
//     out^T = V^T P^T if lane half h counts the tokens {4h + 0..3, 8 + 4h + 0..3} of 16 as its k-slots;
//   * V^T, the A operand, is then 4 consecutive tokens of one dim twice: a transposing read of LDS (ds_read_b64_tr_b16);
//   * both products leave the query on l % 32: the running maximum and the sum are per-lane values, and the maximum that
//     the weights are taken against moves only when a logit passes it by 2^4, as in attend.h.
// Tiles go downwards, so that a lane walks its query's ancestors once, from itself to the first, a word of 32 tokens at a
// time; only tiles with a new token, a missing page or the row's end are masked.
// The chunks' results (maximum, sum, unnormalised out) meet in tree_join_kernel, in a fixed order.
// Precision: the sums are fp32. The weights enter their product as in attend.h, but once rounded to the cache's type (half
// a step of it, as out's own rounding) where the products bound the call: blocks of 128 queries of 16-bit types.
#pragma once

#include "tree_rows.h"

namespace trellis {

typedef float float16_t __attribute__((ext_vector_type(16)));
typedef short short4_t __attribute__((ext_vector_type(4)));

template <class T> struct TreeType;
template <> struct TreeType<_Float16> {
  typedef _Float16 vec8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float16_t mfma(vec8 a, vec8 b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct TreeType<bf16_t> {
  typedef __bf16 vec8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float16_t mfma(vec8 a, vec8 b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// Zeros for those of 64 tokens that no row has.
__device__ __forceinline__ void tree_none(const TreeArgs& a, int z, int lane) {
  const int t = z * 64 + lane;
  bool has = t >= a.tokens;
  for (int s = 0; s < a.c.rows; s += 64) {
    const TreeRow r = tree_row(a, s + lane);
    for (int l = 0; l < min(64, a.c.rows - s); ++l) {
      const int first = __builtin_amdgcn_readlane(r.first, l), n = __builtin_amdgcn_readlane(r.n, l);
      has = has || (t >= first && t - first < n);
    }
  }
  unsigned long long rest = __ballot(!has);
  const long long each = static_cast<long long>(a.hq) * a.c.d;
  while (rest) {
    const int l = __builtin_ctzll(rest);
    rest &= rest - 1;
    for (long long e = 4 * threadIdx.x; e < each; e += 4 * 256)
      store4_dt(a.out, (z * 64 + l) * each + e, a.out_dt, float4_t{0.f, 0.f, 0.f, 0.f});
  }
}

// Workgroups that a CU's registers have to hold.
constexpr int tree_residents(int dp, int wr, bool exact) { return wr == 4 && dp <= 128 && !exact ? 2 : 1; }

// T: the cache's type. DP: head dims padded to 64, 128 or 256; FULL: d == DP. EXACT: q or out is of another type than the
// cache's. WR: waves with queries of their own.
template <class T, int DP, bool FULL, bool EXACT, int WR>
__global__ __launch_bounds__(256, tree_residents(DP, WR, EXACT)) void tree_kernel(TreeArgs a) {
  typedef TreeType<T> AT;
  typedef typename AT::vec8 vec8;
  constexpr bool BF = !std::is_same<T, _Float16>::value;
  constexpr int NQ = EXACT ? (BF ? 3 : 2) : 1;            // terms of q
  constexpr int NP = EXACT ? (BF ? 3 : 2) : WR == 4 ? 1 : 2;   // terms of the weights
  constexpr int UP = BF ? 0 : 15;                         // log2 that q's largest element stays below
  constexpr float TOP = BF ? 0.f : ATT_TOP;
  constexpr int WT = 4 / WR, QR = 32 * WR;
  constexpr int NB = WR == 4 && DP <= 128 && !EXACT ? 2 : 1;   // times 32 tokens a wave and tile
  constexpr int TT = 32 * WT * NB;                        // tokens of a tile
  constexpr int KS = DP / 16, EB = DP / 32;               // k-steps of the first product, blocks of dims of the second
  constexpr int CH = DP / 8, ROW = 2 * DP;                // 16-byte pieces and bytes of a row
  constexpr int PLANE = TT * ROW, STAGE = 2 * PLANE;
  constexpr int UNITS = TT / 32;                          // loads of 16 rows of keys or values a wave and tile
  constexpr int OP = DP + 4;                              // floats of a row where waves meet
  static_assert(WR == 4 || (WT - 1) * WR * 32 * (OP + 2) * 4 <= 2 * STAGE, "the waves' sums fit the tiles' memory");
  __shared__ __align__(1024) char s_kv[2 * STAGE];
  __shared__ __align__(8) uint8_t s_ok[2][8];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c32 = lane & 31, h = lane >> 5;
  const int rw = wave / WT, tw = wave % WT;
  if (static_cast<int>(blockIdx.x) >= a.items) {
    tree_none(a, blockIdx.x - a.items, lane);
    return;
  }
  const int item = blockIdx.x, pos = uniform(item / a.c.heads), head = uniform(item - pos * a.c.heads);
  const TreePlace at = tree_find(a, QR, pos, 0, lane);
  const int b = uniform(at.b);
  if (b < 0) return;
  const TreeRow row = tree_row(a, b);
  const int off = uniform(pos - at.before), chunk = uniform(off / at.blocks), block = uniform(at.blocks - 1 - (off - chunk * at.blocks));
  const int stop = uniform(tree_end(row, block, QR, a.group));
  const int size = a.aim ? at.units * TREE_UNIT : 0x7fffffff;
  const int begin = uniform(a.aim ? chunk * size : 0), end = uniform(min(stop, a.aim ? begin + size : stop));
  if (begin > 0 && begin >= stop) return;
  const bool whole = stop <= size;
  const int d = a.c.d, queries = row.n * a.group;

  // ---- the lane's query
  const int qi = block * QR + 32 * rw + c32;              // of the row's
  const bool is = qi < queries;
  const int token = is ? qi / a.group : 0, qh = head * a.group + (is ? qi - token * a.group : 0);
  const bool active = block * QR + 32 * rw < queries;     // the wave has queries
  const bool fine = is && row.base + token >= 0 && row.base + token < row.len;
  // slots below `plain` are seen by all of the wave's queries
  const int tok0 = (block * QR + 32 * rw) / a.group, tok1 = min(row.n - 1, (block * QR + 32 * rw + 31) / a.group);
  const int plain = uniform(row.base + tok0 < 0 || row.base + tok1 >= row.len ? -1 : a.parents ? row.base : row.base + tok0 + 1);
  const int below = a.parents ? row.base : row.base + token + 1;   // slots that the lane's query sees all of
  int walk = a.parents && fine ? token : -1;              // the ancestor that comes next

  // ---- tiles into LDS
  const int sstr = static_cast<int>(a.c.slot_stride) * 2;   // bytes
  const unsigned lds = lds_addr(s_kv);
  constexpr int PER = 64 / CH;                            // rows of one load of a wave
  const int lr = lane / CH, lp = lane % CH;
  const auto piece_k = [](int r) { return CH == 8 ? (r >> 1) & 7 : r & 15; };
  const auto piece_v = [](int r) { return CH == 8 ? 4 * ((r >> 1) & 1) : 4 * (r & 3); };
  const auto pages_of = [&](int t0, int (&pg)[UNITS]) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int j = t0 + 16 * ((wave * UNITS + u) >> 1);
      pg[u] = load_const(a.c.table + b * a.c.table_stride + (min(j, row.len - 1) >> a.c.page_shift));
    }
  };
  const auto load_tile = [&](int t0, int buf, const int (&pg)[UNITS]) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int id = wave * UNITS + u, g16 = id >> 1, kv = id & 1, j = t0 + 16 * g16;
      const int page = __builtin_amdgcn_readfirstlane(pg[u]);
      const bool ok = static_cast<unsigned>(page) < static_cast<unsigned>(a.c.pages) && j < row.len;
      const long long at16 = a.c.row_at(ok ? page : 0, head, j);
      const rsrc_t r = make_rsrc(static_cast<const char*>(kv ? a.c.v : a.c.k) + 2 * at16, ok ? 16 * static_cast<unsigned>(sstr) : 0);
      const unsigned to = lds + buf * STAGE + kv * PLANE + g16 * 16 * ROW;
#pragma unroll
      for (int m = 0; m < 16 / PER; ++m) {
        const int rr = m * PER + lr, piece = lp ^ (kv ? piece_v(rr) : piece_k(rr));
        unsigned voff = rr * sstr + 16 * piece;
        if ((!FULL && 8 * piece >= d) || j + rr >= row.len) voff = RSRC_PAST;
        load_lds16<false>(r, to + m * 1024, voff);
      }
      if (kv == 0 && lane == 0) s_ok[buf][g16] = ok;
    }
  };

  const int tiles = end > begin ? (end - begin + TT - 1) / TT : 0;
  int pg[UNITS];
  if (tiles > 0) pages_of(begin + (tiles - 1) * TT, pg);

  // ---- q: lane (query c32, dims 16 j + 8 h ..), in NQ terms of T; zeros for queries and dims that are none
  vec8 q[NQ][KS];
  float fold = fabsf(a.scale);
  const float sign = a.scale < 0.f ? -1.f : 1.f;
  const long long q_at = static_cast<long long>(row.first + token) * a.q_t + qh * a.q_h;
  const auto is_q = [&](int j) { return is && (FULL || 16 * j + 8 * h < d); };
  const auto load_q = [&](const auto* p, auto vec) {
    float f[KS][8];
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      const int o = FULL || 16 * j + 8 * h < d ? 16 * j + 8 * h : d - 8;
      load8<std::remove_cv_t<std::remove_pointer_t<decltype(p)>>, decltype(vec)::value>(p + q_at + o, f[j]);
    }
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) f[j][i] = is_q(j) ? f[j][i] * sign : 0.f;
    if constexpr (EXACT) {
      // the query's largest element to just below 2^UP (attend.h)
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[j][i]));
      top = fmaxf(top, lane_xor<32>(top, lane));
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
        for (int i = 0; i < 8; ++i) q[0][j][i] = static_cast<T>(f[j][i]);
    }
  };
  const auto load_q_as = [&](const auto* p) {
    if (a.q_vec) load_q(p, std::true_type{});
    else load_q(p, std::false_type{});
  };
  if (a.q_dt == DT_F32) load_q_as(static_cast<const float*>(a.q));
  else if (a.q_dt == DT_F16) load_q_as(static_cast<const _Float16*>(a.q));
  else load_q_as(static_cast<const bf16_t*>(a.q));
  fold = fmaxf(fold, 1.17549435e-38f);   // (above 0: a masked logit is -inf before it)

  float16_t o[EB];
#pragma unroll
  for (int e = 0; e < EB; ++e) o[e] = float16_t{};
  float m = ATT_LOW, l = 0.f;

  // the lane's places in a tile: of keys (token c32), and of values (4 tokens of 16 dims a group of 16 lanes)
  const int kx = (h ^ piece_k(c32 & 15)) * 16, krow = c32 * ROW;
  const int l16 = lane & 15, vrow = (4 * h + (l16 >> 2)) * ROW;
  const int vx = piece_v(4 * h + (l16 >> 2)) * 16, vcol = 32 * ((lane >> 4) & 1) + 8 * (l16 & 3);

  const auto use_tile = [&](int t0, int buf) {
    const char* kp = s_kv + buf * STAGE + tw * NB * 32 * ROW;
    const char* vp = kp + PLANE;
    // S^T = K Q^T
    float16_t s[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      s[nb] = float16_t{};
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const vec8 k = *reinterpret_cast<const vec8*>(kp + nb * 32 * ROW + krow + ((32 * j) ^ kx));
#pragma unroll
        for (int t = 0; t < NQ; ++t) s[nb] = AT::mfma(k, q[t][j], s[nb]);
      }
    }
    // what the queries see
    const unsigned long long okay = *reinterpret_cast<const unsigned long long*>(s_ok[buf]);
    const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(okay)), hi = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(okay >> 32));
    const int j0 = t0 + tw * NB * 32;
    if (j0 + 32 * NB > plain || (TT > 64 ? (lo & hi) : TT > 32 ? lo : (lo & 0xFFFFu) | 0x01010000u) != 0x01010101u) {
#pragma unroll
      for (int nb = NB - 1; nb >= 0; --nb) {
        const int j = j0 + 32 * nb, g16 = 2 * (tw * NB + nb);
        const int k = below - j;
        unsigned sees = k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1;
        const int rel = j - row.base;
        while (walk >= 0 && walk >= rel) {
          if (walk - rel < 32) sees |= 1u << (walk - rel);
          const int p = a.parents[row.first + walk];
          walk = p >= 0 && p < walk ? p : -1;
        }
        if (!fine) sees = 0;
        const unsigned flags = (g16 < 4 ? lo : hi) >> (8 * (g16 & 3));
        if (!(flags & 1)) sees &= 0xFFFF0000u;
        if (!(flags & 0x100)) sees &= 0x0000FFFFu;
        sees >>= 4 * h;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[nb][r] = (sees >> (8 * (r / 4) + r % 4)) & 1 ? s[nb][r] : -__builtin_inff();
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[nb][r]);
    top *= fold;
    if (__any(top - m > TOP + ATT_SLACK)) {
      const float most = fmaxf(top, lane_xor<32>(top, lane));
      // (only a query whose own logit has passed moves: its result goes by its row alone)
      float to = most - m > TOP + ATT_SLACK ? most - TOP : m;
      if (most - to > TOP + ATT_SLACK) to = most;   // (of 2^27 and more that difference is rounded, up to 16)
      const float by = exp2f(m - to);
      m = to;
      l *= by;
#pragma unroll
      for (int e = 0; e < EB; ++e) o[e] *= by;
    }
    // the weights, and out^T += V^T P^T
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        vec8 p[NP];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nb][8 * u + i], fold, -m));
          l += x;
#pragma unroll
          for (int t = 0; t < NP; ++t) {
            const T part = static_cast<T>(x);
            p[t][i] = part;
            if (t + 1 < NP) x -= static_cast<float>(part);
          }
        }
        const char* at16 = vp + (nb * 32 + 16 * u) * ROW + vrow + vcol;
#pragma unroll
        for (int e = 0; e < EB; ++e) {
          typedef __attribute__((address_space(3))) short4_t* lds4_t;
          const char* v4 = at16 + ((64 * e) ^ vx);
          const short4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(v4));
          const short4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(v4 + 8 * ROW));
          const vec8 v = __builtin_bit_cast(vec8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int t = 0; t < NP; ++t) o[e] = AT::mfma(v, p[t], o[e]);
        }
      }
  };

  // (the barrier: the tile has arrived for every wave, and none still reads the one whose place the next one takes)
  const auto arrive = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  if (tiles > 0) {
    int t = tiles - 1, buf = 0;
    load_tile(begin + t * TT, 0, pg);
    if (t > 0) pages_of(begin + (t - 1) * TT, pg);
    for (; t >= 0; --t, buf ^= 1) {
      arrive();
      if (t > 0) load_tile(begin + (t - 1) * TT, buf ^ 1, pg);
      if (t > 1) pages_of(begin + (t - 2) * TT, pg);
      if (active) use_tile(begin + t * TT, buf);
    }
  }
  l += lane_xor<32>(l, lane);

  // ---- the results of waves that share their queries meet
  if constexpr (WT > 1) {
    lds_barrier();
    float* meet = reinterpret_cast<float*>(s_kv);
    const auto place = [&](int w) { return meet + ((rw * (WT - 1) + w - 1) * 32 + c32) * OP; };
    float* ml = meet + (WT - 1) * WR * 32 * OP;
    if (tw > 0) {
      float* to = place(tw);
#pragma unroll
      for (int e = 0; e < EB; ++e)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          *reinterpret_cast<float4_t*>(to + 32 * e + 2 * r + 4 * h) = float4_t{o[e][r], o[e][r + 1], o[e][r + 2], o[e][r + 3]};
      if (h == 0) *reinterpret_cast<float2*>(ml + 2 * ((rw * (WT - 1) + tw - 1) * 32 + c32)) = make_float2(m, l);
    }
    lds_barrier();
    if (tw > 0) return;
    float mx = m, ms[WT - 1], ls[WT - 1];
#pragma unroll
    for (int w = 1; w < WT; ++w) {
      const float2 v = *reinterpret_cast<const float2*>(ml + 2 * ((rw * (WT - 1) + w - 1) * 32 + c32));
      ms[w - 1] = v.x;
      ls[w - 1] = v.y;
      mx = fmaxf(mx, v.x);
    }
    const float by = exp2f(m - mx);
    l *= by;
#pragma unroll
    for (int e = 0; e < EB; ++e) o[e] *= by;
#pragma unroll
    for (int w = 1; w < WT; ++w) {
      const float f = exp2f(ms[w - 1] - mx);
      l = __builtin_fmaf(ls[w - 1], f, l);
      const float* from = place(w);
#pragma unroll
      for (int e = 0; e < EB; ++e)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const float4_t v = *reinterpret_cast<const float4_t*>(from + 32 * e + 2 * r + 4 * h);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[e][r + i] = __builtin_fmaf(v[i], f, o[e][r + i]);
        }
    }
    m = mx;
  }
  if (!is) return;
  if (whole) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const long long to = (static_cast<long long>(row.first + token) * a.hq + qh) * d;
#pragma unroll
    for (int e = 0; e < EB; ++e)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int dim = 32 * e + 2 * r + 4 * h;
        if (FULL || dim < d) store4_dt(a.out, to + dim, a.out_dt, float4_t{o[e][r], o[e][r + 1], o[e][r + 2], o[e][r + 3]} * inv);
      }
  } else {
    const long long to = static_cast<long long>(item) * QR + 32 * rw + c32;
#pragma unroll
    for (int e = 0; e < EB; ++e)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int dim = 32 * e + 2 * r + 4 * h;
        if (FULL || dim < d)
          *reinterpret_cast<float4_t*>(a.part + to * d + dim) = float4_t{o[e][r], o[e][r + 1], o[e][r + 2], o[e][r + 3]};
      }
    if (h == 0) *reinterpret_cast<float2*>(a.ml + 2 * to) = make_float2(m, l);
  }
}

// ---- the host's side: the kernel for a call, one cache type a translation unit (tree_f16.hip, tree_bf16.hip)
struct TreeLaunch {
  TreeArgs a;
  bool exact;
  int waves;
  unsigned grid;
  hipStream_t stream;
};

void launch_tree_f16(const TreeLaunch& l);
void launch_tree_bf16(const TreeLaunch& l);

template <class T, int DP, bool FULL, bool EXACT>
void launch_tree_waves(const TreeLaunch& l) {
  if (l.waves == 4) hipLaunchKernelGGL((tree_kernel<T, DP, FULL, EXACT, 4>), dim3(l.grid), dim3(256), 0, l.stream, l.a);
  else if (l.waves == 2) hipLaunchKernelGGL((tree_kernel<T, DP, FULL, EXACT, 2>), dim3(l.grid), dim3(256), 0, l.stream, l.a);
  else if constexpr (DP < 256) hipLaunchKernelGGL((tree_kernel<T, DP, FULL, EXACT, 1>), dim3(l.grid), dim3(256), 0, l.stream, l.a);
}

template <class T, int DP>
void launch_tree_dp(const TreeLaunch& l) {
  if (l.a.c.d == DP) {
    if (l.exact) launch_tree_waves<T, DP, true, true>(l);
    else launch_tree_waves<T, DP, true, false>(l);
  } else {
    if (l.exact) launch_tree_waves<T, DP, false, true>(l);
    else launch_tree_waves<T, DP, false, false>(l);
  }
}

template <class T>
void launch_tree(const TreeLaunch& l) {
  if (l.a.c.d <= 64) launch_tree_dp<T, 64>(l);
  else if (l.a.c.d <= 128) launch_tree_dp<T, 128>(l);
  else launch_tree_dp<T, 256>(l);
}

}  // namespace trellis
