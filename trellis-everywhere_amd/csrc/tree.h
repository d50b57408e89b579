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
// time; only tiles with a new token, a missing page or the row's end are masked. The walk is a chain of loads: a line of 128
// tokens costs a call 9 to 11 us more than no parents at all, one of 512 43.
// The chunks' results (maximum, sum, unnormalised out) meet in tree_join_kernel, in a fixed order.
// Precision: the sums are fp32. Where q, cache and out are of one 16-bit type (not EXACT) the weights are rounded once to
// it, half a step, as out is itself: the error against float64 (rms) is 1.1 (rows of thousands of tokens in f16) to 1.3 times
// (bf16, 1024 tokens behind 8192) that of a result rounded once, and the terms that attend.h takes would be two or three times
// the second product's instructions. Other types take those terms, of q too: 1024 fp32 queries behind 8192 f16 tokens 366 us,
// bf16 ones 457, for the 170 of 16-bit types. The sums are of weights up to 2^15 (f16) or 2^4 (bf16): bf16 values of 2^124 /
// tokens and more in size can overflow them.
// Bound: new tokens of few queries a key (32 rows of up to 8192 tokens, up to 26 new each, 32 heads over 8 of 128) by
// memory: 107-112 us, 4.9 TB/s and 13 MiB of partial sums. Many by the loop's own latencies: 1024 tokens behind 8192
// 160-177 us, 870 TFLOP/s, the matrix cores busy 48 % of the time and the vector units 44 %; LDS has no conflicts (heads of 64
// 104 us, of 80 and 96, which take the products of 128, 150 and 158, of 192 and 256 390). The waves
// of a SIMD, two, are all that fills one's waits: taken out one by one (of 185 us) the exponentials are worth 17, the second
// product 38, the loads into LDS 36, the maximum 4. Small calls by the chain plan, length, page, keys, weights, values: 7 tokens
// behind 149 9.8 us.
// 32 queries a wave: of 16 (16x16x32) each key read from LDS would serve half as many, and LDS would bound the loop. 64
// tokens a step: with 32 and three workgroups a CU 1024 tokens behind 8192 took 192-201 us instead of 177.
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

// Blocks of 32 tokens a wave and step (two slots of their keys and values have to fit LDS), and workgroups that a CU's
// registers hold.
constexpr int tree_wide(int dp, bool exact) { return dp > 128 && exact ? 1 : 2; }
constexpr int tree_residents(int dp, bool exact) { return dp > 128 || exact ? 1 : 2; }

// T: the cache's type. DP: head dims padded to 64, 128 or 256; FULL: d == DP. EXACT: q or out is of another type than the
// cache's.
template <class T, int DP, bool FULL, bool EXACT>
__global__ __launch_bounds__(256, tree_residents(DP, EXACT)) void tree_kernel(TreeArgs a) {
  typedef TreeType<T> AT;
  typedef typename AT::vec8 vec8;
  constexpr bool BF = !std::is_same<T, _Float16>::value;
  constexpr int NQ = EXACT ? (BF ? 3 : 2) : 1;            // terms of q
  constexpr int NP = EXACT ? (BF ? 3 : 2) : 1;            // terms of the weights
  constexpr int UP = BF ? 0 : 15;                         // log2 that q's largest element stays below
  constexpr float TOP = BF ? 0.f : ATT_TOP;
  constexpr int WR = tree_waves(EXACT), WT = 4 / WR, QR = 32 * WR;
  constexpr int NB = tree_wide(DP, EXACT);                // times 32 tokens a wave and step
  constexpr int BT = 32 * WT * NB;                        // tokens of a step
  constexpr int KS = DP / 16, EB = DP / 32;               // k-steps of the first product, blocks of dims of the second
  constexpr int CH = DP / 8, ROW = 2 * DP;                // 16-byte pieces and bytes of a row
  constexpr int SLOT = BT * ROW;                          // bytes of a step's keys, and of its values: two slots of each
  constexpr int PER = 64 / CH;                            // rows of one load of a wave
  constexpr int OWN = BT / 4, GROUPS = OWN / 16;          // rows that a wave loads a step, and their 16-row groups
  constexpr int OP = DP + 4;                              // floats of a row where waves meet
  static_assert(OWN % 16 == 0, "a wave loads whole groups: a group's flag has one writer");
  static_assert(WR == 4 || (WT - 1) * WR * 32 * (OP + 2) * 4 <= 4 * SLOT, "the waves' sums fit the slots' memory");
  __shared__ __align__(1024) char s_kv[4 * SLOT];
  __shared__ __align__(8) uint8_t s_ok[2][8];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c32 = lane & 31, h = lane >> 5;
  const int rw = wave / WT, tw = wave % WT;
  if (static_cast<int>(blockIdx.x) >= a.items) {
    tree_none(a, blockIdx.x - a.items, lane);
    return;
  }
  const int item = blockIdx.x, pos = uniform(item / a.c.heads), head = uniform(item - pos * a.c.heads);
  const TreePlace at = tree_find(a, QR, pos, lane);
  const int b = uniform(at.b);
  if (b < 0) {
    if (a.aim && item == 0 && threadIdx.x == 0) a.done[0].live = 0;   // no row has a token
    return;
  }
  const TreeRow read = tree_row(a, b), row = {uniform(read.first), uniform(read.n), uniform(read.base), uniform(read.len)};
  const int off = uniform(pos - at.before), chunk = uniform(off / at.blocks), block = uniform(at.blocks - 1 - (off - chunk * at.blocks));
  const int stop = uniform(tree_end(row, block, QR, a.group));
  const int size = a.aim ? at.units * TREE_UNIT : 0x7fffffff;
  const int begin = uniform(a.aim ? chunk * size : 0), end = uniform(min(stop, a.aim ? begin + size : stop));
  if (a.aim && head == 0 && threadIdx.x == 0) {
    if (chunk == 0) {
      const int live = (stop + size - 1) / size;
      a.done[1 + at.skipped + block] = {live, at.before + at.blocks - 1 - block, at.blocks, row.first, row.n * a.group, block};
    }
    if (item == 0) a.done[0].live = at.all;
  }
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

  // ---- keys and values into LDS, blocks going downwards, the next one's while one is used. A wave loads OWN rows of each, in
  // 16-row groups that lie in one page each.
  const int sstr = static_cast<int>(a.c.slot_stride) * 2;   // bytes
  const unsigned lds = lds_addr(s_kv);
  const auto piece_k = [](int r) { return CH == 8 ? (r >> 1) & 7 : r & 15; };
  const auto piece_v = [](int r) { return CH == 8 ? 4 * ((r >> 1) & 1) : 4 * (r & 3); };
  constexpr int TIMES = 16 / PER;                            // loads of a group
  const int group0 = wave * OWN;
  unsigned koff[TIMES], voff[TIMES];                         // the lane's places within a group
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    const int r = t * PER + lane / CH, pk = lane % CH ^ piece_k(r), pv = lane % CH ^ piece_v(r);
    koff[t] = FULL || 8 * pk < d ? r * sstr + 16 * pk : RSRC_PAST;
    voff[t] = FULL || 8 * pv < d ? r * sstr + 16 * pv : RSRC_PAST;
  }
  const int steps = uniform(end > begin ? (end - begin + BT - 1) / BT : 0);
  const auto block_at = [&](int i) { return begin + (steps - 1 - i) * BT; };
  const auto flat = [](uintptr_t p) {   // into scalar registers
    return static_cast<uintptr_t>(static_cast<unsigned>(uniform(static_cast<int>(p >> 32)))) << 32 |
           static_cast<unsigned>(uniform(static_cast<int>(p)));
  };
  const uintptr_t k_base = flat(reinterpret_cast<uintptr_t>(a.c.k) + 2 * head * a.c.head_stride);
  const uintptr_t v_base = flat(reinterpret_cast<uintptr_t>(a.c.v) + 2 * head * a.c.head_stride);
  const int32_t* pages = a.c.table + b * a.c.table_stride;
  int page[GROUPS];                     // of the next block to load
  const auto pages_of = [&](int i) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
      page[g] = load_const(pages + (min(block_at(i) + group0 + 16 * g, row.len - 1) >> a.c.page_shift));
  };
  // block i, whose pages are known, into the slots `place`
  const auto load_block = [&](int i, int place) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int j = block_at(i) + group0 + 16 * g, id = uniform(page[g]);
      const bool ok = static_cast<unsigned>(id) < static_cast<unsigned>(a.c.pages) && j < row.len;
      const long long at = ok ? 2 * (id * a.c.page_stride + a.c.in_page(j) * static_cast<int>(a.c.slot_stride)) : 0;
      // (past the row's end, and without a page, zeros)
      const int bytes = uniform(ok ? min(16, row.len - j) * sstr : 0);
      const rsrc_t k = make_rsrc(reinterpret_cast<const void*>(flat(k_base + at)), bytes);
      const rsrc_t v = make_rsrc(reinterpret_cast<const void*>(flat(v_base + at)), bytes);
      const unsigned to = lds + place * SLOT + (group0 + 16 * g) * ROW;
#pragma unroll
      for (int t = 0; t < TIMES; ++t) load_lds16<false>(k, uniform(to + t * 1024), koff[t]);
#pragma unroll
      for (int t = 0; t < TIMES; ++t) load_lds16<false>(v, uniform(to + 2 * SLOT + t * 1024), voff[t]);
      if (lane == 0) s_ok[place][group0 / 16 + g] = ok;
    }
  };
  if (steps > 0) pages_of(0);

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

  struct Logits {
    float16_t v[NB];
  };
  // (place: the block's slot)
  // S^T = K Q^T of a block
  const auto logits = [&](int place) {
    const char* kp = s_kv + place * SLOT + tw * NB * 32 * ROW + krow;
    Logits r;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      r.v[nb] = float16_t{};
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const vec8 k = *reinterpret_cast<const vec8*>(kp + nb * 32 * ROW + ((32 * j) ^ kx));
#pragma unroll
        for (int t = 0; t < NQ; ++t) r.v[nb] = AT::mfma(k, q[t][j], r.v[nb]);
      }
    }
    return r;
  };
  // what the queries see of it, and the maximum
  const auto settle = [&](Logits& s, int i, int place) {
    const unsigned flags = uniform(NB == 2 ? *reinterpret_cast<const int*>(s_ok[place] + 4 * tw) : *reinterpret_cast<const uint16_t*>(s_ok[place] + 2 * tw));
    const int j0 = block_at(i) + 32 * NB * tw;
    if (j0 + 32 * NB > plain || flags != (NB == 2 ? 0x01010101u : 0x0101u)) {
#pragma unroll
      for (int nb = NB - 1; nb >= 0; --nb) {
        const int j = j0 + 32 * nb, k = below - j;
        unsigned sees = k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1;
        const int rel = j - row.base;
        while (walk >= 0 && walk >= rel) {
          if (walk - rel < 32) sees |= 1u << (walk - rel);
          const int p = a.parents[row.first + walk];
          walk = p >= 0 && p < walk ? p : -1;
        }
        if (!fine) sees = 0;
        if (!(flags >> 16 * nb & 1)) sees &= 0xFFFF0000u;
        if (!(flags >> 16 * nb & 0x100)) sees &= 0x0000FFFFu;
        sees >>= 4 * h;
#pragma unroll
        for (int r = 0; r < 16; ++r) s.v[nb][r] = (sees >> (8 * (r / 4) + r % 4)) & 1 ? s.v[nb][r] : -__builtin_inff();
      }
    }
    float top = s.v[0][0];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s.v[nb][r]);
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
  };
  // the weights of a block, and out^T += V^T P^T
  const auto accumulate = [&](const Logits& s, int place) {
    const char* vp = s_kv + (2 + place) * SLOT + tw * NB * 32 * ROW + vrow + vcol;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        vec8 p[NP];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s.v[nb][8 * u + r], fold, -m));
          l += x;
#pragma unroll
          for (int t = 0; t < NP; ++t) {
            const T part = static_cast<T>(x);
            p[t][r] = part;
            if (t + 1 < NP) x -= static_cast<float>(part);
          }
        }
#pragma unroll
        for (int e = 0; e < EB; ++e) {
          typedef __attribute__((address_space(3))) short4_t* lds4_t;
          const char* v4 = vp + (nb * 32 + 16 * u) * ROW + ((64 * e) ^ vx);
          const short4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(v4));
          const short4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(v4 + 8 * ROW));
          const vec8 v = __builtin_bit_cast(vec8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int t = 0; t < NP; ++t) o[e] = AT::mfma(v, p[t], o[e]);
        }
      }
  };

  if (steps > 0) {
    load_block(0, 0);
    if (steps > 1) pages_of(1);
    int i = 0;
    while (true) {
#pragma unroll
      for (int place = 0; place < 2; ++place) {
        if (i >= steps) break;
        // the block has arrived, for every wave, and none still reads the one whose place the next one takes
        wait_vmcnt<0>();
        lds_barrier();
        if (i + 1 < steps) load_block(i + 1, 1 - place);
        if (i + 2 < steps) pages_of(i + 2);
        if (active) {
          Logits s = logits(place);
          settle(s, i, place);
          // (the waves of a SIMD drift apart then, so that one's exponentials meet another's products: a call of 1024 tokens
          // behind 8192 172.7 -> 163.1 us, of five prompts of 6007 tokens in all 105.9 -> 102.1; less with the logits too)
          __builtin_amdgcn_s_setprio(1);
          accumulate(s, place);
          __builtin_amdgcn_s_setprio(0);
        }
        ++i;
      }
      if (i >= steps) break;
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
  unsigned grid;
  hipStream_t stream;
};

void launch_tree_f16(const TreeLaunch& l);
void launch_tree_bf16(const TreeLaunch& l);

template <class T, int DP, bool FULL, bool EXACT>
void launch_tree_as(const TreeLaunch& l) {
  hipLaunchKernelGGL((tree_kernel<T, DP, FULL, EXACT>), dim3(l.grid), dim3(256), 0, l.stream, l.a);
}

template <class T, int DP>
void launch_tree_dp(const TreeLaunch& l) {
  if (l.a.c.d == DP) {
    if (l.exact) launch_tree_as<T, DP, true, true>(l);
    else launch_tree_as<T, DP, true, false>(l);
  } else {
    if (l.exact) launch_tree_as<T, DP, false, true>(l);
    else launch_tree_as<T, DP, false, false>(l);
  }
}

template <class T>
void launch_tree(const TreeLaunch& l) {
  if (l.a.c.d <= 64) launch_tree_dp<T, 64>(l);
  else if (l.a.c.d <= 128) launch_tree_dp<T, 128>(l);
  else launch_tree_dp<T, 256>(l);
}

}  // namespace trellis
