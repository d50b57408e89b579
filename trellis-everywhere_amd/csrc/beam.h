// beam.h — beam search's selection over beams and vocabulary. Per batch element, of the candidates
//   c(j, v) = score_j + x_jv - lse_j,  lse_j = log sum_v exp(x_jv)
// of beam j's logits x_j (an ended beam offers (j, end token) alone, at score_j), the k largest, equal ones by the
// lower beam, then the lower token. A candidate that is -inf or not a number is none.
// Within a beam the order is that of its logits, exactly. Beams meet in 64 bits, so that a score's size costs nothing, but on
// sums of fp32 exponentials, up to 64 of them added in fp32: log sum exp is off by less than 5e-6 (some 1e-7 for a model's
// logits), and candidates of two beams within twice that of each other may change places. Equal rows have equal sums.
//
// beam_part_kernel: a wave takes a run of a beam's logits, R x 512 at a time, read once and held in registers: their
// maximum, the sum of their exponentials, and their k best. Of the maxima of the 256 lanes of four waves side by side (or of
// every four of them), sorted, the k-th is a bound that k of their logits reach: the few that do (k and a handful) are
// gathered through LDS and sorted by (logit, token) into each wave's list of 64.
// beam_join_kernel, a workgroup a batch element: per beam the runs' sums and lists, then the beams' lists.
// Bound: of large calls the vector units, busy 71 % of the time: 13 instructions a logit of 16 bits, some 6 of them its own
// (unpacked twice, maximum, fma, exponential at a quarter rate, sum), the rest a wave's bounds, loads, sorting and gathering.
// 64 x 8 beams of 151936 bf16 logits, a fifth of the beams ended: part 39.1 us (3.2 TB/s), join 7.0. Smaller ones by the chain
// load, maximum, sort, sum, gather, sort, which a wave runs once with nothing of another run under way: 16 x 4 of f16 12.1 +
// 4.4 (vector units busy 41 %), one beam of 49152 fp32 logits 4.5 + 3.8. Many beams or a large k by the join, whose last merge
// is one wave that sorts 64 / beams entries of a beam at a time: 4 x 16 beams with k = 32 / 64 28 / 40 us the call, 64 beams of
// 49152 with k = 64 59. With a bound of each wave's own
// logits the first call took 69 us instead of 57; with the candidates' pieces brought into one loop body 54 instead of 47.
#pragma once

#include "serve.h"

namespace trellis {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int BEAM_MOST = 64;   // beams, candidates kept of each, runs of a beam (TRELLIS_BEAM_MAX)
constexpr float BEAM_LOW = -__FLT_MAX__;   // no finite logit lies below it: what the sums are taken against begins here

// Up to this k the bound is the k-th of 64 maxima of four lanes each: one sort instead of a sort and three merges (64 x 8
// beams, k = 16: 41.7 -> 39.1 us, the short sort of a list's first 16 included). Beyond, of the 256 lanes' own: the 64th of 64
// would let some 300 of a run's logits pass (a call with k = 32 / 33: 53.2 / 53.9 us).
constexpr int BEAM_QUADS = 32;

struct BeamArgs {
  const void* x;
  long long x_b, x_j;           // strides of batch and beam in elements
  int batch, beams, vocab, k, end_token;
  int runs, per;                // waves a beam, and the pieces of 8 logits of each
  const float* scores;          // [batch][beams]
  const uint8_t* ended;         // [batch][beams] or null
  float* out_scores;            // [batch][k]
  int32_t* out_beams;
  int32_t* out_tokens;
  double* sums;                 // workspace: [batch x beams][runs] (sum of exponentials, and against which power of e)
  unsigned long long* best;     // workspace: [batch x beams][runs / 4][k] keys in order
};

typedef unsigned long long beam_t;   // a candidate: (order-preserving logit, ~token); 0: none

__device__ __forceinline__ uint32_t beam_order(float x) {   // of a logit above -inf: above 0
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);   // -0 counts as 0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float beam_logit(beam_t c) {
  const uint32_t key = c >> 32;
  return __builtin_bit_cast(float, (key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

template <int H>
__device__ __forceinline__ beam_t lane_xor64(beam_t v, int lane) {
  const uint32_t lo = __builtin_bit_cast(uint32_t, lane_xor<H>(__builtin_bit_cast(float, static_cast<uint32_t>(v)), lane));
  const uint32_t hi = __builtin_bit_cast(uint32_t, lane_xor<H>(__builtin_bit_cast(float, static_cast<uint32_t>(v >> 32)), lane));
  return static_cast<beam_t>(hi) << 32 | lo;
}
template <int H> __device__ __forceinline__ float lane_xor_t(float v, int lane) { return lane_xor<H>(v, lane); }
template <int H> __device__ __forceinline__ beam_t lane_xor_t(beam_t v, int lane) { return lane_xor64<H>(v, lane); }

// One level of a sorting network over the wave: of lanes H apart the one that `up` names for the pair gets the larger.
template <int H, class V>
__device__ __forceinline__ V sort_level(V v, bool lower_larger, int lane) {
  const V o = lane_xor_t<H>(v, lane);
  const bool larger = lower_larger == ((lane & H) == 0);
  return (o > v) == larger ? o : v;
}
template <int H, class V>
__device__ __forceinline__ V sort_merge(V v, bool lower_larger, int lane) {   // of 2 H lanes that rise and fall
  v = sort_level<H>(v, lower_larger, lane);
  if constexpr (H > 1) v = sort_merge<H / 2>(v, lower_larger, lane);
  return v;
}
// The wave's values in order, the largest first (or last).
template <class V>
__device__ __forceinline__ V wave_sort(V v, bool falling, int lane) {
  v = sort_merge<1>(v, (lane & 2) == 0, lane);
  v = sort_merge<2>(v, (lane & 4) == 0, lane);
  v = sort_merge<4>(v, (lane & 8) == 0, lane);
  v = sort_merge<8>(v, (lane & 16) == 0, lane);
  v = sort_merge<16>(v, (lane & 32) == 0, lane);
  return sort_merge<32>(v, falling, lane);
}

// The same of each 16 lanes.
template <class V>
__device__ __forceinline__ V row_sort(V v, bool falling, int lane) {
  v = sort_merge<1>(v, (lane & 2) == 0, lane);
  v = sort_merge<2>(v, (lane & 4) == 0, lane);
  v = sort_merge<4>(v, (lane & 8) == 0, lane);
  return sort_merge<8>(v, falling, lane);
}

// The same for (value, where it is from): of equal values the lower place counts as larger.
template <int H>
__device__ __forceinline__ void pair_merge(beam_t& v, uint32_t& from, bool lower_larger, int lane) {
  const beam_t o = lane_xor64<H>(v, lane);
  const uint32_t f = __builtin_bit_cast(uint32_t, lane_xor<H>(__builtin_bit_cast(float, from), lane));
  const bool larger = lower_larger == ((lane & H) == 0), above = o > v || (o == v && f < from);
  if (above == larger) {
    v = o;
    from = f;
  }
  if constexpr (H > 1) pair_merge<H / 2>(v, from, lower_larger, lane);
}
__device__ __forceinline__ void pair_sort(beam_t& v, uint32_t& from, bool falling, int lane) {
  pair_merge<1>(v, from, (lane & 2) == 0, lane);
  pair_merge<2>(v, from, (lane & 4) == 0, lane);
  pair_merge<4>(v, from, (lane & 8) == 0, lane);
  pair_merge<8>(v, from, (lane & 16) == 0, lane);
  pair_merge<16>(v, from, (lane & 32) == 0, lane);
  pair_merge<32>(v, from, falling, lane);
}

__device__ __forceinline__ beam_t readlane64(beam_t v, int l) {
  return static_cast<beam_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), l))) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), l));
}

// The 64 largest of a list in order and of a wave's values in none.
__device__ __forceinline__ beam_t beam_insert(beam_t best, beam_t c, int lane) {
  c = wave_sort(c, false, lane);
  return sort_merge<32>(best > c ? best : c, true, lane);
}

// The largest of the wave's values, in every lane.
__device__ __forceinline__ beam_t wave_top(beam_t v, int lane) {
  const auto larger = [&](beam_t o) { v = o > v ? o : v; };
  larger(lane_xor64<1>(v, lane));
  larger(lane_xor64<2>(v, lane));
  larger(lane_xor64<4>(v, lane));
  larger(lane_xor64<8>(v, lane));
  larger(lane_xor64<16>(v, lane));
  larger(lane_xor64<32>(v, lane));
  return v;
}

__device__ __forceinline__ double wave_sum64(double v, int lane) {
  const auto add = [&](beam_t o) { v += __builtin_bit_cast(double, o); };
  const auto bits = [&] { return __builtin_bit_cast(beam_t, v); };
  add(lane_xor64<1>(bits(), lane));
  add(lane_xor64<2>(bits(), lane));
  add(lane_xor64<4>(bits(), lane));
  add(lane_xor64<8>(bits(), lane));
  add(lane_xor64<16>(bits(), lane));
  add(lane_xor64<32>(bits(), lane));
  return v;
}

// A beam that offers no token of its logits: their rows are not read.
__device__ __forceinline__ bool beam_idle(const BeamArgs& a, long long row) {
  return (a.ended && a.ended[row]) || !(a.scores[row] > -__builtin_inff());
}

// Eight logits as they lie in memory.
template <class T> struct BeamPiece {
  typedef T vec8 __attribute__((ext_vector_type(8)));
  vec8 v;
  __device__ __forceinline__ float at(int e) const { return static_cast<float>(v[e]); }
  // What follows converts anew: the 16-bit logits stay in half the registers of their fp32 values.
  __device__ __forceinline__ void keep() {
    if constexpr (sizeof(T) == 2) {
      u32x4_t w = __builtin_bit_cast(u32x4_t, v);
      asm volatile("" : "+v"(w));
      v = __builtin_bit_cast(vec8, w);
    }
  }
};

template <class T, int R>
__global__ __launch_bounds__(256) void beam_part_kernel(BeamArgs a) {
  __shared__ beam_t s_few[4][64 + 512];
  __shared__ float s_top[4][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // a workgroup's four waves take runs of one beam
  const int quads = a.runs / 4, row = uniform(blockIdx.x / quads), run = (blockIdx.x - row * quads) * 4 + wave;
  if (beam_idle(a, row)) return;
  const int b = uniform(row / a.beams), j = row - b * a.beams;
  const T* x = static_cast<const T*>(a.x) + b * a.x_b + j * a.x_j;
  // (pieces of 8 count from the row's first logit, wherever that lies: equal rows have equal sums)
  const int pieces = static_cast<int>((static_cast<long long>(a.vocab) + 7) / 8);
  const int first = run * a.per, last = min(pieces, first + a.per);
  beam_t* few = s_few[wave];
  const float none = -__builtin_inff();

  beam_t best = 0, least = 0;    // the list, and its k-th
  float m = BEAM_LOW;
  double total = 0.0, base = BEAM_LOW;   // the sum against exp(base)
  bool begun = false;
  for (int p0 = first; p0 < first + a.per; p0 += 64 * R) {
    BeamPiece<T> piece[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int p = p0 + 64 * r + lane;
      const long long i0 = 8ll * p;
      if (p < last && i0 + 8 <= a.vocab) {
        __builtin_memcpy(&piece[r].v, x + i0, sizeof(piece[r].v));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) piece[r].v[e] = p < last && i0 + e < a.vocab ? x[i0 + e] : static_cast<T>(none);
      }
    }
    // the maximum (of a NaN and a number fmaxf takes the number)
    float tops[R], top = none;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      tops[r] = piece[r].at(0);
#pragma unroll
      for (int e = 1; e < 8; ++e) tops[r] = fmaxf(tops[r], piece[r].at(e));
      top = fmaxf(top, tops[r]);
    }
    top = top == top ? top : none;
    const float most = wave_max(top, lane);
    // what k of the workgroup's logits reach
    float bound = most;
    const bool quads_do = a.k > 1 && a.k <= BEAM_QUADS;
    if (quads_do) {
      bound = fmaxf(top, lane_xor<1>(top, lane));
      bound = fmaxf(bound, lane_xor<2>(bound, lane));
    } else if (a.k > 1) {
      bound = wave_sort(top, true, lane);
    }
    __syncthreads();
    if (!quads_do) s_top[wave][lane] = bound;
    else if ((lane & 3) == 0) s_top[wave][lane >> 2] = bound;
    __syncthreads();
    if (quads_do) {
      bound = wave_sort(s_top[lane >> 4][lane & 15], true, lane);
    } else {
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        if (a.k > 1) bound = sort_merge<32>(fmaxf(bound, s_top[wave ^ w][63 - lane]), true, lane);
        else bound = fmaxf(bound, s_top[wave ^ w][lane]);
      }
    }
    bound = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, bound), a.k > 1 ? a.k - 1 : 0));
    bound = fmaxf(bound, least ? beam_logit(least) : BEAM_LOW);
    if (most == none) continue;
    const float to = fmaxf(m, most);
    // The sum, of 2^(x log2(e) - top log2(e)) with the second product rounded once and kept as it is (its error is no term's
    // own): up to 4 R additions in fp32, then in 64 bits.
    const float shift = to * LOG2E;
    float sum[2] = {0.f, 0.f};
    const auto add_all = [&](auto careful) {
      sum[0] = sum[1] = 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        piece[r].keep();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x1 = piece[r].at(e);
          if constexpr (decltype(careful)::value) {
            const float v = __builtin_amdgcn_exp2f((x1 - to) * LOG2E);
            sum[e & 1] += v == v ? v : 0.f;
          } else {
            sum[e & 1] += __builtin_amdgcn_exp2f(__builtin_fmaf(x1, LOG2E, -shift));
          }
        }
      }
    };
    double against = static_cast<double>(shift) / static_cast<double>(LOG2E);
    // (beyond 2^20 half a step of the product is no small power of 2)
    const bool far = fabsf(to) > 1048576.f;
    if (!far) add_all(std::false_type{});
    if (far || __any(sum[0] + sum[1] != sum[0] + sum[1])) {   // not a number among them: those are none
      add_all(std::true_type{});
      against = to;
    }
    const double mine = static_cast<double>(sum[0]) + static_cast<double>(sum[1]);
    total = total * static_cast<double>(__builtin_amdgcn_exp2f(static_cast<float>((base - against) * static_cast<double>(LOG2E)))) +
            wave_sum64(mine, lane);
    m = to;
    base = against;
    unsigned with = 0;             // rounds that have some
#pragma unroll
    for (int r = 0; r < R; ++r) with |= (__any(tops[r] >= bound) ? 1u : 0u) << r;
    int count = 0;
    while (with || count) {
      // (every round in its own place: to bring the round's piece into one costs more than all else here)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (!(with >> r & 1) || count >= 64) continue;
        with &= ~(1u << r);
        BeamPiece<T> now = piece[r];
        now.keep();
        uint32_t own = lane;
        asm volatile("" : "+v"(own));   // (or every place in the run is formed beforehand and kept)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = now.at(e);
          if (!__any(v >= bound)) continue;       // mostly one logit of one lane does
          const beam_t c = static_cast<beam_t>(beam_order(v)) << 32 | ~(8u * (p0 + 64 * r + own) + e);
          const bool is = v >= bound && c > least;
          const unsigned long long who = __ballot(is);
          if (is) few[count + __popcll(who & ((1ull << lane) - 1))] = c;
          count += __popcll(who);
        }
      }
      // into the list, 64 at a time, the last ones when there are no more
      while (count >= 64 || (count && !with)) {
        const int some = min(count, 64);
        count -= some;
        __builtin_amdgcn_wave_barrier();
        const beam_t c = lane < some ? few[count + lane] : 0;
        if (a.k == 1) best = wave_top(c > best ? c : best, lane);
        else best = begun ? beam_insert(best, c, lane) : some <= 16 ? row_sort(c, true, lane) : wave_sort(c, true, lane);
        begun = true;
        least = readlane64(best, a.k - 1);
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
  if (lane == 0) {
    const long long at = static_cast<long long>(row) * a.runs + run;
    a.sums[2 * at] = total;
    a.sums[2 * at + 1] = base;
  }
  // the four lists as one
  __syncthreads();
  few[lane] = best;
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    const beam_t c = s_few[w][63 - lane];
    best = best > c ? best : c;
    if (a.k > 1) best = sort_merge<32>(best, true, lane);
  }
  if (lane < a.k) a.best[static_cast<long long>(blockIdx.x) * a.k + lane] = best;
}

// Order-preserving bits of a double above -inf.
__device__ __forceinline__ beam_t beam_order64(double v) {
  const beam_t u = __builtin_bit_cast(beam_t, v + 0.0);
  return (u >> 63) ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double beam_value64(beam_t key) {
  return __builtin_bit_cast(double, (key >> 63) ? key ^ 1ull << 63 : ~key);
}

// A workgroup a batch element, a wave a beam at a time.
__global__ __launch_bounds__(1024) void beam_join_kernel(BeamArgs a) {
  __shared__ beam_t s_value[BEAM_MOST * BEAM_MOST];
  __shared__ int32_t s_token[BEAM_MOST * BEAM_MOST];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, lane = threadIdx.x & 63;
  const int b = blockIdx.x;
  for (int j = wave; j < a.beams; j += waves) {
    const long long row = static_cast<long long>(b) * a.beams + j;
    const double score = a.scores[row];
    double value = -__builtin_inf();
    int token = a.end_token;
    if (beam_idle(a, row)) {
      if (lane == 0 && a.ended && a.ended[row]) value = score;
    } else {
      const bool is = lane < a.runs;
      // the lists, as many of each one's first entries at once as lanes hold
      const int lists = a.runs / 4, per = 64 / lists, of = lane / per, nth = lane - of * per;
      const beam_t* list = a.best + (row * lists + min(of, lists - 1)) * a.k;
      const auto entry = [&](int i) { return of < lists && i + nth < a.k ? list[i + nth] : 0; };
      const beam_t first = entry(0), second = entry(per);
      const double sum = is ? a.sums[2 * (row * a.runs + lane)] : 0.0, base = is ? a.sums[2 * (row * a.runs + lane) + 1] : BEAM_LOW;
      const float most = wave_max(static_cast<float>(base), lane);
      // lse = most + rest, never added: from 1e16 on the logarithm would be lost beside the maximum. (One lane's, for all: each
      // one's first addition takes its own product unrounded.)
      const double each = log(wave_sum64(sum * exp(base - static_cast<double>(most)), lane));
      const double rest = __builtin_bit_cast(double, readlane64(__builtin_bit_cast(beam_t, each), 0));
      // they are in order: no further ones when none of these can pass the k-th
      beam_t best = a.k == 1 ? wave_top(first, lane) : wave_sort(first, true, lane);
      for (int i = per; i < a.k; i += per) {
        const beam_t c = i == per ? second : entry(i);
        if (!__any(c > readlane64(best, a.k - 1))) break;
        best = beam_insert(best, c, lane);
      }
      token = static_cast<int>(~static_cast<uint32_t>(best));
      if (best) value = score + (static_cast<double>(beam_logit(best)) - static_cast<double>(most) - rest);
    }
    if (lane < a.k) {
      const bool is = value > -__builtin_inf();
      s_value[j * a.k + lane] = is ? beam_order64(value) : 0;
      s_token[j * a.k + lane] = token;
    }
  }
  __syncthreads();
  if (wave > 0) return;
  // the beams' lists together, by the value and then the beam: their first 64 / beams candidates, then the next, until none
  // can pass the k-th
  const int per = 64 / a.beams, mine = lane / per, nth = lane - mine * per;
  beam_t best = 0;
  uint32_t from = ~0u;       // beam x k + place
  for (int i0 = 0; i0 < a.k; i0 += per) {
    const int at = mine * a.k + i0 + nth;
    const bool is = mine < a.beams && i0 + nth < a.k;
    beam_t c = is ? s_value[at] : 0;
    uint32_t f = is && c ? at : ~0u;
    if (i0 > 0) {
      // (an equal one passes only if its beam is lower)
      const beam_t last = readlane64(best, a.k - 1);
      const uint32_t last_from = __builtin_amdgcn_readlane(from, a.k - 1);
      if (!__any(c > last || (c == last && f < last_from))) break;
      pair_sort(c, f, false, lane);
      const bool lower = c > best || (c == best && f < from);
      best = lower ? c : best;
      from = lower ? f : from;
      pair_merge<32>(best, from, true, lane);
    } else {
      pair_sort(c, f, true, lane);
      best = c;
      from = f;
    }
  }
  if (lane < a.k) {
    const long long o = static_cast<long long>(b) * a.k + lane;
    a.out_scores[o] = best ? static_cast<float>(beam_value64(best)) : -__builtin_inff();
    a.out_beams[o] = best ? from / a.k : 0;
    a.out_tokens[o] = best ? s_token[from] : a.end_token;
  }
}

}  // namespace trellis
