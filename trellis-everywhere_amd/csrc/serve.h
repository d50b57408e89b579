// serve.h — what the kernels between a block's packed linears share: element types, wave and lane-group
// sums, and the paged key-value cache as the kernels see it.
#pragma once

#include "common.h"

namespace trellis {

typedef __bf16 bf16_t;

enum : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };   // enum trellis_dtype

// Eight consecutive elements as fp32. VEC: the address is 16-byte aligned.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (VEC) {
    typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
    for (int c = 0; c < static_cast<int>(sizeof(T)) / 2; ++c) {
      const vec_t w = *reinterpret_cast<const vec_t*>(p + c * (16 / sizeof(T)));
#pragma unroll
      for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) v[c * (16 / sizeof(T)) + i] = static_cast<float>(w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(p[i]);
  }
}

// Eight values rounded once to the type `dt` names and stored. VEC: element i0 of p is 16-byte aligned.
template <class T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (VEC) {
    typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
    for (int c = 0; c < static_cast<int>(sizeof(T)) / 2; ++c) {
      vec_t w;
#pragma unroll
      for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) w[i] = static_cast<T>(v[c * (16 / sizeof(T)) + i]);
      *reinterpret_cast<vec_t*>(p + c * (16 / sizeof(T))) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = static_cast<T>(v[i]);
  }
}

template <bool VEC>
__device__ __forceinline__ void store8_dt(void* p, long long i0, int dt, const float (&v)[8]) {
  if (dt == DT_F32) store8<float, VEC>(static_cast<float*>(p) + i0, v);
  else if (dt == DT_F16) store8<_Float16, VEC>(static_cast<_Float16*>(p) + i0, v);
  else store8<bf16_t, VEC>(static_cast<bf16_t*>(p) + i0, v);
}

// Four elements as fp32. VEC: the address is aligned to all four of them. Stores: it always is.
template <class T, bool VEC>
__device__ __forceinline__ float4_t load4(const T* p) {
  float4_t v;
  if constexpr (VEC) {
    typedef T vec_t __attribute__((ext_vector_type(4)));
    const vec_t w = *reinterpret_cast<const vec_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(p[i]);
  }
  return v;
}

// NT: a nontemporal store.
template <bool NT = false, class T>
__device__ __forceinline__ void store4(T* p, float4_t v) {
  typedef T vec_t __attribute__((ext_vector_type(4)));
  vec_t w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = static_cast<T>(v[i]);
  if constexpr (NT) __builtin_nontemporal_store(w, reinterpret_cast<vec_t*>(p));
  else *reinterpret_cast<vec_t*>(p) = w;
}

template <bool NT = false>
__device__ __forceinline__ void store4_dt(void* p, long long i0, int dt, float4_t v) {
  if (dt == DT_F32) store4<NT>(static_cast<float*>(p) + i0, v);
  else if (dt == DT_F16) store4<NT>(static_cast<_Float16*>(p) + i0, v);
  else store4<NT>(static_cast<bf16_t*>(p) + i0, v);
}

__device__ __forceinline__ void store_dt(void* p, long long i, int dt, float v) {
  if (dt == DT_F32) static_cast<float*>(p)[i] = v;
  else if (dt == DT_F16) static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
  else static_cast<bf16_t*>(p)[i] = static_cast<bf16_t>(v);
}

// The sum over a wave, in every lane.
__device__ __forceinline__ float wave_sum(float v, int lane) {
  v += lane_xor<1>(v, lane);
  v += lane_xor<2>(v, lane);
  v += lane_xor<4>(v, lane);
  v += lane_xor<8>(v, lane);
  v += lane_xor<16>(v, lane);
  v += lane_xor<32>(v, lane);
  return v;
}

__device__ __forceinline__ float wave_max(float v, int lane) {
  v = fmaxf(v, lane_xor<1>(v, lane));
  v = fmaxf(v, lane_xor<2>(v, lane));
  v = fmaxf(v, lane_xor<4>(v, lane));
  v = fmaxf(v, lane_xor<8>(v, lane));
  v = fmaxf(v, lane_xor<16>(v, lane));
  return fmaxf(v, lane_xor<32>(v, lane));
}

// Inclusive sum over the wave's lanes up to this one (DPP row shifts, then row broadcasts).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast:31 into rows 2 and 3
  return v;
}

// The sum over aligned groups of n lanes (a power of 2 up to 64).
__device__ __forceinline__ float group_sum(float v, int n, int lane) {
  if (n > 1) v += lane_xor<1>(v, lane);
  if (n > 2) v += lane_xor<2>(v, lane);
  if (n > 4) v += lane_xor<4>(v, lane);
  if (n > 8) v += lane_xor<8>(v, lane);
  if (n > 16) v += lane_xor<16>(v, lane);
  if (n > 32) v += lane_xor<32>(v, lane);
  return v;
}

// A load of what no kernel of the call writes: where the address is the same in every lane, by the scalar unit (from
// plain memory the compiler does that only if nothing the kernel stores could be there).
template <class T>
__device__ __forceinline__ T load_const(const T* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) T*>(reinterpret_cast<uintptr_t>(p));
}

// A paged cache (struct trellis_kv_cache). Offsets in elements, 64-bit: a cache passes 2^31 elements.
struct Cache {
  void* k;
  void* v;
  float* scores;
  int32_t* pos;
  const int32_t* table;
  const int32_t* lens;
  long long page_stride, head_stride, slot_stride, table_stride;
  int pages, heads, page_shift, d, rows, width, max_len;

  // tokens of row b that a call sees: the row's length within what the call and its table can hold
  __device__ __forceinline__ int length(int b) const {
    const int cap = min(static_cast<long long>(max_len), static_cast<long long>(width) << page_shift);
    return max(0, min(load_const(lens + b), cap));
  }
  // the page of logical slot j of row b (j within the table), or -1 where the table holds no page
  __device__ __forceinline__ int page_of(int b, int j) const {
    const int id = load_const(table + b * table_stride + (j >> page_shift));
    return static_cast<unsigned>(id) < static_cast<unsigned>(pages) ? id : -1;
  }
  __device__ __forceinline__ int in_page(int j) const { return j & ((1 << page_shift) - 1); }
  __device__ __forceinline__ long long row_at(int page, int head, int j) const {   // of k and v
    return page * page_stride + head * head_stride + in_page(j) * slot_stride;
  }
  __device__ __forceinline__ long long slot_at(int page, int head, int j) const {  // of scores and pos
    return ((static_cast<long long>(page) * heads + head) << page_shift) + in_page(j);
  }
};

}  // namespace trellis
