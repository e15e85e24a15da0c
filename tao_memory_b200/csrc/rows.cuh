// Rows of 16- or 32-bit values, read and written in vectors of 16 bytes (or single elements where a row or its
// address does not allow it) and computed in fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "../../include/tao_b200.h"
#include "common.cuh"

namespace tao {
namespace rows {

template <class T>
TAO_DEVI float wide_of(T v) {
  if constexpr (std::is_same<T, bf16>::value) return __bfloat162float(v);
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return v;
}
template <class T>
TAO_DEVI T rounded(float v) {
  if constexpr (std::is_same<T, bf16>::value) return __float2bfloat16_rn(v);
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return v;
}

// N values of a row that a thread has: neighbours, read and written at once (WIDE), or `step` apart, one by one, so
// that a warp's are neighbours.  What lies beyond the width reads as zeros and is not written.
template <class T, int N, bool WIDE>
struct alignas(sizeof(T) * N) Part {
  T v[N];
  TAO_DEVI void load(const T* row, int first, int step, int width) {
    if constexpr (WIDE) {
      *this = *reinterpret_cast<const Part*>(row + first);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = first + i * step < width ? row[first + i * step] : rounded<T>(0.f);
    }
  }
  TAO_DEVI void store(T* row, int first, int step, int width) const {
    if constexpr (WIDE) {
      *reinterpret_cast<Part*>(row + first) = *this;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (first + i * step < width) row[first + i * step] = v[i];
    }
  }
  TAO_DEVI void widen(float (&f)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = wide_of(v[i]);
  }
  static TAO_DEVI Part of(const float (&f)[N]) {
    Part r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = rounded<T>(f[i]);
    return r;
  }
};
// The first of thread `x` of `across` in slab `slab` of N x across values.
template <int N, bool WIDE>
TAO_DEVI int first_of(int slab, int across, int x) {
  return WIDE ? (slab * across + x) * N : slab * across * N + x;
}

// A value of a type known at run time.
TAO_DEVI float value_of(const void* p, long long i, int type) {
  if (type == TAO_TYPE_BF16) return wide_of(static_cast<const bf16*>(p)[i]);
  if (type == TAO_TYPE_FP16) return wide_of(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
TAO_DEVI void set_value(void* p, long long i, float v, int type) {
  if (type == TAO_TYPE_BF16) static_cast<bf16*>(p)[i] = rounded<bf16>(v);
  else if (type == TAO_TYPE_FP16) static_cast<__half*>(p)[i] = rounded<__half>(v);
  else static_cast<float*>(p)[i] = v;
}

template <int N>
using Int = std::integral_constant<int, N>;

inline size_t size_of(int type) { return type == TAO_TYPE_FP32 ? 4 : 2; }
inline bool known(int type) { return type == TAO_TYPE_BF16 || type == TAO_TYPE_FP16 || type == TAO_TYPE_FP32; }
// Whether rows of this base and stride start on 16 bytes (an absent operand's do).
inline bool on16(const void* p, long long stride, size_t size) {
  return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * (long long)size % 16 == 0);
}

// f(element type, values of a thread, whether they are neighbours) as compile-time constants.
template <class F>
int by_part(int type, bool wide, F f) {
  using True = std::true_type;
  using False = std::false_type;
  if (type == TAO_TYPE_FP32) return wide ? f(float(), Int<4>(), True()) : f(float(), Int<4>(), False());
  if (type == TAO_TYPE_FP16) return wide ? f(__half(), Int<8>(), True()) : f(__half(), Int<8>(), False());
  return wide ? f(bf16(), Int<8>(), True()) : f(bf16(), Int<8>(), False());
}

// A part of a row a thread: blocks of `across` x 256 / across threads, and their grid over rows and slabs.
struct Mapping {
  dim3 grid, block;
};
inline Mapping mapping(long long rows, int vectors) {
  int across = 32;
  while (across < vectors && across < 256) across *= 2;
  const int down = 256 / across;
  return {dim3((unsigned)((rows + down - 1) / down), (vectors + across - 1) / across), dim3(across, down)};
}

}  // namespace rows
}  // namespace tao
