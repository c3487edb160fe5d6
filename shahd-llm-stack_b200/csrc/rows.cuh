// Values of packed rows as the operators read and write them, and the sequence that a row belongs to.
#pragma once

#include <type_traits>

#include "ops_common.cuh"

namespace shahd {

template <class T>
__device__ __forceinline__ float ToFloat(T x) {
  return float(x);
}
template <class T>
__device__ __forceinline__ T FromFloat(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

// Eight values as they lie in memory, and as floats.
template <class T>
struct Raw8 {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void Load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void Get(float (&v)[8]) const {
    const T* h = reinterpret_cast<const T*>(u);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = ToFloat(h[i]);
  }
};
template <class T>
__device__ __forceinline__ void Store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint4 u;
    T* h = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = FromFloat<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

// The sequence that holds packed row `row`: the last s with offsets[s] <= row (empty sequences before it share its start).
__device__ __forceinline__ int SequenceOf(const int* offsets, int n, int row) {
  int lo = 0, hi = n;  // offsets[lo] <= row < offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace shahd
