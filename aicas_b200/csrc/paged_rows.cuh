// What the appends to paged caches do to a row on the way: loads, per-head norm and
// rotate-half rotation of the two vectors of a row that a thread holds (its own of the
// first half and the matching one of the second).
#pragma once
#include <type_traits>

#include "common.cuh"

namespace aicas {

template <typename T>
__device__ __forceinline__ float rounded(float x) {
  return Elem<T>::to_float(Elem<T>::from_float(x));
}

// 16 bytes of T from floats, two a conversion.
template <typename T>
__device__ __forceinline__ uint4 pack_vec(const float* f) {
  union {
    uint4 u;
    __nv_bfloat162 b[4];
    __half2 h[4];
    float f[4];
  } r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      r.b[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    else if constexpr (std::is_same<T, __half>::value)
      r.h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    else
      r.f[i] = f[i];
  }
  return r.u;
}

// N floats of a row.
template <typename CS, int N>
__device__ __forceinline__ void load_floats(const CS* p, float* f) {
  constexpr int kV = Elem<CS>::kPerVec;
  if constexpr (N >= kV) {
#pragma unroll
    for (int i = 0; i < N / kV; ++i) Elem<CS>::unpack(reinterpret_cast<const uint4*>(p)[i], f + i * kV);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = Elem<CS>::to_float(p[i]);
  }
}

// x * inv * w; with EACH every product rounded to T, as Hugging Face's module rounds.
template <typename T, bool EACH, int N>
__device__ __forceinline__ void normed_pair(float* x1, float* x2, const float* w1, const float* w2, float inv) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (EACH) {
      x1[i] = rounded<T>(__fmul_rn(w1[i], rounded<T>(__fmul_rn(x1[i], inv))));
      x2[i] = rounded<T>(__fmul_rn(w2[i], rounded<T>(__fmul_rn(x2[i], inv))));
    } else {
      x1[i] *= inv * w1[i];
      x2[i] *= inv * w2[i];
    }
  }
}

// x cos + rotate_half(x) sin; with EACH the products rounded to T (the sum by whoever stores it).
template <typename T, bool EACH, int N>
__device__ __forceinline__ void rotated_pair(float* x1, float* x2, const float* c1, const float* c2, const float* s1,
                                             const float* s2) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float p1 = x1[i], p2 = x2[i];
    if (EACH) {
      x1[i] = __fadd_rn(rounded<T>(__fmul_rn(p1, c1[i])), rounded<T>(__fmul_rn(-p2, s1[i])));
      x2[i] = __fadd_rn(rounded<T>(__fmul_rn(p2, c2[i])), rounded<T>(__fmul_rn(p1, s2[i])));
    } else {
      x1[i] = p1 * c1[i] - p2 * s1[i];
      x2[i] = p2 * c2[i] + p1 * s2[i];
    }
  }
}

}  // namespace aicas
