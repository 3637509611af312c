// Rows of logits: what the verification of drafts (kf_spec.hip) and the beams' selection
// (kf_beam.hip) read them with.
#pragma once

#include "kf_common.h"

namespace kf {

// 16 bytes of a row as floats: granule k of the row's aligned granules, the
// row's first element at place `lead` of granule 0.  Places outside the row are
// -inf, and never read.
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* x;
  int lead, V;
  __device__ __forceinline__ Row(const T* p, int V_) : x(p), V(V_) {
    lead = (int)(((uintptr_t)p & 15) / sizeof(T));
  }
  __device__ __forceinline__ int granules() const { return (lead + V + E - 1) / E; }
  __device__ __forceinline__ int first(int k) const { return k * E - lead; }
  __device__ __forceinline__ u32x4 raw(int k) const {
    const int v0 = first(k);
    if (v0 >= 0 && v0 + E <= V) return *(const u32x4*)(x + v0);
    T t[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      t[e] = v0 + e >= 0 && v0 + e < V ? x[v0 + e] : from_f32<T>(-INFINITY);
    u32x4 u;
    __builtin_memcpy(&u, t, 16);
    return u;
  }
  static __device__ __forceinline__ void unpack(const u32x4& u, float* f) {
    if constexpr (sizeof(T) == 4)
      __builtin_memcpy(f, &u, 16);
    else
      unpack8<T>(u, f);
  }
};

// 2^x for x <= 0 in 64 bits: 2^round(x) times the Taylor polynomial of 2^r, |r| <=
// 1/2, whose first term left out is (ln 2 / 2)^12 / 12! = 6e-15.
__device__ __forceinline__ double exp2_64(double x) {
  const double n = __builtin_rint(x), r = x - n;
  constexpr double L = 0.69314718055994530942;
  constexpr double c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5,
                   c6 = c5 * L / 6, c7 = c6 * L / 7, c8 = c7 * L / 8, c9 = c8 * L / 9,
                   c10 = c9 * L / 10, c11 = c10 * L / 11;
  double p = c11;
  p = fma(p, r, c10);
  p = fma(p, r, c9);
  p = fma(p, r, c8);
  p = fma(p, r, c7);
  p = fma(p, r, c6);
  p = fma(p, r, c5);
  p = fma(p, r, c4);
  p = fma(p, r, c3);
  p = fma(p, r, c2);
  p = fma(p, r, L);
  p = fma(p, r, 1.0);
  // (below 2^-1070 nothing is left; -inf has no r)
  return x > -1070.0 ? __builtin_ldexp(p, (int)n) : x <= -1070.0 ? 0.0 : x;
}

}  // namespace kf
