// Row access shared by the row kernels: 16-byte vectors of a row at any
// element address, its partial last vector, and the totals of the waves that
// share a row.
#pragma once

#include <cstdint>

#include "device_util.h"

namespace hxm {

// Waves of a workgroup whose rows take S waves each.
constexpr int row_waves(int S) { return S < 4 ? 4 : S; }

template <typename T>
struct RowVec {
  static constexpr int N = 16 / sizeof(T);  // elements per 16-byte vector
};

// One 16-byte vector of a row in its storage type.
template <typename T>
using RawVec = T __attribute__((ext_vector_type(RowVec<T>::N)));

// The same vector at any element address (a row may start anywhere).
template <typename T>
using AnyVec = T __attribute__((ext_vector_type(RowVec<T>::N), aligned(sizeof(T))));

// Row loads are plain (cacheable) and row stores nontemporal.  On a stream
// that reads and writes HBM at once this pairing ran fastest of the four
// (64 MiB copy, one box: plain loads + nontemporal stores 20.2 us,
// nontemporal both 22.2-22.6, nontemporal loads + plain stores 22.5, plain
// both 24.6); RMSNorm 22.1 -> 20.8 us and softmax 22.9 -> 20.9 us at
// 8192 x 4096 f16 with nontemporal loads replaced.  A read-only stream is the
// other way round (the GEMV's weights stay nontemporal).
template <typename T>
__device__ __forceinline__ RawVec<T> load_any(const T* p) {
  return *reinterpret_cast<const AnyVec<T>*>(p);
}
template <typename T>
__device__ __forceinline__ void store_any(T* p, RawVec<T> v) {
  __builtin_nontemporal_store(static_cast<AnyVec<T>>(v), reinterpret_cast<AnyVec<T>*>(p));
}

// The row's last, partial vector (elements [c0, cols), at least one): element
// by element, the rest of the vector set to `fill`.
template <typename T>
__device__ __forceinline__ RawVec<T> load_tail(const T* __restrict__ row, int64_t c0, int64_t cols,
                                               T fill) {
  constexpr int N = RowVec<T>::N;
  const int rem = static_cast<int>(cols - c0);
  RawVec<T> v;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const T e = row[c0 + min(j, rem - 1)];
    v[j] = j < rem ? e : fill;
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void store_tail(T* __restrict__ row, int64_t c0, int64_t cols,
                                           RawVec<T> v) {
#pragma unroll
  for (int j = 0; j < RowVec<T>::N; ++j)
    if (c0 + j < cols) row[c0 + j] = v[j];
}

// The S wave totals of a row combined pairwise (the rounding of S sequential
// adds of near-equal totals showed in f32 LayerNorm means).
template <int S, typename Op>
__device__ __forceinline__ float wave_totals(const float* t, Op op) {
  float v[S];
#pragma unroll
  for (int k = 0; k < S; ++k) v[k] = t[k];
#pragma unroll
  for (int w = 1; w < S; w *= 2)
#pragma unroll
    for (int k = 0; k + w < S; k += 2 * w) v[k] = op(v[k], v[k + w]);
  return v[0];
}

}  // namespace hxm
