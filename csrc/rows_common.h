// Shared device helpers of the row operators (rows_*.hip): typed 16-byte vectors at any
// alignment, element access and small reductions.
#pragma once
#include "tdc_common.h"
#include "kernels.h"

#include <algorithm>
#include <type_traits>

namespace tdc {
namespace rows {

// Elements of one 16-byte access.
template <typename T> struct Vec { static constexpr int N = 16 / (int)sizeof(T); };

// 16 bytes at the alignment of their elements: gfx950 reads and writes a dwordx4 at any
// address, so rows of odd widths and strides keep the wide accesses (a row of 1001 fp16
// values starts on every second byte pair).
struct __attribute__((packed, aligned(2))) Raw16 { unsigned w[4]; };

template <typename T> __device__ __forceinline__ float up(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T down(float v) { return (T)v; }

// Elements [c, c + Vec<T>::N) of a row of `width` as floats; those past its end are 0.
// The row's last, partial vector is read element by element.
template <typename T>
__device__ __forceinline__ void load_vec(const T* __restrict__ row, int c, int width,
                                         float (&v)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
  if (c + N <= width) {
    const Raw16 raw = *reinterpret_cast<const Raw16*>(row + c);
    T t[N];
    __builtin_memcpy(t, &raw, 16);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = up(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = c + i < width ? up(row[c + i]) : 0.f;
  }
}

// The same for N fp32 values next to a vector of N elements of T (weights, partial sums).
template <int N>
__device__ __forceinline__ void load_f32(const float* __restrict__ row, int c, int width,
                                         float (&v)[N]) {
  static_assert(N % 4 == 0, "whole dwordx4");
  if (c + N <= width) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
      const Raw16 raw = *reinterpret_cast<const Raw16*>(row + c + 4 * q);
      __builtin_memcpy(&v[4 * q], &raw, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = c + i < width ? row[c + i] : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store_vec(T* __restrict__ row, int c, int width,
                                          const float (&v)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
  T t[N];
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = down<T>(v[i]);
  if (c + N <= width) {
    Raw16 raw;
    __builtin_memcpy(&raw, t, 16);
    *reinterpret_cast<Raw16*>(row + c) = raw;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < width) row[c + i] = t[i];
  }
}

// Sum over G neighbouring lanes (a power of two up to 64), the same value in each.
template <int G> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Sum over the G threads of a row: G <= 64 within the wave, above through LDS, where the
// block is the row (G == blockDim.x).  `turn` alternates between two LDS rows, so one
// barrier per sum is enough.
template <int G> __device__ __forceinline__ float group_sum(float v, float (*s)[16], int& turn) {
  if constexpr (G <= 64) {
    return lanes_sum<G>(v);
  } else {
    v = lanes_sum<64>(v);
    float* p = s[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < G / 64; ++i) t += p[i];
    return t;
  }
}

// f(T()) for the rows' type; hipErrorInvalidValue for one that the row operators lack.
template <typename F> int with_type(int dtype, F&& f) {
  switch (dtype) {
    case TDC_F32: return f(float());
    case TDC_F16: return f(_Float16());
    case TDC_BF16: return f(__bf16());
    default: return (int)hipErrorInvalidValue;
  }
}

}  // namespace rows
}  // namespace tdc
