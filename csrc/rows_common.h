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

template <typename T> __device__ __forceinline__ Raw16 load16(const T* p) {
  return *reinterpret_cast<const Raw16*>(p);
}
template <typename T> __device__ __forceinline__ void store16(T* p, const Raw16& r) {
  *reinterpret_cast<Raw16*>(p) = r;
}
// r, or zeros (word by word: a choice between two structs goes through scratch memory).
__device__ __forceinline__ Raw16 if_kept(bool kept, const Raw16& r) {
  Raw16 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o.w[i] = kept ? r.w[i] : 0u;
  return o;
}
template <typename T>
__device__ __forceinline__ void unpack(const Raw16& r, float (&v)[Vec<T>::N]) {
  T t[Vec<T>::N];
  __builtin_memcpy(t, &r, 16);
#pragma unroll
  for (int i = 0; i < Vec<T>::N; ++i) v[i] = up(t[i]);
}
template <typename T> __device__ __forceinline__ Raw16 pack(const float (&v)[Vec<T>::N]) {
  T t[Vec<T>::N];
#pragma unroll
  for (int i = 0; i < Vec<T>::N; ++i) t[i] = down<T>(v[i]);
  Raw16 r;
  __builtin_memcpy(&r, t, 16);
  return r;
}

// How a row of `width` splits into vectors of N elements: TAIL_NONE: without rest;
// TAIL_SHIFT: its last vector is partial; TAIL_SHORT: it is shorter than one vector (the norm
// of 16-bit rows that short puts 40 bytes a lane into scratch memory).
// A load must not sit in a branch of its own lanes: the wait for it would sit there too,
// and the loads of a thread would go out one after the other (the gradients of 131072 x 1024
// combined bf16 rows took 202 us with a branch around each load, 111 without).
enum Tail { TAIL_NONE = 0, TAIL_SHIFT = 1, TAIL_SHORT = 2 };

// Elements [c, c + N) of a row; fetch() issues the load, value() gives the floats, 0 past
// the row's end.  The last vector is read N elements before the end and shifted.
template <typename T, int TAIL> struct RowVec {
  static constexpr int N = Vec<T>::N;
  static __device__ __forceinline__ Raw16 fetch(const T* __restrict__ row, int c, int width) {
    if constexpr (TAIL == TAIL_SHORT) {
      T t[N];
#pragma unroll
      for (int i = 0; i < N; ++i) t[i] = c + i < width ? row[c + i] : T(0.f);
      Raw16 r;
      __builtin_memcpy(&r, t, 16);
      return r;
    } else {
      return load16(row + min(c, width - N));
    }
  }
  static __device__ __forceinline__ void value(Raw16 r, int c, int width, float (&v)[N]) {
    if constexpr (TAIL == TAIL_SHIFT) {
      const int by = (c - min(c, width - N)) * (int)sizeof(T);  // bytes to drop in front
      unsigned long long lo, hi;
      __builtin_memcpy(&lo, &r.w[0], 8);
      __builtin_memcpy(&hi, &r.w[2], 8);
      if (by >= 16) {
        lo = hi = 0;
      } else if (by >= 8) {
        lo = hi >> (8 * (by - 8));
        hi = 0;
      } else if (by > 0) {
        lo = (lo >> (8 * by)) | (hi << (64 - 8 * by));
        hi >>= 8 * by;
      }
      __builtin_memcpy(&r.w[0], &lo, 8);
      __builtin_memcpy(&r.w[2], &hi, 8);
      unpack<T>(r, v);
    } else if constexpr (TAIL == TAIL_NONE) {
      unpack<T>(if_kept(c < width, r), v);
    } else {
      unpack<T>(r, v);
    }
  }
  static __device__ __forceinline__ void store(T* __restrict__ row, int c, int width,
                                               const float (&v)[N]) {
    const Raw16 r = pack<T>(v);
    if (TAIL != TAIL_SHORT && c + N <= width) {
      store16(row + c, r);
    } else if (TAIL != TAIL_NONE && c < width) {
      T t[N];
      __builtin_memcpy(t, &r, 16);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c + i < width) row[c + i] = t[i];
    }
  }
};

// f(integral_constant<TAIL>) for a row of d elements in vectors of n.
template <typename F> int with_tail(int d, int n, F&& f) {
  if (d < n) return f(std::integral_constant<int, TAIL_SHORT>());
  if (d % n) return f(std::integral_constant<int, TAIL_SHIFT>());
  return f(std::integral_constant<int, TAIL_NONE>());
}

// Blocks over two grid dimensions: a dimension times the block's threads has to stay below
// 2^32, which one dimension alone does not for 17M rows of a block each.  Blocks past the
// last row find nothing to do.
inline dim3 grid_of(int64_t blocks, unsigned z = 1) {
  const int64_t x = blocks < (1 << 21) ? blocks : (1 << 21);
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x), z);
}
__device__ __forceinline__ int64_t block_index() {
  return (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
}

// The lane of this 16-lane row that DPP control CTRL names.
template <int CTRL> __device__ __forceinline__ unsigned dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(dpp<CTRL>(__float_as_uint(v)));
}
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
  return __hiloint2double((int)dpp<CTRL>((unsigned)__double2hiint(v)),
                          (int)dpp<CTRL>((unsigned)__double2loint(v)));
}
constexpr int DPP_XOR1 = 0xb1, DPP_XOR2 = 0x4e;  // quad_perm [1,0,3,2] and [2,3,0,1]
constexpr int DPP_HALF_MIRROR = 0x141;           // lane i of 8 from lane 7 - i
constexpr int DPP_ROR = 0x120;                   // + n: rotate the row by n lanes

// Sum over G neighbouring lanes (4 to 64, a power of two), the same value in each: rotations
// and quad permutations within a row of 16, then across rows.
template <int G, typename A> __device__ __forceinline__ A lanes_sum(A v) {
  if constexpr (G >= 16) {
    v += dpp<DPP_ROR + 8>(v);
    v += dpp<DPP_ROR + 4>(v);
    v += dpp<DPP_ROR + 2>(v);
    v += dpp<DPP_ROR + 1>(v);
    if constexpr (G >= 32) v += __shfl_xor(v, 16, 64);
    if constexpr (G >= 64) v += __shfl_xor(v, 32, 64);
  } else {
    v += dpp<DPP_XOR1>(v);
    v += dpp<DPP_XOR2>(v);
    if constexpr (G >= 8) v += dpp<DPP_HALF_MIRROR>(v);
  }
  return v;
}

// Sum over the G threads of a row: G <= 64 within the wave, above through LDS, where the
// block is the row (G == blockDim.x).  `turn` alternates between two LDS rows, so one
// barrier per sum is enough.
template <int G, typename A> __device__ __forceinline__ A group_sum(A v, A (*s)[16], int& turn) {
  if constexpr (G <= 64) {
    return lanes_sum<G>(v);
  } else {
    v = lanes_sum<64>(v);
    A* p = s[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = v;
    __syncthreads();
    A t = 0;
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
