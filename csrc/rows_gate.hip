// Top-k gate: the k largest scores of each row and their softmax weights, and the gradient.
//
//   chosen: the k largest scores, equal ones in the order of their index; a masked or -inf
//           score is never chosen (label -1, weight 0), NaN orders above every number
//   normalize:     w = softmax over the chosen;        ds_j = w_j (dw_j - sum w dw)
//   not normalize: w = softmax over all allowed p, at the chosen;
//                  ds_i = p_i (dw_i [chosen] - sum w dw)
//
// Scores are compared as 32-bit whole numbers of the same order (0 = not to be chosen), so
// the choice does not depend on any rounding; exp and the sums are fp32.
#include "rows_common.h"

namespace tdc {
namespace rows {

constexpr int GATE_BLOCK = 256;
constexpr int GATE_MAX_K = 16;

// A score's place in the order: larger numbers for larger scores, 0 for one that is not
// allowed, the largest for NaN.  -0 and +0 are the same place.
__device__ __forceinline__ unsigned order_of(float f, bool allowed) {
  f += 0.f;
  const unsigned b = __float_as_uint(f);
  unsigned k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  if (f != f) k = 0xffffffffu;
  return (allowed && f != -INFINITY) ? k : 0u;
}

__device__ __forceinline__ float score_of(unsigned k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

struct Mask {
  const uint8_t* p;  // null: everything is allowed
  int64_t rs, cs;    // strides of rows and columns
  __device__ __forceinline__ bool at(int64_t row, int c) const {
    return p == nullptr || p[row * rs + c * cs] != 0;
  }
};

// L lanes work on a row, each with R scores in registers.  Every round takes the largest
// that is left, over the registers and then over the lanes.
template <typename T, int L, int R, int TAIL>
__global__ __launch_bounds__(GATE_BLOCK) void gate_kernel(const T* __restrict__ scores, int64_t ld,
                                                          Mask mask, int64_t n, int K, int k,
                                                          bool normalize, float* __restrict__ w,
                                                          int* __restrict__ labels,
                                                          float* __restrict__ stat) {
  constexpr int V = Vec<T>::N;
  const int lane = threadIdx.x % L;
  const int64_t row = (int64_t)blockIdx.x * (GATE_BLOCK / L) + threadIdx.x / L;
  if (row >= n) return;
  unsigned key[R];
  unsigned best = 0;
  Raw16 raw[R / V];
#pragma unroll
  for (int i = 0; i < R / V; ++i)
    raw[i] = RowVec<T, TAIL>::fetch(scores + row * ld, (i * L + lane) * V, K);
#pragma unroll
  for (int i = 0; i < R / V; ++i) {
    const int c = (i * L + lane) * V;
    float v[V];
    RowVec<T, TAIL>::value(raw[i], c, K, v);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      key[i * V + j] = order_of(v[j], c + j < K && mask.at(row, c + j));
      best = max(best, key[i * V + j]);
    }
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) best = max(best, (unsigned)__shfl_xor((int)best, o, 64));
  const float top = best ? score_of(best) : 0.f;
  float total = 0.f;
  if (!normalize) {
#pragma unroll
    for (int i = 0; i < R; ++i) total += key[i] ? expf(score_of(key[i]) - top) : 0.f;
    total = lanes_sum<L>(total);
  }
  unsigned mine = 0;
  int at = -1;
  for (int j = 0; j < k; ++j) {
    unsigned b = 0;
    int bi = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = ((i / V) * L + lane) * V + i % V;
      if (key[i] > b) {
        b = key[i];
        bi = c;
      }
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
      const unsigned ob = (unsigned)__shfl_xor((int)b, o, 64);
      const int oi = __shfl_xor(bi, o, 64);
      if (ob > b || (ob == b && oi < bi)) {
        b = ob;
        bi = oi;
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (((i / V) * L + lane) * V + i % V == bi) key[i] = 0;
    if (lane == j && b) {
      mine = b;
      at = bi;
    }
  }
  const float e = mine ? expf(score_of(mine) - top) : 0.f;
  if (normalize) total = lanes_sum<L>(e);
  if (lane < k) {
    w[row * k + lane] = mine ? e / total : 0.f;
    labels[row * k + lane] = at;
  }
  if (stat && lane == 0) {
    stat[2 * row] = top;
    stat[2 * row + 1] = best ? 1.f / total : 0.f;
  }
}

__device__ __forceinline__ void take_larger(unsigned& b, int& bi, unsigned ob, int oi) {
  if (ob > b || (ob == b && oi < bi)) {
    b = ob;
    bi = oi;
  }
}

// Any number of clusters: a block per row, which is read again in every round (from the
// caches).  What is left is what comes after the last choice in the order.
template <typename T>
__global__ __launch_bounds__(GATE_BLOCK) void gate_wide_kernel(
    const T* __restrict__ scores, int64_t ld, Mask mask, int64_t n, int K, int k, bool normalize,
    float* __restrict__ w, int* __restrict__ labels, float* __restrict__ stat) {
  __shared__ unsigned s_key[2][4];
  __shared__ int s_at[2][4];
  __shared__ float s_sum[4];
  const int64_t row = blockIdx.x;
  const T* src = scores + row * ld;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  unsigned last = 0xffffffffu, mine = 0;
  int last_at = -1, at = -1;
  float top = 0.f, total = 0.f;
  for (int j = 0; j < k; ++j) {
    unsigned b = 0;
    int bi = 0x7fffffff;
    for (int c = threadIdx.x; c < K; c += GATE_BLOCK) {
      const unsigned key = order_of(up(src[c]), mask.at(row, c));
      if ((key < last || (key == last && c > last_at)) && key > b) {
        b = key;
        bi = c;
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
      take_larger(b, bi, (unsigned)__shfl_xor((int)b, o, 64), __shfl_xor(bi, o, 64));
    if (lane == 0) {
      s_key[j & 1][wave] = b;
      s_at[j & 1][wave] = bi;
    }
    __syncthreads();
    b = s_key[j & 1][0];
    bi = s_at[j & 1][0];
    for (int i = 1; i < 4; ++i) take_larger(b, bi, s_key[j & 1][i], s_at[j & 1][i]);
    if (j == 0) top = b ? score_of(b) : 0.f;
    if (b == 0) break;  // nothing is left: the same for the whole block
    last = b;
    last_at = bi;
    if ((int)threadIdx.x == j) {
      mine = b;
      at = bi;
    }
  }
  if (!normalize) {
    for (int c = threadIdx.x; c < K; c += GATE_BLOCK) {
      const unsigned key = order_of(up(src[c]), mask.at(row, c));
      total += key ? expf(score_of(key) - top) : 0.f;
    }
    total = lanes_sum<64>(total);
    if (lane == 0) s_sum[wave] = total;
    __syncthreads();
    total = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  }
  const float e = mine ? expf(score_of(mine) - top) : 0.f;
  if (normalize) total = lanes_sum<64>(e);  // the chosen are in the first wave
  if ((int)threadIdx.x < k) {
    w[row * k + threadIdx.x] = mine ? e / total : 0.f;
    labels[row * k + threadIdx.x] = at;
  }
  if (stat && threadIdx.x == 0) {
    stat[2 * row] = top;
    stat[2 * row + 1] = mine ? 1.f / total : 0.f;
  }
}

// The gradient: L lanes per row write what every place gets and then, after those stores
// have arrived, the chosen places.
template <typename T, int L, int TAIL>
__global__ __launch_bounds__(GATE_BLOCK) void gate_bwd_kernel(
    const T* __restrict__ scores, int64_t ld, Mask mask, const float* __restrict__ w,
    const int* __restrict__ labels, const float* __restrict__ stat, const float* __restrict__ dw,
    int64_t n, int K, int k, bool normalize, T* __restrict__ ds) {
  constexpr int V = Vec<T>::N;
  const int lane = threadIdx.x % L;
  const int64_t row = (int64_t)blockIdx.x * (GATE_BLOCK / L) + threadIdx.x / L;
  if (row >= n) return;
  const float wj = lane < k ? w[row * k + lane] : 0.f;
  const float dj = lane < k ? dw[row * k + lane] : 0.f;
  const int at = lane < k ? labels[row * k + lane] : -1;
  const float mean = lanes_sum<L>(at >= 0 ? wj * dj : 0.f);
  float top = 0.f, scale = 0.f;
  if (!normalize) {
    top = stat[2 * row];
    scale = stat[2 * row + 1] * mean;
  }
  for (int c = lane * V; c < K; c += L * V) {
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
    if (!normalize) {
      RowVec<T, TAIL>::value(RowVec<T, TAIL>::fetch(scores + row * ld, c, K), c, K, v);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool in = c + j < K && mask.at(row, c + j) && v[j] != -INFINITY;
        v[j] = in ? -expf(v[j] - top) * scale : 0.f;
      }
    }
    RowVec<T, TAIL>::store(ds + row * K, c, K, v);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (at >= 0 && at < K) ds[row * K + at] = down<T>(wj * (dj - mean));
}

}  // namespace rows
}  // namespace tdc

using namespace tdc::rows;

int tdc_topk_gate(int dtype, const void* scores, int64_t ld, const uint8_t* mask, int64_t mask_rs,
                  int64_t mask_cs, int64_t n, int K, int k, int normalize, float* w, int* labels,
                  float* stat, hipStream_t stream) {
  if (n == 0) return 0;
  if (k < 1 || k > GATE_MAX_K || K < 1 || n > 0x7fffffff) return (int)hipErrorInvalidValue;
  const Mask m{mask, mask_rs, mask_cs};
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel, int lanes) {
      const int rows = GATE_BLOCK / lanes;
      hipLaunchKernelGGL(kernel, dim3((unsigned)((n + rows - 1) / rows)), dim3(GATE_BLOCK), 0,
                         stream, (const T*)scores, ld, m, n, K, k, normalize != 0, w, labels, stat);
    };
    return with_tail(K, Vec<T>::N, [&](auto tail) {
      constexpr int TAIL = decltype(tail)::value;
      if (K <= 128)
        go(gate_kernel<T, 16, 8, TAIL>, 16);
      else if (K <= 256)
        go(gate_kernel<T, 16, 16, TAIL>, 16);
      else if (K <= 1024)
        go(gate_kernel<T, 64, 16, TAIL>, 64);
      else
        go(gate_wide_kernel<T>, GATE_BLOCK);
      TDC_CHECK_LAUNCH();
      return 0;
    });
  });
}

int tdc_topk_gate_bwd(int dtype, const void* scores, int64_t ld, const uint8_t* mask,
                      int64_t mask_rs, int64_t mask_cs, const float* w, const int* labels,
                      const float* stat, const float* dw, int64_t n, int K, int k, int normalize,
                      void* ds, hipStream_t stream) {
  if (n == 0) return 0;
  if (k < 1 || k > GATE_MAX_K || K < 1 || n > 0x7fffffff) return (int)hipErrorInvalidValue;
  const Mask m{mask, mask_rs, mask_cs};
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel, int lanes) {
      const int rows = GATE_BLOCK / lanes;
      hipLaunchKernelGGL(kernel, dim3((unsigned)((n + rows - 1) / rows)), dim3(GATE_BLOCK), 0,
                         stream, (const T*)scores, ld, m, w, labels, stat, dw, n, K, k,
                         normalize != 0, (T*)ds);
    };
    return with_tail(K, Vec<T>::N, [&](auto tail) {
      constexpr int TAIL = decltype(tail)::value;
      if (K <= 256)
        go(gate_bwd_kernel<T, 16, TAIL>, 16);
      else
        go(gate_bwd_kernel<T, 64, TAIL>, 64);
      TDC_CHECK_LAUNCH();
      return 0;
    });
  });
}
