// Rows sorted by cluster and back, with weights, and the gradients.
//
// A plan is a stable counting sort of the N*k slots (slot n*k + j: row n's j-th label):
//   order[p] = slot at place p, pos[slot] = p, offsets[c] .. offsets[c + 1] = the places of
//   cluster c.  Slots whose label is not in [0, K) come after offsets[K], in slot order.
// The sort goes by digits of at most 11 bits: one pass up to K = 2047, two up to 2^22 - 1.
// A pass counts its digits per chunk of 4096 slots, sums the counts over the chunks and
// scatters; ranks inside a chunk come from ballots, so that equal labels keep their order
// and every run gives the same plan (no atomics on positions).
//
//   group:    xg[p] = x[order[p] / k]          gradient: dx[n] = sum_j dxg[pos[n, j]]
//   combine:  out[n] = sum_j w[n, j] y[pos[n, j]]
//             gradient: dy[p] = w[slot] dout[row], dw[n, j] = <dout[n], y[pos[n, j]]>
// Places from offsets[K] on are written as zeros and never read.  Sums are fp32, in the
// order of j.  All of it is bound by memory.
#include "rows_common.h"

namespace tdc {
namespace rows {

constexpr int SORT_BLOCK = 256;
constexpr int SORT_WAVES = SORT_BLOCK / 64;
constexpr int SORT_PER_LANE = 16;
constexpr int SORT_CHUNK = SORT_BLOCK * SORT_PER_LANE;
constexpr int DIGIT_BITS = 11;
constexpr int MAX_DIGITS = 1 << DIGIT_BITS;

// The sort key of a slot: its label, or K where that is none of the clusters.
template <typename I> __device__ __forceinline__ int key_of(const I* labels, int64_t i, int K) {
  const I v = labels[i];
  return (v >= 0 && v < (I)K) ? (int)v : K;
}

// Input of a pass: labels (first pass) or the keys that the first pass left in its order.
template <typename I> struct FromLabels {
  const I* labels;
  int K;
  __device__ __forceinline__ int key(int64_t i) const { return key_of(labels, i, K); }
  __device__ __forceinline__ int slot(int64_t i) const { return (int)i; }
};
struct FromPairs {
  const int2* pairs;  // key, slot
  __device__ __forceinline__ int key(int64_t i) const { return pairs[i].x; }
  __device__ __forceinline__ int slot(int64_t i) const { return pairs[i].y; }
};

template <typename In>
__global__ __launch_bounds__(SORT_BLOCK) void sort_count_kernel(In in, int64_t m, int shift,
                                                                int digits, int* __restrict__ hist) {
  __shared__ int cnt[MAX_DIGITS];
  for (int d = threadIdx.x; d < digits; d += SORT_BLOCK) cnt[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * SORT_CHUNK;
#pragma unroll
  for (int i = 0; i < SORT_PER_LANE; ++i) {
    const int64_t at = base + i * SORT_BLOCK + threadIdx.x;
    if (at < m) atomicAdd(&cnt[(in.key(at) >> shift) & (MAX_DIGITS - 1)], 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += SORT_BLOCK)
    hist[(int64_t)d * gridDim.x + blockIdx.x] = cnt[d];
}

// Exclusive sum over the 256 threads of a block; total: the whole sum.
__device__ __forceinline__ int block_scan(int v, int* s_wave, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(inc, o, 64);
    if (lane >= o) inc += t;
  }
  __syncthreads();  // s_wave may still be read by the last call
  if (lane == 63) s_wave[wave] = inc;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < SORT_WAVES; ++i) {
    before += i < wave ? s_wave[i] : 0;
    total += s_wave[i];
  }
  return before + inc - v;
}

// One block per digit: its counts become sums over the chunks before, totals[d] the digit's.
__global__ __launch_bounds__(SORT_BLOCK) void sort_scan_kernel(int* __restrict__ hist, int chunks,
                                                               int* __restrict__ totals) {
  __shared__ int s_wave[SORT_WAVES];
  int* row = hist + (int64_t)blockIdx.x * chunks;
  int run = 0;
  for (int b = 0; b < chunks; b += SORT_BLOCK) {
    const int i = b + threadIdx.x;
    const int v = i < chunks ? row[i] : 0;
    int total;
    const int e = block_scan(v, s_wave, total);
    if (i < chunks) row[i] = run + e;
    run += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = run;
}

// Places of a chunk's slots.  With one chunk (hist == null) the block's own counts are the
// totals, and the whole sort is this launch.
template <typename In, bool LAST>
__global__ __launch_bounds__(SORT_BLOCK) void sort_scatter_kernel(
    In in, int64_t m, int shift, int digits, int bits, const int* __restrict__ hist,
    const int* __restrict__ totals, int2* __restrict__ pairs, int* __restrict__ keys,
    int* __restrict__ order, int* __restrict__ pos, int* __restrict__ offsets) {
  __shared__ int cnt[SORT_WAVES][MAX_DIGITS];
  __shared__ int s_wave[SORT_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int d = threadIdx.x; d < digits; d += SORT_BLOCK)
#pragma unroll
    for (int i = 0; i < SORT_WAVES; ++i) cnt[i][d] = 0;
  __syncthreads();
  // a wave owns 1024 slots in a row, 64 of them at a time
  const int64_t base = (int64_t)blockIdx.x * SORT_CHUNK + wave * (64 * SORT_PER_LANE) + lane;
  int key[SORT_PER_LANE];
#pragma unroll
  for (int i = 0; i < SORT_PER_LANE; ++i) {
    const int64_t at = base + i * 64;
    key[i] = at < m ? in.key(at) : -1;
    if (at < m) atomicAdd(&cnt[wave][(key[i] >> shift) & (MAX_DIGITS - 1)], 1);
  }
  __syncthreads();
  // first place of each digit, then of each wave's part of it: 8 digits per thread
  constexpr int PER = MAX_DIGITS / SORT_BLOCK;
  int sum = 0, have[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int d = threadIdx.x * PER + i;
    int t = 0;
    if (d < digits) {
      if (totals) {
        t = totals[d];
      } else {
        for (int q = 0; q < SORT_WAVES; ++q) t += cnt[q][d];
      }
    }
    have[i] = t;
    sum += t;
  }
  int total;
  int first = block_scan(sum, s_wave, total);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int d = threadIdx.x * PER + i;
    if (d < digits) {
      if (offsets && blockIdx.x == 0) offsets[d] = first;
      int at = first + (hist ? hist[(int64_t)d * gridDim.x + blockIdx.x] : 0);
      for (int q = 0; q < SORT_WAVES; ++q) {
        const int c = cnt[q][d];
        cnt[q][d] = at;
        at += c;
      }
    }
    first += have[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SORT_PER_LANE; ++i) {
    const int64_t at = base + i * 64;
    const bool in_range = at < m;
    const int d = in_range ? (key[i] >> shift) & (MAX_DIGITS - 1) : 0;
    // lanes with the same digit as this one
    unsigned long long same = __ballot(in_range);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long has = __ballot((d >> b) & 1);
      same &= ((d >> b) & 1) ? has : ~has;
    }
    if (in_range) {
      const int rank = __popcll(same & ((1ull << lane) - 1));
      volatile int* next = &cnt[wave][d];
      const int p = *next + rank;
      // the last lane of the digit moves its next place on, after all have read it
      __builtin_amdgcn_wave_barrier();
      if ((same >> lane) == 1ull) *next = p + 1;
      if constexpr (LAST) {
        const int slot = in.slot(at);
        order[p] = slot;
        pos[slot] = p;
        if (keys) keys[p] = key[i];
      } else {
        pairs[p] = make_int2(key[i], in.slot(at));
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// offsets[c] = first place whose key is c or more, for c in 0..K: the places where the key
// steps up write those they step over, a whole wave at a time.
__global__ __launch_bounds__(SORT_BLOCK) void sort_offsets_kernel(const int* __restrict__ keys,
                                                                  int m, int K,
                                                                  int* __restrict__ offsets) {
  const int lane = threadIdx.x & 63;
  const int64_t p = (int64_t)blockIdx.x * SORT_BLOCK + threadIdx.x;
  int lo = 0, hi = 0;  // this place writes offsets lo .. hi - 1
  if (p <= m) {
    lo = p == 0 ? 0 : keys[p - 1] + 1;
    hi = p == m ? K + 1 : keys[p] + 1;
  }
  unsigned long long todo = __ballot(hi > lo);
  while (todo) {
    const int l = __ffsll((long long)todo) - 1;
    todo &= todo - 1;
    const int a = __shfl(lo, l, 64), b = __shfl(hi, l, 64);
    const int place = __shfl((int)p, l, 64);
    for (int c = a + lane; c < b; c += 64) offsets[c] = place;
  }
}

// ------------------------------------------------------------------ rows
__device__ __forceinline__ int kept_places(const int* offsets, int K, int64_t m) {
  const int t = offsets[K];
  return t < 0 ? 0 : (t > m ? (int)m : t);
}

// A row's slots: L lanes read the row once and write it to each of its places (zeros at a
// place behind the kept ones).
template <typename T>
__global__ __launch_bounds__(256) void group_kernel(const T* __restrict__ x, int64_t ldx, int64_t n,
                                                    int k, int d, const int* __restrict__ offsets,
                                                    int K, const int* __restrict__ pos,
                                                    T* __restrict__ out, int L) {
  constexpr int V = Vec<T>::N;
  const int lane = threadIdx.x & (L - 1);
  const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (row >= n) return;
  const int kept = kept_places(offsets, K, n * k);
  for (int c = lane * V; c < d; c += L * V) {
    float v[V], zero[V];
    load_vec<T>(x + row * ldx, c, d, v);
#pragma unroll
    for (int i = 0; i < V; ++i) zero[i] = 0.f;
    for (int j = 0; j < k; ++j) {
      const int p = pos[row * k + j];
      if ((unsigned)p < (unsigned)(n * k)) {
        if (p < kept)
          store_vec<T>(out + (int64_t)p * d, c, d, v);
        else
          store_vec<T>(out + (int64_t)p * d, c, d, zero);
      }
    }
  }
}

// out[n] = sum_j w[n, j] y[pos[n, j]] (w null: 1).
template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(const T* __restrict__ y, int64_t ldy, int64_t n,
                                                      int k, int d, const int* __restrict__ offsets,
                                                      int K, const int* __restrict__ pos,
                                                      const void* __restrict__ w, bool w32,
                                                      T* __restrict__ out, int L) {
  constexpr int V = Vec<T>::N;
  const int lane = threadIdx.x & (L - 1);
  const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (row >= n) return;
  const unsigned kept = (unsigned)kept_places(offsets, K, n * k);
  for (int c = lane * V; c < d; c += L * V) {
    float a[V];
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = 0.f;
    for (int j = 0; j < k; ++j) {
      const int64_t slot = row * k + j;
      const unsigned p = (unsigned)pos[slot];
      if (p < kept) {
        const float wj = w ? (w32 ? ((const float*)w)[slot] : up(((const T*)w)[slot])) : 1.f;
        float v[V];
        load_vec<T>(y + (int64_t)p * ldy, c, d, v);
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = fmaf(wj, v[i], a[i]);
      }
    }
    store_vec<T>(out + row * d, c, d, a);
  }
}

// Gradients of a slot: dy[p] = w dout[row], dw = <dout[row], y[p]>; either may be left out.
template <typename T>
__global__ __launch_bounds__(256) void combine_bwd_kernel(
    const T* __restrict__ dout, int64_t lddo, const T* __restrict__ y, int64_t ldy, int64_t n, int k,
    int d, const int* __restrict__ offsets, int K, const int* __restrict__ pos,
    const void* __restrict__ w, bool w32, T* __restrict__ dy, void* __restrict__ dw, int L) {
  constexpr int V = Vec<T>::N;
  const int lane = threadIdx.x & (L - 1);
  const int64_t slot = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const int64_t m = n * k;
  float dot = 0.f;
  if (slot < m) {
    const int64_t row = slot / k;
    const unsigned kept = (unsigned)kept_places(offsets, K, m);
    const unsigned p = (unsigned)pos[slot];
    const float wj = w ? (w32 ? ((const float*)w)[slot] : up(((const T*)w)[slot])) : 1.f;
    if (p < (unsigned)m)
      for (int c = lane * V; c < d; c += L * V) {
        float g[V], o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = 0.f;
        if (p < kept) {
          load_vec<T>(dout + row * lddo, c, d, g);
          if (dw) {
            float v[V];
            load_vec<T>(y + (int64_t)p * ldy, c, d, v);
#pragma unroll
            for (int i = 0; i < V; ++i) dot = fmaf(g[i], v[i], dot);
          }
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] = wj * g[i];
        }
        if (dy) store_vec<T>(dy + (int64_t)p * d, c, d, o);
      }
  }
  if (!dw) return;
  for (int o = L / 2; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
  if (slot < m && lane == 0) {
    if (w32)
      ((float*)dw)[slot] = dot;
    else
      ((T*)dw)[slot] = down<T>(dot);
  }
}

// Lanes of a row: as many as it has 16-byte vectors, a power of two up to a wave.
inline int lanes_for(int d, int v) {
  const int vecs = (d + v - 1) / v;
  int l = 4;
  while (l < 64 && l < vecs) l *= 2;
  return l;
}

struct SortShape {
  int64_t m;
  int bits, low, high;  // digits of the first and the second pass (0: one pass)
  int64_t chunks;
};

inline SortShape sort_shape(int64_t m, int K) {
  SortShape s;
  s.m = m;
  s.bits = 1;
  while ((K >> s.bits) != 0) ++s.bits;  // keys 0..K
  s.low = s.bits <= DIGIT_BITS ? s.bits : DIGIT_BITS;
  s.high = s.bits - s.low;
  s.chunks = (m + SORT_CHUNK - 1) / SORT_CHUNK;
  return s;
}

inline int digits_of(const SortShape& s, int pass, int K) {
  if (s.high == 0) return K + 1;
  return pass == 0 ? 1 << s.low : (K >> s.low) + 1;
}

}  // namespace rows
}  // namespace tdc

using namespace tdc::rows;

// int32 words of scratch of a plan (counts, totals and, with two passes, pairs and keys).
int64_t tdc_group_plan_work(int64_t m, int K) {
  if (m <= 0) return 0;
  const SortShape s = sort_shape(m, K);
  const int64_t digits = std::max(digits_of(s, 0, K), s.high ? digits_of(s, 1, K) : 0);
  int64_t words = s.chunks > 1 ? digits * (s.chunks + 1) : 0;
  words += words & 1;  // the pairs are 8-byte aligned
  if (s.high) words += 3 * m;
  return words;
}

int tdc_group_plan(int wide_labels, const void* labels, int64_t m, int K, int* work, int* order,
                   int* pos, int* offsets, hipStream_t stream) {
  if (K < 1 || K >= (1 << 22) || m < 0 || m > 0x7ffffffe) return (int)hipErrorInvalidValue;
  const SortShape s = sort_shape(m, K);
  const int most = std::max(digits_of(s, 0, K), s.high ? digits_of(s, 1, K) : 0);
  int* hist = nullptr;
  int* totals = nullptr;
  int64_t used = 0;
  if (s.chunks > 1) {
    hist = work;
    totals = work + (int64_t)most * s.chunks;
    used = (int64_t)most * (s.chunks + 1);
    used += used & 1;
  }
  int2* pairs = s.high ? reinterpret_cast<int2*>(work + used) : nullptr;
  int* keys = s.high ? work + used + 2 * m : nullptr;
  const dim3 grid((unsigned)std::max<int64_t>(s.chunks, 1)), block(SORT_BLOCK);
  auto pass = [&](auto in, auto last, int shift, int bits, int digits) {
    constexpr bool LAST = decltype(last)::value;
    using In = decltype(in);
    if (s.chunks > 1) {
      hipLaunchKernelGGL(sort_count_kernel<In>, grid, block, 0, stream, in, m, shift, digits, hist);
      TDC_CHECK_LAUNCH();
      hipLaunchKernelGGL(sort_scan_kernel, dim3(digits), block, 0, stream, hist, (int)s.chunks,
                         totals);
      TDC_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL((sort_scatter_kernel<In, LAST>), grid, block, 0, stream, in, m, shift, digits,
                       bits, hist, totals, pairs, LAST ? keys : nullptr, order, pos,
                       s.high ? nullptr : offsets);
    TDC_CHECK_LAUNCH();
    return 0;
  };
  auto all = [&](auto in) {
    if (s.high == 0) return pass(in, std::true_type(), 0, s.low, digits_of(s, 0, K));
    int rc = 0;
    if (m > 0) {
      rc = pass(in, std::false_type(), 0, s.low, digits_of(s, 0, K));
      if (rc == 0)
        rc = pass(FromPairs{pairs}, std::true_type(), s.low, s.high, digits_of(s, 1, K));
    }
    if (rc) return rc;
    hipLaunchKernelGGL(sort_offsets_kernel, dim3((unsigned)((m + 1 + SORT_BLOCK - 1) / SORT_BLOCK)),
                       block, 0, stream, keys, (int)m, K, offsets);
    TDC_CHECK_LAUNCH();
    return 0;
  };
  if (wide_labels) return all(FromLabels<int64_t>{(const int64_t*)labels, K});
  return all(FromLabels<int32_t>{(const int32_t*)labels, K});
}

int tdc_group_rows(int dtype, const void* x, int64_t ldx, int64_t n, int k, int d,
                   const int* offsets, int K, const int* pos, void* out, hipStream_t stream) {
  if (n == 0) return 0;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int L = lanes_for(d, Vec<T>::N);
    const int64_t blocks = (n + 256 / L - 1) / (256 / L);
    hipLaunchKernelGGL(group_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)x,
                       ldx, n, k, d, offsets, K, pos, (T*)out, L);
    TDC_CHECK_LAUNCH();
    return 0;
  });
}

int tdc_combine_rows(int dtype, const void* y, int64_t ldy, int64_t n, int k, int d,
                     const int* offsets, int K, const int* pos, const void* w, int w32, void* out,
                     hipStream_t stream) {
  if (n == 0) return 0;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int L = lanes_for(d, Vec<T>::N);
    const int64_t blocks = (n + 256 / L - 1) / (256 / L);
    hipLaunchKernelGGL(combine_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)y,
                       ldy, n, k, d, offsets, K, pos, w, w32 != 0, (T*)out, L);
    TDC_CHECK_LAUNCH();
    return 0;
  });
}

int tdc_combine_rows_bwd(int dtype, const void* dout, int64_t lddo, const void* y, int64_t ldy,
                         int64_t n, int k, int d, const int* offsets, int K, const int* pos,
                         const void* w, int w32, void* dy, void* dw, hipStream_t stream) {
  if (n == 0 || (!dy && !dw)) return 0;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int L = lanes_for(d, Vec<T>::N);
    const int64_t blocks = (n * k + 256 / L - 1) / (256 / L);
    hipLaunchKernelGGL(combine_bwd_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream,
                       (const T*)dout, lddo, (const T*)y, ldy, n, k, d, offsets, K, pos, w, w32 != 0,
                       (T*)dy, dw, L);
    TDC_CHECK_LAUNCH();
    return 0;
  });
}
