// Top-k gate: the k largest scores of each row and their softmax weights, and the gradient.
//
//   chosen: the k largest scores, equal ones in the order of their index; a masked or -inf
//           score is never chosen (label -1, weight 0), NaN orders above every number
//   normalize:     w = softmax over the chosen;        ds_j = w_j (dw_j - sum w dw)
//   not normalize: w = softmax over all allowed p, at the chosen;
//                  ds_i = p_i (dw_i [chosen] - sum w dw)
//
// Scores are compared as whole numbers of the same order (0 = not to be chosen), so the
// choice does not depend on any rounding; exp and the sums are fp32.
//
// Up to 8192 clusters a row stays in the registers of L threads, 8 to 32 scores each: as few
// threads as hold it, since a round's part over the threads costs each of them the same (64M
// bf16 scores, k = 8, in rows of 600: 57 us as 32 x 24, 78 as 64 x 16; in rows of 64: 60 us
// as 8 x 8, 111 as 16 x 8).
//
// A score and its index become one number, the index in place of the score's last 6 to 13
// bits as fp32: 16-bit types have nothing there.  The j-th choice is the largest number
// below the (j-1)-th, found as the smallest of (limit - number), where what is above the
// limit wraps around to more than the rest: 1.5 instructions per score and round, nothing
// is taken out.  Where fp32 loses bits that are not zero and two neighbours among the first
// k + 1 choices agree in the bits that are left, the rows of that wave are chosen again by
// the whole scores.  65536 x 256 fp32, k = 8: 21 us, 37 with whole scores in every round.
// With k = 1 it takes 13 us (5.3 TB/s), with k = 4 15: the rounds are what is added.  Vector
// instructions fill 0.43, 0.55 and 0.59 of the issue slots at k = 1, 4 and 8, the cycles of
// the launch itself counted in; 12289 x 1000 bf16, masked and over all, 20 us, 0.59 as well,
// where a score is held twice.
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

// The mask of a vector of N scores: bit i of bits() is element c + i's.  Neighbouring bytes
// are one load, taken N bytes before the row's end for its last, partial vector.
template <int N, int TAIL> struct MaskVec {
  uint64_t r;
  __device__ __forceinline__ void fetch(const Mask& m, int64_t row, int c, int K) {
    r = ~0ull;
    if (m.p == nullptr) return;
    if (TAIL != TAIL_SHORT && m.cs == 1) {
      r = 0;
      __builtin_memcpy(&r, m.p + row * m.rs + min(c, K - N), N);
    }
  }
  __device__ __forceinline__ unsigned bits(const Mask& m, int64_t row, int c, int K) const {
    unsigned in = 0;
    if (m.p != nullptr && (TAIL == TAIL_SHORT || m.cs != 1)) {
#pragma unroll
      for (int i = 0; i < N; ++i) in |= (c + i < K && m.at(row, c + i)) ? 1u << i : 0u;
      return in;
    }
    uint64_t v = r;
    if (m.p != nullptr && TAIL == TAIL_SHIFT) v >>= 8 * min(c - min(c, K - N), N - 1);
#pragma unroll
    for (int i = 0; i < N; ++i) in |= (c + i < K && (v >> (8 * i) & 0xff)) ? 1u << i : 0u;
    return in;
  }
};

// Over the L threads of a row, the result in each: rotations within 16 lanes, the four rows
// of a wave through scalars, the waves of a block through LDS (two rows in turn, one
// barrier).
template <typename Op> __device__ __forceinline__ unsigned row_all(unsigned v, Op op) {
  v = op(v, dpp<DPP_ROR + 8>(v));
  v = op(v, dpp<DPP_ROR + 4>(v));
  v = op(v, dpp<DPP_ROR + 2>(v));
  return op(v, dpp<DPP_ROR + 1>(v));
}
template <int L, typename Op>
__device__ __forceinline__ unsigned group_all(unsigned v, Op op, unsigned (*s)[4], int& turn) {
  if constexpr (L == 8) {
    v = op(v, dpp<DPP_XOR1>(v));
    v = op(v, dpp<DPP_XOR2>(v));
    return op(v, dpp<DPP_HALF_MIRROR>(v));
  }
  v = row_all(v, op);
  if constexpr (L == 32) v = op(v, (unsigned)__shfl_xor((int)v, 16, 64));
  if constexpr (L > 32) {
    v = op(op((unsigned)__builtin_amdgcn_readlane((int)v, 0),
              (unsigned)__builtin_amdgcn_readlane((int)v, 16)),
           op((unsigned)__builtin_amdgcn_readlane((int)v, 32),
              (unsigned)__builtin_amdgcn_readlane((int)v, 48)));
  }
  if constexpr (L > 64) {
    unsigned* p = s[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = v;
    __syncthreads();
    v = op(op(p[0], p[1]), op(p[2], p[3]));
  }
  return v;
}
struct Least {
  __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return min(a, b); }
};
struct Most {
  __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return max(a, b); }
};
struct Any {
  __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return a | b; }
};
struct Sum {
  __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }
};

// The fewest low bits, as a mask, that number n things.
constexpr unsigned low_bits(int n) {
  unsigned b = 1;
  while ((int)b < n) b *= 2;
  return b - 1;
}

template <int R> constexpr int column(int i, int v, int L, int lane) {
  return ((i / v) * L + lane) * v + i % v;
}

// One choice of a row.  `chosen` (label, weight): what the gradient goes by, apart from the
// caller's tensors, which a router edits (labels over a capacity become -1).
__device__ __forceinline__ void store_choice(int at, float weight, int64_t i, float* __restrict__ w,
                                             int* __restrict__ labels, int2* __restrict__ chosen) {
  w[i] = weight;
  labels[i] = at;
  if (chosen) chosen[i] = make_int2(at, __float_as_int(weight));
}

template <typename T, int L, int R, int TAIL, bool MASKED>
__global__ __launch_bounds__(GATE_BLOCK) void gate_kernel(const T* __restrict__ scores, int64_t ld,
                                                          Mask mask, int64_t n, int K, int k,
                                                          bool normalize, float* __restrict__ w,
                                                          int* __restrict__ labels,
                                                          int2* __restrict__ chosen,
                                                          float* __restrict__ stat) {
  constexpr int V = Vec<T>::N;
  constexpr unsigned INDEX = low_bits(L * R);  // the bits of a column
  constexpr unsigned NONE = 0x007fffffu;       // the place of -inf: it and less is not chosen
  __shared__ unsigned s_all[2][4];
  int turn = 0;
  const int lane = threadIdx.x % L;
  const int64_t row = block_index() * (GATE_BLOCK / L) + threadIdx.x / L;
  if (row >= n) return;  // whole groups of L; L >= 64: a whole wave or block
  const T* src = scores + row * ld;
  Raw16 raw[R / V];
  MaskVec<V, TAIL> ok[R / V];
#pragma unroll
  for (int i = 0; i < R / V; ++i) {
    raw[i] = RowVec<T, TAIL>::fetch(src, (i * L + lane) * V, K);
    if (MASKED) ok[i].fetch(mask, row, (i * L + lane) * V, K);
  }
  float v[R];
  unsigned num[R], lost = 0;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < R / V; ++i) {
    const int c = (i * L + lane) * V;
    float f[V];
    RowVec<T, TAIL>::value(raw[i], c, K, f);
    const unsigned in = MASKED ? ok[i].bits(mask, row, c, K) : 0u;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool there = MASKED ? (in >> j & 1) != 0 : c + (TAIL == TAIL_NONE ? 0 : j) < K;
      v[i * V + j] = f[j];
      // order_of() but for NaN, which is put right below where there is one
      const unsigned b = __float_as_uint(f[j] + 0.f);
      const unsigned key = b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
      nan |= there && f[j] != f[j];
      if (sizeof(T) == 4) lost |= b & INDEX;
      num[i * V + j] = there ? (key & ~INDEX) | (INDEX - (unsigned)(c + j)) : 0u;
    }
  }
  if (__any(nan)) {
    // by what is allowed, not by the number so far: that of a NaN of all ones may be 0
#pragma unroll
    for (int i = 0; i < R / V; ++i) {
      const int c = (i * L + lane) * V;
      const unsigned in = MASKED ? ok[i].bits(mask, row, c, K) : 0u;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool there = MASKED ? (in >> j & 1) != 0 : c + j < K;
        if (there && v[i * V + j] != v[i * V + j])
          num[i * V + j] = ~INDEX | (INDEX - (unsigned)(c + j));
      }
    }
  }
  if (sizeof(T) == 4) lost = group_all<L>(lost, Any(), s_all, turn);
  unsigned limit = 0xffffffffu, before = 0, unsure = 0;
  int at = -1;
  bool left = true;
  const int rounds = sizeof(T) == 4 ? k + 1 : k;
  for (int j = 0; j < rounds; ++j) {
    unsigned d = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < R; ++i) d = min(d, limit - num[i]);
    d = group_all<L>(d, Least(), s_all, turn);
    const unsigned best = limit - d;
    left = left && best > NONE;
    if (sizeof(T) == 4) unsure |= j > 0 && left && ((best ^ before) & ~INDEX) == 0;
    before = best;
    limit = best - 1;
    if (lane == j && j < k && left) at = (int)(INDEX - (best & INDEX));
  }
  if (sizeof(T) == 4) {
    // the same for a row's threads; a wave of several rows does all of them again
    const bool again = L > 64 ? (unsure && lost) : __any(unsure && lost);
    if (again) {
      unsigned key[R];
#pragma unroll
      for (int i = 0; i < R; ++i) key[i] = order_of(v[i], num[i] > NONE);
      at = -1;
      for (int j = 0; j < k; ++j) {
        unsigned b = 0;
        int bi = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (key[i] > b) {
            b = key[i];
            bi = column<R>(i, V, L, lane);
          }
        }
        const unsigned most = group_all<L>(b, Most(), s_all, turn);
        bi = (int)group_all<L>(b == most ? (unsigned)bi : 0x7fffffffu, Least(), s_all, turn);
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (column<R>(i, V, L, lane) == bi) key[i] = 0;
        if (lane == j && most) at = bi;
      }
    }
  }
  // the chosen are in lanes 0 .. k - 1 of the row
  const float mine = at >= 0 ? up(src[at]) : 0.f;
  float first = mine;
  if constexpr (L > 64) {
    unsigned* p = s_all[turn];
    turn ^= 1;
    if (threadIdx.x == 0) p[0] = __float_as_uint(mine);
    __syncthreads();
    first = __uint_as_float(p[0]);
  } else {
    first = __shfl(mine, (threadIdx.x & 63) / L * L, 64);
  }
  const float e = at >= 0 ? expf(mine - first) : 0.f;
  float sum = normalize ? e : 0.f;
  if (!normalize) {
#pragma unroll
    for (int i = 0; i < R; ++i) sum += num[i] > NONE ? expf(v[i] - first) : 0.f;
  }
  sum = __uint_as_float(group_all<L>(__float_as_uint(sum), Sum(), s_all, turn));
  if (lane < k) store_choice(at, at >= 0 ? e / sum : 0.f, row * k + lane, w, labels, chosen);
  if (stat && lane == 0) {
    stat[2 * row] = first;
    stat[2 * row + 1] = at >= 0 ? 1.f / sum : 0.f;
  }
}

// More clusters: a block per row takes 8192 scores at a time into its registers and their
// best into a list of the k best so far, lane j of each wave holding the j-th: after the
// first part few are better than its last.  65536 clusters, 1024 rows bf16, k = 8: 92 us (1.5
// TB/s: a part is loaded when the one before it is done), 840 with the row read again in every
// round.
template <typename T, int TAIL, bool MASKED>
__global__ __launch_bounds__(GATE_BLOCK) void gate_wide_kernel(
    const T* __restrict__ scores, int64_t ld, Mask mask, int64_t n, int K, int k, bool normalize,
    float* __restrict__ w, int* __restrict__ labels, int2* __restrict__ chosen,
    float* __restrict__ stat) {
  constexpr int V = Vec<T>::N, L = GATE_BLOCK, R = 32;
  __shared__ unsigned s_all[2][4];
  int turn = 0;
  const int64_t row = block_index();
  if (row >= n) return;
  const T* src = scores + row * ld;
  const int lane = threadIdx.x & 63;
  unsigned list = 0, last = 0, top = 0;  // this lane's entry, the k-th, the first
  int at = -1;
  float total = 0.f;
  for (int c0 = 0; c0 < K; c0 += L * R) {
    Raw16 raw[R / V];
    MaskVec<V, TAIL> ok[R / V];
#pragma unroll
    for (int i = 0; i < R / V; ++i) {
      const int c = c0 + (i * L + (int)threadIdx.x) * V;
      raw[i] = RowVec<T, TAIL>::fetch(src, c, K);
      if (MASKED) ok[i].fetch(mask, row, c, K);
    }
    unsigned key[R];
#pragma unroll
    for (int i = 0; i < R / V; ++i) {
      const int c = c0 + (i * L + (int)threadIdx.x) * V;
      float f[V];
      RowVec<T, TAIL>::value(raw[i], c, K, f);
      const unsigned in = MASKED ? ok[i].bits(mask, row, c, K) : 0u;
#pragma unroll
      for (int j = 0; j < V; ++j)
        key[i * V + j] = order_of(f[j], MASKED ? (in >> j & 1) != 0 : c + j < K);
    }
    for (bool fresh = true;; fresh = false) {
      unsigned b = 0;
      int bi = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (key[i] > b) {
          b = key[i];
          bi = c0 + column<R>(i, V, L, threadIdx.x);
        }
      }
      const unsigned most = group_all<L>(b, Most(), s_all, turn);
      if (fresh && !normalize && most) {
        // the sum so far, to the largest score so far
        const unsigned now = max(top, most);
        if (top && now != top) total *= expf(score_of(top) - score_of(now));
#pragma unroll
        for (int i = 0; i < R; ++i) total += key[i] ? expf(score_of(key[i]) - score_of(now)) : 0.f;
      }
      // an equal score of an earlier part has the smaller index: it stays
      if (most <= last) break;
      bi = (int)group_all<L>(b == most ? (unsigned)bi : 0x7fffffffu, Least(), s_all, turn);
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (c0 + column<R>(i, V, L, threadIdx.x) == bi) key[i] = 0;
      const unsigned long long before = __ballot(list >= most);  // a prefix of the list
      const int place = __popcll(before);
      const unsigned up_list = (unsigned)__shfl_up((int)list, 1, 64);
      const int up_at = __shfl_up(at, 1, 64);
      if (lane > place) {
        list = up_list;
        at = up_at;
      } else if (lane == place) {
        list = most;
        at = bi;
      }
      if (lane >= k) list = 0;
      last = (unsigned)__builtin_amdgcn_readlane((int)list, k - 1);
      top = (unsigned)__builtin_amdgcn_readlane((int)list, 0);
    }
  }
  if (list == 0) at = -1;
  const float first = top ? score_of(top) : 0.f;
  const float e = list ? expf(score_of(list) - first) : 0.f;
  if (normalize)
    total = lanes_sum<64>(e);
  else
    total = __uint_as_float(group_all<L>(__float_as_uint(total), Sum(), s_all, turn));
  if ((int)threadIdx.x < k)
    store_choice(at, list ? e / total : 0.f, row * k + threadIdx.x, w, labels, chosen);
  if (stat && threadIdx.x == 0) {
    stat[2 * row] = first;
    stat[2 * row + 1] = top ? 1.f / total : 0.f;
  }
}

// The gradient: L lanes per row, U vectors of each at a time.  What the chosen places get on
// top of the rest goes through LDS, so that every place is stored once (a second store of
// the chosen places would have to wait until the first have arrived).  65536 x 256 fp32:
// 16 to 17 us, bound by its 67 MB of stores and the latency of the few loads before them.
template <typename T, int L, int TAIL>
__global__ __launch_bounds__(GATE_BLOCK) void gate_bwd_kernel(
    const T* __restrict__ scores, int64_t ld, Mask mask, const int2* __restrict__ chosen,
    const float* __restrict__ stat, const float* __restrict__ dw,
    int64_t n, int K, int k, bool normalize, T* __restrict__ ds) {
  constexpr int V = Vec<T>::N, U = 16 / V;
  constexpr int PASS = L * V * U;  // columns
  __shared__ float more[GATE_BLOCK / L][PASS];
  const int lane = threadIdx.x % L;
  float* mine = more[threadIdx.x / L];
  const int64_t row = block_index() * (GATE_BLOCK / L) + threadIdx.x / L;
  if (row >= n) return;
  const int2 choice = lane < k ? chosen[row * k + lane] : make_int2(-1, 0);
  const float dj = lane < k ? dw[row * k + lane] : 0.f;
  const int at = choice.x;
  const float wj = __int_as_float(choice.y);
  const float top = normalize ? 0.f : stat[2 * row];
  const float inv = normalize ? 0.f : stat[2 * row + 1];
  const float mean = lanes_sum<L>(at >= 0 ? wj * dj : 0.f);
  const float gain = wj * (normalize ? dj - mean : dj);
  for (int c0 = 0; c0 < K; c0 += PASS) {
    Raw16 raw[U];
    MaskVec<V, TAIL> ok[U];
    if (!normalize) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        raw[u] = RowVec<T, TAIL>::fetch(scores + row * ld, c0 + (u * L + lane) * V, K);
        ok[u].fetch(mask, row, c0 + (u * L + lane) * V, K);
      }
    }
    // a row's part of LDS is its own lanes': they run together, in the order of the program
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) mine[(u * L + lane) * V + j] = 0.f;
    __builtin_amdgcn_wave_barrier();
    if (at >= c0 && at < c0 + PASS && at < K) mine[at - c0] = gain;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + (u * L + lane) * V;
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = mine[(u * L + lane) * V + j];
      if (!normalize) {
        float f[V];
        RowVec<T, TAIL>::value(raw[u], c, K, f);
        const unsigned in = ok[u].bits(mask, row, c, K);
#pragma unroll
        for (int j = 0; j < V; ++j)
          if ((in >> j & 1) && f[j] != -INFINITY) v[j] -= expf(f[j] - top) * inv * mean;
      }
      if (c < K) RowVec<T, TAIL>::store(ds + row * K, c, K, v);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace rows
}  // namespace tdc

using namespace tdc::rows;

int tdc_topk_gate(int dtype, const void* scores, int64_t ld, const uint8_t* mask, int64_t mask_rs,
                  int64_t mask_cs, int64_t n, int K, int k, int normalize, float* w, int* labels,
                  void* chosen, float* stat, hipStream_t stream) {
  if (n == 0) return 0;
  if (k < 1 || k > GATE_MAX_K || K < 1 || n > 0x7fffffff) return (int)hipErrorInvalidValue;
  const Mask m{mask, mask_rs, mask_cs};
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel, int lanes) {
      const int rows = GATE_BLOCK / lanes;
      hipLaunchKernelGGL(kernel, grid_of((n + rows - 1) / rows), dim3(GATE_BLOCK), 0,
                         stream, (const T*)scores, ld, m, n, K, k, normalize != 0, w, labels,
                         (int2*)chosen, stat);
    };
    return with_tail(K, Vec<T>::N, [&](auto tail) {
      constexpr int TAIL = decltype(tail)::value;
      auto one = [&](auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        if (K <= 64 && k <= 8)
          go(gate_kernel<T, 8, 8, TAIL, MASKED>, 8);
        else if (K <= 128)
          go(gate_kernel<T, 16, 8, TAIL, MASKED>, 16);
        else if (K <= 256)
          go(gate_kernel<T, 16, 16, TAIL, MASKED>, 16);
        else if (K <= 384)
          go(gate_kernel<T, 16, 24, TAIL, MASKED>, 16);
        else if (K <= 512)
          go(gate_kernel<T, 16, 32, TAIL, MASKED>, 16);
        else if (K <= 768)
          go(gate_kernel<T, 32, 24, TAIL, MASKED>, 32);
        else if (K <= 1024)
          go(gate_kernel<T, 32, 32, TAIL, MASKED>, 32);
        else if (K <= 1536)
          go(gate_kernel<T, 64, 24, TAIL, MASKED>, 64);
        else if (K <= 2048)
          go(gate_kernel<T, 64, 32, TAIL, MASKED>, 64);
        else if (K <= 4096)
          go(gate_kernel<T, 256, 16, TAIL, MASKED>, 256);
        else if (K <= 8192)
          go(gate_kernel<T, 256, 32, TAIL, MASKED>, 256);
        else
          go(gate_wide_kernel<T, TAIL, MASKED>, GATE_BLOCK);
      };
      if (mask)
        one(std::true_type());
      else
        one(std::false_type());
      TDC_CHECK_LAUNCH();
      return 0;
    });
  });
}

int tdc_topk_gate_bwd(int dtype, const void* scores, int64_t ld, const uint8_t* mask,
                      int64_t mask_rs, int64_t mask_cs, const void* chosen, const float* stat,
                      const float* dw, int64_t n, int K, int k, int normalize, void* ds,
                      hipStream_t stream) {
  if (n == 0) return 0;
  if (k < 1 || k > GATE_MAX_K || K < 1 || n > 0x7fffffff) return (int)hipErrorInvalidValue;
  const Mask m{mask, mask_rs, mask_cs};
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel, int lanes) {
      const int rows = GATE_BLOCK / lanes;
      hipLaunchKernelGGL(kernel, grid_of((n + rows - 1) / rows), dim3(GATE_BLOCK), 0,
                         stream, (const T*)scores, ld, m, (const int2*)chosen, stat, dw, n, K,
                         k, normalize != 0, (T*)ds);
    };
    return with_tail(K, Vec<T>::N, [&](auto tail) {
      constexpr int TAIL = decltype(tail)::value;
      if (K <= 256)
        go(gate_bwd_kernel<T, 16, TAIL>, 16);
      else if (K <= 512)
        go(gate_bwd_kernel<T, 32, TAIL>, 32);
      else
        go(gate_bwd_kernel<T, 64, TAIL>, 64);
      TDC_CHECK_LAUNCH();
      return 0;
    });
  });
}
