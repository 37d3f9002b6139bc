// Rows sorted by cluster and back, with weights, and the gradients.
//
// A plan is a stable counting sort of the N*k slots (slot n*k + j: row n's j-th label):
//   order[p] = slot at place p, pos[slot] = p, offsets[c] .. offsets[c + 1] = the places of
//   cluster c.  Slots whose label is not in [0, K) come after offsets[K], in slot order.
// The sort goes by digits of at most 11 bits: one pass up to K = 2047, two up to 2^22 - 1.
// A pass counts its digits per chunk of 1024 to 4096 slots, sums the counts over the chunks
// and scatters; ranks inside a chunk come from ballots, so that equal labels keep their order
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
constexpr int DIGIT_BITS = 11;
constexpr int MAX_DIGITS = 1 << DIGIT_BITS;
// Chunks whose counts every block sums itself; above, a kernel of its own does (131072
// labels of 257 keys: 16 us in two launches, 30 in three).
constexpr int DIRECT_CHUNKS = 64;

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

// The keys of a wave's 64 * PER slots, -1 past the end; the loads go out together.
template <int PER, typename In>
__device__ __forceinline__ void load_keys(const In& in, int64_t at, int64_t m, int (&key)[PER]) {
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = in.key(min(at + i * 64, m - 1));
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = at + i * 64 < m ? key[i] : -1;
}

// hist[digit * ds + chunk * cs] = slots of the chunk with that digit
template <typename In, int PER>
__global__ __launch_bounds__(SORT_BLOCK) void sort_count_kernel(In in, int64_t m, int shift,
                                                                int bits, int digits,
                                                                int* __restrict__ hist,
                                                                int64_t ds, int64_t cs) {
  __shared__ int cnt[MAX_DIGITS];
  const int mask = (1 << bits) - 1;
  int key[PER];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  load_keys<PER>(in, (int64_t)blockIdx.x * (SORT_BLOCK * PER) + wave * (64 * PER) + lane, m, key);
  for (int d = threadIdx.x; d < digits; d += SORT_BLOCK) cnt[d] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (key[i] >= 0) atomicAdd(&cnt[(key[i] >> shift) & mask], 1);
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += SORT_BLOCK) hist[d * ds + blockIdx.x * cs] = cnt[d];
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

// Places of a chunk's slots.  One chunk: its own counts are the totals, and the whole sort
// is this launch.  A few: every block sums the counts hist[chunk][digit].  Many (totals):
// sort_scan_kernel has summed hist[digit][chunk].
template <typename In, int PER, bool LAST>
__global__ __launch_bounds__(SORT_BLOCK) void sort_scatter_kernel(
    In in, int64_t m, int shift, int digits, int bits, const int* __restrict__ hist,
    const int* __restrict__ totals, int2* __restrict__ pairs, int* __restrict__ keys,
    int* __restrict__ order, int* __restrict__ pos, int* __restrict__ starts) {
  __shared__ int cnt[SORT_WAVES][MAX_DIGITS];
  __shared__ int s_total[MAX_DIGITS], s_before[MAX_DIGITS];
  __shared__ int s_wave[SORT_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int chunk = blockIdx.x, chunks = gridDim.x, mask = (1 << bits) - 1;
  // a wave owns 64 * PER slots in a row, 64 of them at a time
  const int64_t first = (int64_t)chunk * (SORT_BLOCK * PER) + wave * (64 * PER);
  int key[PER];
  if (m > 0) load_keys<PER>(in, first + lane, m, key);
  for (int d = threadIdx.x; d < digits; d += SORT_BLOCK) {
#pragma unroll
    for (int i = 0; i < SORT_WAVES; ++i) cnt[i][d] = 0;
    s_total[d] = 0;
    s_before[d] = 0;
  }
  __syncthreads();
  if (m > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] >= 0) atomicAdd(&cnt[wave][(key[i] >> shift) & mask], 1);
  }
  if (totals) {
    for (int d = threadIdx.x; d < digits; d += SORT_BLOCK) {
      s_total[d] = totals[d];
      s_before[d] = hist[(int64_t)d * chunks + chunk];
    }
  } else if (chunks > 1) {
    // pieces of 64 digits by 16 chunks, all of a piece's loads in flight: the counts come from
    // other XCDs, a microsecond away.  The waves share the chunks first, then the digits.
    constexpr int DEEP = DIRECT_CHUNKS / SORT_WAVES;
    const int parts = chunks <= DEEP ? 1 : chunks <= 2 * DEEP ? 2 : SORT_WAVES;
    const int c = (wave & (parts - 1)) * DEEP;
    for (int d = wave / parts * 64 + lane; d < digits; d += SORT_WAVES / parts * 64) {
      int v[DEEP], t = 0, before = 0;
#pragma unroll
      for (int i = 0; i < DEEP; ++i) v[i] = hist[min(c + i, chunks - 1) * digits + d];
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        t += c + i < chunks ? v[i] : 0;
        before += c + i < chunk ? v[i] : 0;
      }
      atomicAdd(&s_total[d], t);
      atomicAdd(&s_before[d], before);
    }
  }
  __syncthreads();
  // first place of each digit, then of each wave's part of it
  const int own = (digits + SORT_BLOCK - 1) / SORT_BLOCK;  // digits of a thread, in a row
  int sum = 0;
  for (int i = 0; i < own; ++i) {
    const int d = threadIdx.x * own + i;
    if (d < digits) {
      if (chunks == 1) {
        int t = 0;
#pragma unroll
        for (int q = 0; q < SORT_WAVES; ++q) t += cnt[q][d];
        s_total[d] = t;
      }
      sum += s_total[d];
    }
  }
  int total;
  int at = block_scan(sum, s_wave, total);
  for (int i = 0; i < own; ++i) {
    const int d = threadIdx.x * own + i;
    if (d < digits) {
      if (starts && chunk == 0) starts[d] = at;
      int next = at + s_before[d];
#pragma unroll
      for (int q = 0; q < SORT_WAVES; ++q) {
        const int c = cnt[q][d];
        cnt[q][d] = next;
        next += c;
      }
      at += s_total[d];
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (first + i * 64 >= m) break;  // the same for the wave
    const int64_t slot_at = first + i * 64 + lane;
    const bool in_range = slot_at < m;
    const int d = in_range ? (key[i] >> shift) & mask : 0;
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
      // always, unless someone writes the labels meanwhile
      if ((unsigned)p < (unsigned)m) {
        pos[slot_at] = p;  // of what stood here before the pass
        if constexpr (LAST) {
          order[p] = in.slot(slot_at);
          if (keys) keys[p] = key[i];
        } else {
          pairs[p] = make_int2(key[i], in.slot(slot_at));
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The end of a sort in two passes.  pos[slot] holds the place after the first pass, `moved`
// where the second put what stood there: the slot's place is read through both (1M labels:
// 16 us for the second scatter and 11 here; 31 and 5 where it wrote pos[slot] itself, 4 bytes
// at a time all over).  offsets[c] is the first place whose key is c or more, looked
// up by halving among the places of its upper digit (`starts`): as long for clusters that
// are all empty as for full ones.
__global__ __launch_bounds__(SORT_BLOCK) void sort_finish_kernel(
    const int* __restrict__ keys, const int* __restrict__ moved, const int* __restrict__ starts,
    int shift, int digits, int m, int K, int* __restrict__ pos, int* __restrict__ offsets) {
  const int64_t i = (int64_t)blockIdx.x * SORT_BLOCK + threadIdx.x;
  if (i < m) pos[i] = moved[min((unsigned)pos[i], (unsigned)m - 1)];
  if (i > K) return;
  int lo = 0, hi = 0;
  if (m > 0) {
    const int d = (int)(i >> shift);
    lo = starts[d];
    hi = d + 1 < digits ? starts[d + 1] : m;
  }
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (keys[mid] < i)
      lo = mid + 1;
    else
      hi = mid;
  }
  offsets[i] = lo;
}

// ------------------------------------------------------------------ rows
__device__ __forceinline__ int kept_places(const int* offsets, int K, int64_t m) {
  const int t = offsets[K];
  return t < 0 ? 0 : (t > m ? (int)m : t);
}

// The three kernels below move rows of whole 16-byte vectors.  L lanes (a power of two up to
// a wave) work on a row; a thread has U pieces of it in flight: U rows where a row is at
// most L vectors, else (LONG) U vectors of one row, L apart, the rest of the row being the
// next grid row's or pass's.  The last vector of a row that is no multiple is taken N
// elements before the row's end: what overlaps is written twice with the same values.
// Rows shorter than a vector (SHORT) go element by element.
template <typename T, bool SHORT> __device__ __forceinline__ Raw16 take(const T* row, int c, int d) {
  return RowVec<T, SHORT ? TAIL_SHORT : TAIL_NONE>::fetch(row, c, d);
}

// f(STREAM): whether the sorted rows are stored past the caches: where they are as large as
// the last level (256 MiB) they would only push out what the next kernel reads, and still be
// on their way to memory then (131072 x 1024 bf16: grouped and the gradient summed 134 us
// past the caches, 154 through them; grouped and read 422 us either way).  Smaller ones are
// kept for their reader (64 MiB grouped and read: 104 us past the caches, 85 through them).
template <typename F> int with_stream(int64_t bytes, F&& f) {
  if (bytes >= (int64_t)256 << 20) return f(std::true_type());
  return f(std::false_type());
}

template <typename T, bool SHORT, bool STREAM = false>
__device__ __forceinline__ void put(T* row, int c, int d, const Raw16& r) {
  if constexpr (SHORT) {
    T t[Vec<T>::N];
    __builtin_memcpy(t, &r, 16);
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i)
      if (c + i < d) row[c + i] = t[i];
  } else {
    T* p = row + min(c, d - Vec<T>::N);
    if constexpr (STREAM) {
      typedef unsigned Words __attribute__((ext_vector_type(4), aligned(2)));
      const Words v = {r.w[0], r.w[1], r.w[2], r.w[3]};
      __builtin_nontemporal_store(v, reinterpret_cast<Words*>(p));
    } else {
      store16(p, r);
    }
  }
}

// Row and column of a thread's piece u; false where there is none.
template <int N, int U, bool LONG>
__device__ __forceinline__ bool piece(int u, int L, int64_t n, int d, int pass, int64_t& row, int& c) {
  const int lane = threadIdx.x & (L - 1), group = threadIdx.x / L, groups = 256 / L;
  if (LONG) {
    row = block_index() * groups + group;
    c = ((pass * U + u) * L + lane) * N;
  } else {
    row = (block_index() * U + u) * groups + group;
    c = lane * N;
  }
  return row < n && c < d;
}

// xg: every row is read once and written to the places of its k slots (zeros behind the
// kept ones), J slots at a time: their places are all there before the first store, as a
// wait for a load waits for the stores before it too (rows of 2 KiB with k = 8, 302 MB: 47 us
// through the caches, 86 with a place fetched before each store; 61 us, 5.0 TB/s, past the
// caches, which pays in the next kernel).
template <typename T, int J, int U, bool LONG, bool SHORT, bool STREAM>
__global__ __launch_bounds__(256) void group_kernel(const T* __restrict__ x, int64_t ldx, int64_t n,
                                                    int k, int d, const int* __restrict__ offsets,
                                                    int K, const int* __restrict__ pos,
                                                    T* __restrict__ out, int L) {
  constexpr int N = Vec<T>::N;
  const int kept = kept_places(offsets, K, n * k);
  Raw16 v[U];
  int64_t row[U];
  int c[U];
  bool in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    in[u] = piece<N, U, LONG>(u, L, n, d, blockIdx.z, row[u], c[u]);
    v[u] = take<T, SHORT>(x + (in[u] ? row[u] : 0) * ldx, in[u] ? c[u] : 0, d);
  }
  for (int j0 = 0; j0 < k; j0 += J) {
    int p[U][J];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int at = pos[(in[u] ? row[u] : 0) * k + min(j0 + j, k - 1)];
        p[u][j] = in[u] && j0 + j < k ? at : -1;
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < J; ++j)
        if ((unsigned)p[u][j] < (unsigned)(n * k))
          put<T, SHORT, STREAM>(out + (int64_t)p[u][j] * d, c[u], d, if_kept(p[u][j] < kept, v[u]));
  }
}

template <typename T>
__device__ __forceinline__ float weight_at(const void* __restrict__ w, bool w32, int64_t slot) {
  return w ? (w32 ? ((const float*)w)[slot] : up(((const T*)w)[slot])) : 1.f;
}

// out[n] = sum_j w[n, j] y[pos[n, j]] (w null: 1), J slots at a time.  A slot without a
// place reads the row at place 0 (there is one) and drops it: the J * U loads have no
// branch between them.  131072 x 1024 bf16 to 16384 rows: 55 us, 5.5 TB/s.
template <typename T, int J, int U, bool LONG, bool SHORT>
__global__ __launch_bounds__(256) void combine_kernel(const T* __restrict__ y, int64_t ldy, int64_t n,
                                                      int k, int d, const int* __restrict__ offsets,
                                                      int K, const int* __restrict__ pos,
                                                      const void* __restrict__ w, bool w32,
                                                      T* __restrict__ out, int L) {
  constexpr int N = Vec<T>::N;
  const unsigned kept = (unsigned)kept_places(offsets, K, n * k);
  int64_t row[U];
  int c[U];
  bool in[U];
  float a[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    in[u] = piece<N, U, LONG>(u, L, n, d, blockIdx.z, row[u], c[u]);
    if (!in[u]) {
      row[u] = 0;
      c[u] = 0;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) a[u][i] = 0.f;
  }
  for (int j0 = 0; j0 < k; j0 += J) {
    unsigned p[U][J];
    float wj[U][J];
    Raw16 v[U][J];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int64_t slot = row[u] * k + min(j0 + j, k - 1);
        p[u][j] = j0 + j < k ? (unsigned)pos[slot] : kept;
        wj[u][j] = weight_at<T>(w, w32, slot);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < J; ++j)
        v[u][j] = take<T, SHORT>(y + (int64_t)(p[u][j] < kept ? p[u][j] : 0) * ldy, c[u], d);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float f[N];
        unpack<T>(v[u][j], f);
        if (p[u][j] < kept)
#pragma unroll
          for (int i = 0; i < N; ++i) a[u][i] = fmaf(wj[u][j], f[i], a[u][i]);
      }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (in[u]) put<T, SHORT>(out + row[u] * d, c[u], d, pack<T>(a[u]));
}

// Gradients of a row's slots, J at a time: dy[p] = w dout[row], dw = <dout[row], y[p]>;
// either may be left out (dy null, y null).  The row's passes and the sum over its lanes
// are this thread group's, so dw needs no atomics.  131072 x 1024 bf16: 120 us, 4.8 TB/s
// (y, dout and dy once each).
template <typename T, int J, int U, bool LONG, bool SHORT, bool STREAM>
__global__ __launch_bounds__(256) void combine_bwd_kernel(
    const T* __restrict__ dout, int64_t lddo, const T* __restrict__ y, int64_t ldy, int64_t n, int k,
    int d, const int* __restrict__ offsets, int K, const int* __restrict__ pos,
    const void* __restrict__ w, bool w32, T* __restrict__ dy, void* __restrict__ dw, int L) {
  constexpr int N = Vec<T>::N;
  const unsigned m = (unsigned)(n * k);
  const unsigned kept = (unsigned)kept_places(offsets, K, n * k);
  const int lane = threadIdx.x & (L - 1);
  const int passes = LONG ? (d + U * L * N - 1) / (U * L * N) : 1;
  for (int j0 = 0; j0 < k; j0 += J) {
    constexpr int S = LONG ? 1 : U;  // rows of a thread
    float dot[S][J];
    unsigned p[S][J];
    float wj[S][J];
#pragma unroll
    for (int u = 0; u < S; ++u) {
      int64_t row;
      int c;
      // every lane of the row takes its places, those without a column too
      piece<N, U, LONG>(u, L, n, d, 0, row, c);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int64_t slot = (row < n ? row : 0) * k + min(j0 + j, k - 1);
        p[u][j] = row < n && j0 + j < k ? (unsigned)pos[slot] : m;
        wj[u][j] = weight_at<T>(w, w32, slot);
        dot[u][j] = 0.f;
      }
    }
    for (int pass = 0; pass < passes; ++pass) {
      int64_t row[U];
      int c[U];
      bool in[U];
      Raw16 g[U], v[U][J];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        in[u] = piece<N, U, LONG>(u, L, n, d, pass, row[u], c[u]);
        g[u] = take<T, SHORT>(dout + (in[u] ? row[u] : 0) * lddo, in[u] ? c[u] : 0, d);
      }
      if (y) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const unsigned at = p[LONG ? 0 : u][j];
            v[u][j] = take<T, SHORT>(y + (int64_t)(at < kept ? at : 0) * ldy, in[u] ? c[u] : 0, d);
          }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[N];
        unpack<T>(g[u], f);
        // elements that the vector before this one has counted already
        const int twice = SHORT ? 0 : c[u] - min(c[u], d - N);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const unsigned at = p[LONG ? 0 : u][j];
          const float ww = wj[LONG ? 0 : u][j];
          if (dy && in[u] && at < m) {
            float o[N];
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = ww * f[i];
            put<T, SHORT, STREAM>(dy + (int64_t)at * d, c[u], d, if_kept(at < kept, pack<T>(o)));
          }
          if (y && in[u] && at < kept) {
            float q[N];
            unpack<T>(v[u][j], q);
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) t = fmaf(i >= twice ? f[i] : 0.f, i >= twice ? q[i] : 0.f, t);
            dot[LONG ? 0 : u][j] += t;
          }
        }
      }
    }
    if (!dw) continue;
#pragma unroll
    for (int u = 0; u < S; ++u) {
      int64_t row;
      int c;
      piece<N, U, LONG>(u, L, n, d, 0, row, c);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float t = dot[u][j];
        for (int o = L / 2; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
        if (lane == 0 && row < n && j0 + j < k) {
          if (w32)
            ((float*)dw)[row * k + j0 + j] = t;
          else
            ((T*)dw)[row * k + j0 + j] = down<T>(t);
        }
      }
    }
  }
}

// Lanes of a row: as many as it has 16-byte vectors, a power of two up to a wave.
inline int lanes_for(int d, int v) {
  const int vecs = (d + v - 1) / v;
  int l = 4;
  while (l < 64 && l < vecs) l *= 2;
  return l;
}

// f(LONG, SHORT) for rows of d elements in vectors of v.
template <typename F> int with_rows(int d, int v, F&& f) {
  if (d < v) return f(std::false_type(), std::true_type());
  if (d > 64 * v) return f(std::true_type(), std::false_type());
  return f(std::false_type(), std::false_type());
}

// Grid of U pieces per thread: rows, and (LONG) the passes over a row as its third dimension.
inline dim3 grid_for(int64_t n, int d, int v, int L, int U, bool is_long, bool passes) {
  const int64_t rows = (int64_t)(256 / L) * (is_long ? 1 : U);
  return grid_of((n + rows - 1) / rows,
                 is_long && passes ? ((unsigned)d + U * L * v - 1) / (U * L * v) : 1);
}

// f(J, U): slots at once and pieces of a thread, 8 to 16 loads in flight.
template <typename F> int with_slots(int k, F&& f) {
#define TDC_SLOTS(J, U) f(std::integral_constant<int, J>(), std::integral_constant<int, U>())
  if (k == 1) return TDC_SLOTS(1, 4);
  if (k == 2) return TDC_SLOTS(2, 4);
  if (k <= 4) return TDC_SLOTS(4, 2);
  return TDC_SLOTS(8, 2);
#undef TDC_SLOTS
}

struct SortShape {
  int low, high;  // bits of the first and the second pass's digit (0: one pass)
  // slots per thread: one block sorts up to 2048 alone; from there enough chunks to fill the
  // chip (1M labels, 65536 clusters: 63 us with 8, 66 with 16), then few enough counts (3M:
  // 154 us)
  int per;
  int64_t chunks;
  int digits[2];

  SortShape(int64_t m, int K) {
    int bits = 1;
    while ((K >> bits) != 0) ++bits;  // keys 0..K
    low = bits <= DIGIT_BITS ? bits : (bits + 1) / 2;
    high = bits - low;
    if (m <= SORT_BLOCK * 8)
      per = m <= SORT_BLOCK * 4 ? 4 : 8;
    else
      per = m <= SORT_BLOCK * 4 * DIRECT_CHUNKS ? 4 : m <= (2 << 20) ? 8 : 16;
    chunks = std::max<int64_t>(1, (m + SORT_BLOCK * per - 1) / (SORT_BLOCK * per));
    digits[0] = high ? 1 << low : K + 1;
    digits[1] = high ? (K >> low) + 1 : 0;
  }
  int64_t most() const { return std::max(digits[0], digits[1]); }
  // Whether every block sums the chunks' counts itself, which saves a launch, or a kernel of
  // its own does.
  bool direct() const { return chunks <= DIRECT_CHUNKS && (most() <= 512 || chunks <= 16); }
  // counts of a pass, totals behind them, to whole int2
  int64_t count_words() const {
    return chunks == 1 ? 0 : (most() * (chunks + (direct() ? 0 : 1)) + 1) / 2 * 2;
  }
};

}  // namespace rows
}  // namespace tdc

using namespace tdc::rows;

// int32 words of scratch of a plan (counts, totals and, with two passes, pairs, keys, moves and starts).
int64_t tdc_group_plan_work(int64_t m, int K) {
  const SortShape s(m, K);
  return s.count_words() + (s.high ? 4 * m + s.digits[1] : 0);
}

int tdc_group_plan(int wide_labels, const void* labels, int64_t m, int K, int* work, int* order,
                   int* pos, int* offsets, hipStream_t stream) {
  if (K < 1 || K >= (1 << 22) || m < 0 || m > 0x7ffffffe) return (int)hipErrorInvalidValue;
  const SortShape s(m, K);
  int* hist = s.chunks > 1 ? work : nullptr;
  int* totals = s.chunks > 1 && !s.direct() ? work + s.most() * s.chunks : nullptr;
  int2* pairs = s.high ? reinterpret_cast<int2*>(work + s.count_words()) : nullptr;
  int* keys = s.high ? work + s.count_words() + 2 * m : nullptr;
  int* moved = s.high ? keys + m : nullptr;
  int* starts = s.high ? moved + m : nullptr;
  const dim3 grid((unsigned)s.chunks), block(SORT_BLOCK);
  auto pass = [&](auto in, auto last, auto per, int shift, int bits, int digits) {
    constexpr bool LAST = decltype(last)::value;
    constexpr int PER = decltype(per)::value;
    using In = decltype(in);
    if (hist) {
      hipLaunchKernelGGL((sort_count_kernel<In, PER>), grid, block, 0, stream, in, m, shift, bits,
                         digits, hist, totals ? s.chunks : 1, totals ? 1 : (int64_t)digits);
      TDC_CHECK_LAUNCH();
    }
    if (totals) {
      hipLaunchKernelGGL(sort_scan_kernel, dim3(digits), block, 0, stream, hist, (int)s.chunks,
                         totals);
      TDC_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL((sort_scatter_kernel<In, PER, LAST>), grid, block, 0, stream, in, m, shift,
                       digits, bits, hist, totals, pairs, LAST ? keys : nullptr, order,
                       LAST && s.high ? moved : pos,
                       LAST ? (s.high ? starts : offsets) : nullptr);
    TDC_CHECK_LAUNCH();
    return 0;
  };
  auto all = [&](auto in, auto per) {
    if (s.high == 0) return pass(in, std::true_type(), per, 0, s.low, s.digits[0]);
    if (m > 0) {
      int rc = pass(in, std::false_type(), per, 0, s.low, s.digits[0]);
      if (rc == 0) rc = pass(FromPairs{pairs}, std::true_type(), per, s.low, s.high, s.digits[1]);
      if (rc) return rc;
    }
    const int64_t items = std::max<int64_t>(m, K + 1);
    hipLaunchKernelGGL(sort_finish_kernel, dim3((unsigned)((items + SORT_BLOCK - 1) / SORT_BLOCK)),
                       block, 0, stream, keys, moved, starts, s.low, s.digits[1], (int)m, K, pos,
                       offsets);
    TDC_CHECK_LAUNCH();
    return 0;
  };
  auto with_per = [&](auto in) {
    if (s.per == 4) return all(in, std::integral_constant<int, 4>());
    if (s.per == 8) return all(in, std::integral_constant<int, 8>());
    return all(in, std::integral_constant<int, 16>());
  };
  if (wide_labels) return with_per(FromLabels<int64_t>{(const int64_t*)labels, K});
  return with_per(FromLabels<int32_t>{(const int32_t*)labels, K});
}

int tdc_group_rows(int dtype, const void* x, int64_t ldx, int64_t n, int k, int d,
                   const int* offsets, int K, const int* pos, void* out, hipStream_t stream) {
  if (n == 0) return 0;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = Vec<T>::N;
    const int L = lanes_for(d, V);
    return with_rows(d, V, [&](auto lng, auto shrt) {
      return with_slots(k, [&](auto jj, auto uu) {
        constexpr bool LONG = decltype(lng)::value, SHORT = decltype(shrt)::value;
        constexpr int J = decltype(jj)::value, U = decltype(uu)::value;
        const dim3 grid = grid_for(n, d, V, L, U, LONG, true);
        return with_stream(n * k * d * (int64_t)sizeof(T), [&](auto past) {
          constexpr bool STREAM = decltype(past)::value;
          hipLaunchKernelGGL((group_kernel<T, J, U, LONG, SHORT, STREAM>), grid, dim3(256), 0, stream,
                             (const T*)x, ldx, n, k, d, offsets, K, pos, (T*)out, L);
          TDC_CHECK_LAUNCH();
          return 0;
        });
      });
    });
  });
}

int tdc_combine_rows(int dtype, const void* y, int64_t ldy, int64_t n, int k, int d,
                     const int* offsets, int K, const int* pos, const void* w, int w32, void* out,
                     hipStream_t stream) {
  if (n == 0) return 0;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = Vec<T>::N;
    const int L = lanes_for(d, V);
    return with_rows(d, V, [&](auto lng, auto shrt) {
      return with_slots(k, [&](auto jj, auto uu) {
        constexpr bool LONG = decltype(lng)::value, SHORT = decltype(shrt)::value;
        constexpr int J = decltype(jj)::value, U = decltype(uu)::value;
        const dim3 grid = grid_for(n, d, V, L, U, LONG, true);
        hipLaunchKernelGGL((combine_kernel<T, J, U, LONG, SHORT>), grid, dim3(256), 0, stream,
                           (const T*)y, ldy, n, k, d, offsets, K, pos, w, w32 != 0, (T*)out, L);
        TDC_CHECK_LAUNCH();
        return 0;
      });
    });
  });
}

int tdc_combine_rows_bwd(int dtype, const void* dout, int64_t lddo, const void* y, int64_t ldy,
                         int64_t n, int k, int d, const int* offsets, int K, const int* pos,
                         const void* w, int w32, void* dy, void* dw, hipStream_t stream) {
  if (n == 0 || (!dy && !dw)) return 0;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = Vec<T>::N;
    const int L = lanes_for(d, V);
    return with_rows(d, V, [&](auto lng, auto shrt) {
      return with_slots(k, [&](auto jj, auto uu) {
        constexpr bool LONG = decltype(lng)::value, SHORT = decltype(shrt)::value;
        constexpr int J = decltype(jj)::value, U = decltype(uu)::value;
        const dim3 grid = grid_for(n, d, V, L, U, LONG, false);
        return with_stream(n * k * d * (int64_t)sizeof(T), [&](auto past) {
          constexpr bool STREAM = decltype(past)::value;
          hipLaunchKernelGGL((combine_bwd_kernel<T, J, U, LONG, SHORT, STREAM>), grid, dim3(256), 0,
                             stream, (const T*)dout, lddo, (const T*)y, ldy, n, k, d, offsets, K,
                             pos, w, w32 != 0, (T*)dy, dw, L);
          TDC_CHECK_LAUNCH();
          return 0;
        });
      });
    });
  });
}
