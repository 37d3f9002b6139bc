// Root-mean-square norm of rows with the residual's addition, to the rows' own type or to
// the block-scaled fp8 operand of the wide assignment, its gradient, and the way back from
// fp8.
//
//   h = x + r                   rounded to the rows' type: the caller keeps it, and the
//                               norm and its gradient are those of the kept row
//   rstd = 1 / sqrt(mean h^2 + eps);  y = h * rstd * w
//   gradient: g = dy * w, t = h * rstd, c = mean(g t):  dx = dr = rstd (g - t c) + dh,
//             dw = sum over rows of dy t
//   fp8: per 32 columns e = floor(log2 max|y|) - 7, q = e4m3(y 2^-e) (the layout of
//        quant_fp8_kernel), columns past the row's end are zero
//
// The sums are fp32, y, h and dx are rounded once; fp8 rows are fp64 up to q.  Bound by memory:
// the row lives in registers between its one read and its one write.  A row is spread over
// G threads with NV vectors of 16 bytes each; several rows share a wave when they are short,
// a block works on one row when it is long.  32768 x 1024 bf16 with a residual: 45 us (5.9 TB/s),
// the gradient 49 us (5.5 TB/s) and 4 us for dw.
#include "rows_common.h"

namespace tdc {
namespace rows {

constexpr int BLOCK = 256;

template <int G> constexpr int block_of() { return G > BLOCK ? G : BLOCK; }

// The weights of a vector of T: of its type, or N / 4 vectors of fp32.
template <typename T, int TAIL> struct WeightVec {
  static constexpr int N = Vec<T>::N;
  // a row of d >= N elements of T has d >= 4: its fp32 weights never are short alone
  using F = RowVec<float, TAIL>;
  Raw16 r[N / 4];
  __device__ __forceinline__ void fetch(const void* __restrict__ w, bool w32, int c, int d) {
    if (w == nullptr) return;
    if (w32) {
#pragma unroll
      for (int q = 0; q < N / 4; ++q) r[q] = F::fetch((const float*)w, c + 4 * q, d);
    } else {
      r[0] = RowVec<T, TAIL>::fetch((const T*)w, c, d);
    }
  }
  __device__ __forceinline__ void value(const void* w, bool w32, int c, int d, float (&v)[N]) const {
    if (w == nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = 1.f;
    } else if (w32) {
#pragma unroll
      for (int q = 0; q < N / 4; ++q) {
        float t[4];
        F::value(r[q], c + 4 * q, d, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * q + i] = t[i];
      }
    } else {
      RowVec<T, TAIL>::value(r[0], c, d, v);
    }
  }
};

// N values of one lane to e4m3 with the exponent of their block of 32 columns (32 / N
// neighbouring lanes).  The block's largest value lies in [2^7, 2^8) after the scaling: no
// saturation.  The scale byte e + 127 is 7 less than the largest value's exponent field.
template <int N>
__device__ __forceinline__ void store_fp8(uint8_t* __restrict__ q, uint8_t* __restrict__ s, int c,
                                          bool in, const float (&y)[N]) {
  float am = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) am = fmaxf(am, fabsf(y[i]));
  am = fmaxf(am, dpp<DPP_XOR1>(am));
  am = fmaxf(am, dpp<DPP_XOR2>(am));
  if constexpr (N == 4) am = fmaxf(am, dpp<DPP_HALF_MIRROR>(am));
  const int byte = max((int)(__float_as_uint(am) >> 23) - 7, 0);
  const float inv = __uint_as_float((unsigned)(254 - byte) << 23);
  int p[N / 4];
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    p[i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i] * inv, y[4 * i + 1] * inv, 0, false);
    p[i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2] * inv, y[4 * i + 3] * inv, p[i], true);
  }
  if (!in) return;
  if constexpr (N == 8)
    *reinterpret_cast<int2*>(q + c) = make_int2(p[0], p[1]);
  else
    *reinterpret_cast<int*>(q + c) = p[0];
  if (c % 32 == 0) s[c / 32] = (uint8_t)byte;
}

// x as a float of 21 bits whose last one also stands for all that follow it: rounding it
// further, to e4m3, gives what rounding x does, and its exponent is x's.
__device__ __forceinline__ float sticky_float(double x) {
  const unsigned rest = min((unsigned)__double2loint(x), 1u);
  return (float)__hiloint2double(__double2hiint(x) | (int)rest, 0);
}

// FP8: the row's sum and products are fp64.  A value next to the border of two e4m3 values
// lands a step of 1/8 away when fp32 puts it on the other side (110 of 201M values of a
// 262144 x 768 batch); in fp64 that takes a value within about 1e-15 of a border (none of
// them).  It stays bound by memory: 262144 x 768 bf16 with a residual in 270 us, 5.2 TB/s.
template <typename T, int G, int NV, int TAIL, bool FP8>
__global__ __launch_bounds__(block_of<G>()) void norm_kernel(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ r, int64_t ldr,
    const void* __restrict__ w, bool w32, int64_t n, int d, double eps, T* __restrict__ y,
    uint8_t* __restrict__ q, uint8_t* __restrict__ s, int dp, T* __restrict__ h,
    float* __restrict__ rstd) {
  constexpr int N = Vec<T>::N;
  using R = RowVec<T, TAIL>;
  using A = std::conditional_t<FP8, double, float>;
  __shared__ A part[2][16];
  int turn = 0;
  const int lane = threadIdx.x % G;
  const int64_t row = block_index() * (block_of<G>() / G) + threadIdx.x / G;
  if (row >= n) return;  // whole groups; G > 64: the block is one row of the grid
  Raw16 xr[NV], rr[NV];
  WeightVec<T, TAIL> wr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) xr[i] = R::fetch(x + row * ldx, (i * G + lane) * N, d);
  if (r) {
#pragma unroll
    for (int i = 0; i < NV; ++i) rr[i] = R::fetch(r + row * ldr, (i * G + lane) * N, d);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) wr[i].fetch(w, w32, (i * G + lane) * N, d);
  float v[NV][N];
  A sq = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + lane) * N;
    R::value(xr[i], c, d, v[i]);
    if (r) {
      float t[N];
      R::value(rr[i], c, d, t);
#pragma unroll
      for (int j = 0; j < N; ++j) v[i][j] = up(down<T>(v[i][j] + t[j]));
      R::store(h + row * d, c, d, v[i]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) sq = std::fma((A)v[i][j], (A)v[i][j], sq);
  }
  sq = group_sum<G>(sq, part, turn);
  const A rs = (A)1 / std::sqrt(sq / (A)d + (A)eps);
  if (rstd && lane == 0) rstd[row] = (float)rs;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + lane) * N;
    float t[N];
    wr[i].value(w, w32, c, d, t);
    if constexpr (FP8) {
      // the exponent's lanes all take part; a block of 32 is stored or not as a whole
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float f = sticky_float((double)v[i][j] * (double)t[j] * rs);
        // a mask, not a choice: that would be a branch around the fp64 products
        const int in = TAIL == TAIL_NONE ? c - d : c + j - d;
        t[j] = __uint_as_float(__float_as_uint(f) & (unsigned)(in >> 31));
      }
      store_fp8<N>(q + row * dp, s + row * (dp / 32), c, c < dp, t);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) t[j] = v[i][j] * rs * t[j];
      R::store(y + row * d, c, d, t);
    }
  }
}

// The gradient.  A block goes over rows with a stride of the grid and keeps its share of dw
// in registers; the shares of its row groups are added in LDS order and leave as one row of
// `part`, which dw_kernel sums: no atomics, the same order in every run.  50M elements with
// dw: fp32 112 to 133 us up to 8200 columns, 152 to 159 above (1024 x 4, which puts up to 27
// registers into scratch memory); 16 bits 54 to 65 up to 2048 columns, 76 to 126 above.
template <typename T, int G, int NV, int TAIL>
__global__ __launch_bounds__(block_of<G>()) void norm_bwd_kernel(
    const T* __restrict__ h, int64_t ldh, const float* __restrict__ rstd, const void* __restrict__ w,
    bool w32, const T* __restrict__ dy, int64_t lddy, const T* __restrict__ dh, int64_t lddh,
    int64_t n, int d, T* __restrict__ dx, float* __restrict__ part) {
  constexpr int N = Vec<T>::N;
  constexpr int GROUPS = block_of<G>() / G;
  using R = RowVec<T, TAIL>;
  __shared__ float sums[2][16];
  __shared__ float fold[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? NV * G * N : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  float dw[NV][N];
  WeightVec<T, TAIL> wr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    wr[i].fetch(w, w32, (i * G + lane) * N, d);
#pragma unroll
    for (int j = 0; j < N; ++j) dw[i][j] = 0.f;
  }
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + group; row < n;
       row += (int64_t)gridDim.x * GROUPS) {
    const float rs = rstd[row];
    Raw16 hr[NV], gr[NV], er[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * N;
      hr[i] = R::fetch(h + row * ldh, c, d);
      gr[i] = R::fetch(dy + row * lddy, c, d);
    }
    if (dh) {
#pragma unroll
      for (int i = 0; i < NV; ++i) er[i] = R::fetch(dh + row * lddh, (i * G + lane) * N, d);
    }
    float t[NV][N], g[NV][N];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * N;
      float wv[N];
      wr[i].value(w, w32, c, d, wv);
      R::value(hr[i], c, d, t[i]);
      R::value(gr[i], c, d, g[i]);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        t[i][j] *= rs;
        dw[i][j] = fmaf(g[i][j], t[i][j], dw[i][j]);
        g[i][j] *= wv[j];
        dot = fmaf(g[i][j], t[i][j], dot);
      }
    }
    if (!dx) continue;  // dw alone is asked for
    const float c1 = group_sum<G>(dot, sums, turn) / (float)d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * N;
      float o[N];
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = rs * (g[i][j] - t[i][j] * c1);
      if (dh) {
        float e[N];
        R::value(er[i], c, d, e);
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] += e[j];
      }
      R::store(dx + row * d, c, d, o);
    }
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * d;
  if constexpr (GROUPS > 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) fold[group][(i * G + lane) * N + j] = dw[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < d; c += block_of<G>()) {
      float a = 0.f;
      for (int k = 0; k < GROUPS; ++k) a += fold[k][c];
      out[c] = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = (i * G + lane) * N + j;
        if (c < d) out[c] = dw[i][j];
      }
  }
}

// dw[c] = sum of part[0..rows)[c].  A block takes 16 columns (one 64-byte line of each
// row), its 64 row groups every 64th row with 8 loads in flight each: 4 MiB of parts
// (1024 x 1024) take 4 us, with 64 columns per block (16 blocks only) 20 us.
constexpr int DW_COLS = 16, DW_ROWS = 64;
template <typename W>
__global__ __launch_bounds__(1024) void dw_kernel(const float* __restrict__ part, int rows, int d,
                                                  W* __restrict__ dw) {
  __shared__ float s[DW_ROWS][DW_COLS + 1];
  const int col = threadIdx.x % DW_COLS, group = threadIdx.x / DW_COLS;
  const int c = blockIdx.x * DW_COLS + col;
  float a = 0.f;
  if (c < d) {
#pragma unroll 8
    for (int k = group; k < rows; k += DW_ROWS) a += part[(int64_t)k * d + c];
  }
  s[group][col] = a;
  __syncthreads();
  // 64 groups to 4 by one thread per column and group, then to one
  if (threadIdx.x < 4 * DW_COLS) {
    a = 0.f;
#pragma unroll
    for (int k = 0; k < DW_ROWS / 4; ++k) a += s[group * (DW_ROWS / 4) + k][col];
    a += __shfl_xor(a, 16, 64);
    a += __shfl_xor(a, 32, 64);
    if (group == 0 && c < d) dw[c] = down<W>(a);
  }
}

// q 2^e: a row is spread over G threads as in the norm, all loads first.  2^e is built from
// its bits (scale 0 is the subnormal 2^-127), the product is exact.
template <typename T, int G, int NV, int TAIL>
__global__ __launch_bounds__(block_of<G>()) void dequant_kernel(const uint8_t* __restrict__ q,
                                                                const uint8_t* __restrict__ s,
                                                                int64_t n, int d, int dp,
                                                                T* __restrict__ out) {
  constexpr int N = Vec<T>::N;
  const int lane = threadIdx.x % G;
  const int64_t row = block_index() * (block_of<G>() / G) + threadIdx.x / G;
  if (row >= n) return;
  unsigned p[NV][N / 4], e[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = min((i * G + lane) * N, dp - N);
    __builtin_memcpy(p[i], __builtin_assume_aligned(q + row * dp + c, N), N);
    e[i] = s[row * (dp / 32) + c / 32];
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float f = __uint_as_float(e[i] ? e[i] << 23 : 0x00400000u);
    float v[N];
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      v[4 * k] = __builtin_amdgcn_cvt_f32_fp8((int)p[i][k], 0) * f;
      v[4 * k + 1] = __builtin_amdgcn_cvt_f32_fp8((int)p[i][k], 1) * f;
      v[4 * k + 2] = __builtin_amdgcn_cvt_f32_fp8((int)p[i][k], 2) * f;
      v[4 * k + 3] = __builtin_amdgcn_cvt_f32_fp8((int)p[i][k], 3) * f;
    }
    const int c = (i * G + lane) * N;
    if (c < d) RowVec<T, TAIL>::store(out + row * d, c, d, v);
  }
}

// Calls f(G, NV) for a row of `width` in vectors of N elements (16 bytes): threads and
// vectors of each that hold the row with few to spare (768 bf16: 32 x 3; as 64 x 2 with a
// quarter idle the fp8 norm took 20 % longer), within a wave, where the row's sum needs no
// barrier, up to 256 vectors (4 KiB).
template <int N, typename F> int with_shape(int width, F&& f) {
  const int vecs = (width + N - 1) / N;
#define TDC_SHAPE(G, NV) f(std::integral_constant<int, G>(), std::integral_constant<int, NV>())
  if (vecs <= 16) return TDC_SHAPE(16, 1);
  if (vecs <= 32) return TDC_SHAPE(32, 1);
  if (vecs <= 64) return TDC_SHAPE(64, 1);
  if (vecs <= 96) return TDC_SHAPE(32, 3);
  if (vecs <= 128) return TDC_SHAPE(64, 2);
  if (vecs <= 192) return TDC_SHAPE(64, 3);
  if (vecs <= 256) return TDC_SHAPE(64, 4);
  if (vecs <= 512) return TDC_SHAPE(256, 2);
  if (vecs <= 768) return TDC_SHAPE(256, 3);
  if (vecs <= 1024) return TDC_SHAPE(256, 4);
  if (vecs <= 2048) return TDC_SHAPE(1024, 2);
  if constexpr (N == 4)  // 16384 columns of fp32
    if (vecs <= 4096) return TDC_SHAPE(1024, 4);
#undef TDC_SHAPE
  return (int)hipErrorInvalidValue;
}

}  // namespace rows
}  // namespace tdc

using namespace tdc::rows;

int tdc_rms_norm(int dtype, const void* x, int64_t ldx, const void* r, int64_t ldr, const void* w,
                 int w32, int64_t n, int d, double eps, void* y, void* q, void* s, int dp, void* h,
                 float* rstd, hipStream_t stream) {
  if (n == 0) return 0;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int width = q ? dp : d;
    return with_shape<Vec<T>::N>(width, [&](auto g, auto nv) {
      constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
      constexpr int B = block_of<G>();
      const int64_t blocks = (n + B / G - 1) / (B / G);
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid_of(blocks), dim3(B), 0, stream, (const T*)x, ldx,
                           (const T*)r, ldr, w, w32 != 0, n, d, eps, (T*)y, (uint8_t*)q,
                           (uint8_t*)s, dp, (T*)h, rstd);
      };
      return with_tail(d, Vec<T>::N, [&](auto tail) {
        constexpr int TAIL = decltype(tail)::value;
        // an fp8 row has 256 columns or more, and a row shorter than a vector few threads
        if (q) {
          if constexpr (G > 16 && (TAIL != TAIL_SHORT || (G <= 64 && NV == 1)))
            go(norm_kernel<T, G, NV, TAIL, true>);
          else
            return (int)hipErrorInvalidValue;
        } else {
          if constexpr (TAIL != TAIL_SHORT || G == 16)
            go(norm_kernel<T, G, NV, TAIL, false>);
          else
            return (int)hipErrorInvalidValue;
        }
        TDC_CHECK_LAUNCH();
        return 0;
      });
    });
  });
}

// Rows of `part` that tdc_rms_norm_bwd fills (0: none needed).
int tdc_rms_norm_bwd_parts(int64_t n, int cus) {
  const int64_t most = (int64_t)cus * 4;
  return (int)(n < most ? n : most);
}

int tdc_rms_norm_bwd(int dtype, const void* h, int64_t ldh, const float* rstd, const void* w,
                     int w32, const void* dy, int64_t lddy, const void* dh, int64_t lddh,
                     int64_t n, int d, void* dx, float* part, int parts, void* dw,
                     hipStream_t stream) {
  if (parts < 1 && n > 0) return (int)hipErrorInvalidValue;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    int used = 0;
    if (n > 0) {
      const int rc = with_shape<Vec<T>::N>(d, [&](auto g, auto nv) {
        constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
        constexpr int B = block_of<G>();
        const int64_t blocks = (n + B / G - 1) / (B / G);
        used = (int)(blocks < parts ? blocks : parts);
        return with_tail(d, Vec<T>::N, [&](auto tail) {
          constexpr int TAIL = decltype(tail)::value;
          if constexpr (TAIL != TAIL_SHORT || G == 16)
            hipLaunchKernelGGL((norm_bwd_kernel<T, G, NV, TAIL>), dim3(used), dim3(B), 0, stream,
                               (const T*)h, ldh, rstd, w, w32 != 0, (const T*)dy, lddy, (const T*)dh,
                               lddh, n, d, (T*)dx, dw ? part : nullptr);
          TDC_CHECK_LAUNCH();
          return 0;
        });
      });
      if (rc) return rc;
    }
    if (dw) {
      const dim3 grid((unsigned)((d + DW_COLS - 1) / DW_COLS));
      if (w32)
        hipLaunchKernelGGL(dw_kernel<float>, grid, dim3(1024), 0, stream, part, used, d, (float*)dw);
      else
        hipLaunchKernelGGL(dw_kernel<T>, grid, dim3(1024), 0, stream, part, used, d, (T*)dw);
      TDC_CHECK_LAUNCH();
    }
    return 0;
  });
}

int tdc_dequant_fp8(int dtype, const void* q, const void* s, int64_t n, int d, int dp, void* out,
                    hipStream_t stream) {
  if (n == 0) return 0;
  if (dp % 32 != 0 || d > dp) return (int)hipErrorInvalidValue;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_shape<Vec<T>::N>(d, [&](auto g, auto nv) {
      constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
      constexpr int B = block_of<G>();
      const int64_t blocks = (n + B / G - 1) / (B / G);
      return with_tail(d, Vec<T>::N, [&](auto tail) {
        constexpr int TAIL = decltype(tail)::value;
        if constexpr (TAIL != TAIL_SHORT || G == 16)
          hipLaunchKernelGGL((dequant_kernel<T, G, NV, TAIL>), grid_of(blocks), dim3(B), 0,
                             stream, (const uint8_t*)q, (const uint8_t*)s, n, d, dp, (T*)out);
        TDC_CHECK_LAUNCH();
        return 0;
      });
    });
  });
}
