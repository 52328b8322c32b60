// Layer norm of rows, forward and backward, fp32 / fp16 / bf16:
//
//   xh = (x - mean) rstd,  y = xh w + b
//   g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Bound by memory: each pass reads its rows once. A row's values stay in the
// registers of `LPR` lanes (a part of a wave, a wave, or a whole workgroup), NV
// chunks of 16 bytes each, through the sums and the output; mean and variance
// are two sums over those registers (no difference of squares). A workgroup
// walks over rows with the weights, and in the backward pass the columns' sums,
// in registers; the workgroups' column sums are added up by a second kernel in
// a fixed order. All sums are fp32. Rows may start at any element: chunks are
// read with the alignment of one element, and the last one of a row whose width
// fills no whole chunk element by element.
#include "tj_common.h"

typedef __bf16 bf16_t;

namespace tj {
namespace {

struct NormArgs {
  const void *x, *dy, *w, *b;
  void *y, *dx, *dw, *db;
  float *mean, *rstd;   // [rows]; the forward pass may have none
  float* part;          // [workgroups, 2, cols]
  int64_t rows, cols, x_stride, y_stride, dy_stride, dx_stride;
  float eps;
  int w_is_f32;         // weight and bias are fp32 rather than T
  int n_parts;
};

template <typename T>
struct Chunk {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec unaligned __attribute__((aligned(sizeof(T))));

  __device__ __forceinline__ static void load(float (&f)[N], const T* p, int left) {
    if (left >= N) {
      const vec v = *reinterpret_cast<const unaligned*>(p);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = (float)v[j];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = j < left ? (float)p[j] : 0.f;
    }
  }
  __device__ __forceinline__ static void store(T* p, const float (&f)[N], int left) {
    if (left >= N) {
      vec v;
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = (T)f[j];
      *reinterpret_cast<unaligned*>(p) = v;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < left) p[j] = (T)f[j];
    }
  }
};

// Weights of a chunk's columns, fp32 or T.
template <typename T>
__device__ __forceinline__ void load_param(float (&f)[Chunk<T>::N], const void* p, int w_is_f32, int64_t col, int left,
                                           float none) {
#pragma unroll
  for (int j = 0; j < Chunk<T>::N; ++j) f[j] = none;
  if (p == nullptr || left <= 0) return;
  if (!w_is_f32) {
    Chunk<T>::load(f, reinterpret_cast<const T*>(p) + col, left);
    return;
  }
#pragma unroll
  for (int j = 0; j < Chunk<T>::N; ++j)
    if (j < left) f[j] = reinterpret_cast<const float*>(p)[col + j];
}

// Sum over the LPR lanes of a row; every lane gets it. Rows of a whole
// workgroup go through `red`, used alternately (parity) so that one barrier a
// sum is enough.
template <int LPR, int NS>
__device__ __forceinline__ void row_sums(float (&s)[NS], float* red, int& parity) {
  constexpr int W = LPR < kWave ? LPR : kWave;
#pragma unroll
  for (int m = W / 2; m > 0; m >>= 1)
#pragma unroll
    for (int i = 0; i < NS; ++i) s[i] += __shfl_xor(s[i], m);
  if constexpr (LPR > kWave) {
    constexpr int NW = LPR / kWave;
    float* r = red + parity * 2 * NW;
    parity ^= 1;
    if (threadIdx.x % kWave == 0)
#pragma unroll
      for (int i = 0; i < NS; ++i) r[i * NW + threadIdx.x / kWave] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      s[i] = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) s[i] += r[i * NW + k];
    }
  }
}

template <int LPR>
constexpr int norm_threads() { return LPR > 256 ? LPR : 256; }

template <typename T, int LPR, int NV>
__global__ __launch_bounds__(norm_threads<LPR>()) void norm_fwd_kernel(NormArgs a) {
  using C = Chunk<T>;
  constexpr int THREADS = norm_threads<LPR>(), RPB = THREADS / LPR;
  __shared__ float red[4 * (LPR > kWave ? LPR / kWave : 1)];
  const int lane = threadIdx.x % LPR;
  int parity = 0;
  float w[NV][C::N], b[NV][C::N];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t col = (int64_t)(lane + v * LPR) * C::N;
    load_param<T>(w[v], a.w, a.w_is_f32, col, (int)min(a.cols - col, (int64_t)C::N), 1.f);
    load_param<T>(b[v], a.b, a.w_is_f32, col, (int)min(a.cols - col, (int64_t)C::N), 0.f);
  }
  const float inv_n = 1.f / (float)a.cols;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + threadIdx.x / LPR;
    const bool on = row < a.rows;
    const T* xp = reinterpret_cast<const T*>(a.x) + (on ? row : 0) * a.x_stride;
    float x[NV][C::N], s[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int64_t col = (int64_t)(lane + v * LPR) * C::N;
      C::load(x[v], xp + col, on ? (int)min(a.cols - col, (int64_t)C::N) : 0);
#pragma unroll
      for (int j = 0; j < C::N; ++j) s[0] += x[v][j];
    }
    row_sums<LPR, 1>(s, red, parity);
    const float mean = s[0] * inv_n;
    s[0] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int64_t col = (int64_t)(lane + v * LPR) * C::N;
#pragma unroll
      for (int j = 0; j < C::N; ++j) {
        x[v][j] -= mean;
        if (col + j < a.cols) s[0] = fmaf(x[v][j], x[v][j], s[0]);
      }
    }
    row_sums<LPR, 1>(s, red, parity);
    const float rstd = 1.f / sqrtf(s[0] * inv_n + a.eps);
    if (on) {
      T* yp = reinterpret_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int64_t col = (int64_t)(lane + v * LPR) * C::N;
#pragma unroll
        for (int j = 0; j < C::N; ++j) x[v][j] = fmaf(x[v][j] * rstd, w[v][j], b[v][j]);
        C::store(yp + col, x[v], (int)min(a.cols - col, (int64_t)C::N));
      }
      if (a.mean != nullptr && lane == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
      }
    }
  }
}

template <typename T, int LPR, int NV>
__global__ __launch_bounds__(norm_threads<LPR>()) void norm_bwd_kernel(NormArgs a) {
  using C = Chunk<T>;
  constexpr int THREADS = norm_threads<LPR>(), RPB = THREADS / LPR;
  __shared__ float red[4 * (LPR > kWave ? LPR / kWave : 1)];
  __shared__ float cols[LPR < THREADS ? THREADS * C::N : 1];
  const int lane = threadIdx.x % LPR;
  int parity = 0;
  float w[NV][C::N], dw[NV][C::N], db[NV][C::N];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t col = (int64_t)(lane + v * LPR) * C::N;
    load_param<T>(w[v], a.w, a.w_is_f32, col, (int)min(a.cols - col, (int64_t)C::N), 1.f);
#pragma unroll
    for (int j = 0; j < C::N; ++j) dw[v][j] = db[v][j] = 0.f;
  }
  const float inv_n = 1.f / (float)a.cols;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + threadIdx.x / LPR;
    const bool on = row < a.rows;
    const T* xp = reinterpret_cast<const T*>(a.x) + (on ? row : 0) * a.x_stride;
    const T* gp = reinterpret_cast<const T*>(a.dy) + (on ? row : 0) * a.dy_stride;
    const float mean = on ? a.mean[row] : 0.f, rstd = on ? a.rstd[row] : 0.f;
    float x[NV][C::N], g[NV][C::N], s[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int64_t col = (int64_t)(lane + v * LPR) * C::N;
      const int left = on ? (int)min(a.cols - col, (int64_t)C::N) : 0;
      C::load(x[v], xp + col, left);
      C::load(g[v], gp + col, left);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int j = 0; j < C::N; ++j) {
        // Past the row's end dy reads as zero, so whatever xh is there adds nothing.
        x[v][j] = (x[v][j] - mean) * rstd;
        dw[v][j] = fmaf(g[v][j], x[v][j], dw[v][j]);
        db[v][j] += g[v][j];
        g[v][j] *= w[v][j];
        s[0] += g[v][j];
        s[1] = fmaf(g[v][j], x[v][j], s[1]);
      }
    }
    row_sums<LPR, 2>(s, red, parity);
    const float c0 = s[0] * inv_n, c1 = s[1] * inv_n;
    if (on && a.dx != nullptr) {
      T* dp = reinterpret_cast<T*>(a.dx) + row * a.dx_stride;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int64_t col = (int64_t)(lane + v * LPR) * C::N;
#pragma unroll
        for (int j = 0; j < C::N; ++j) g[v][j] = rstd * (g[v][j] - fmaf(x[v][j], c1, c0));
        C::store(dp + col, g[v], (int)min(a.cols - col, (int64_t)C::N));
      }
    }
  }
  if (a.part == nullptr) return;
  // The workgroup's column sums: lanes of different rows hold the same columns.
  float* out = a.part + (int64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float(&f)[C::N] = k == 0 ? dw[v] : db[v];
      if constexpr (LPR < THREADS) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < C::N; ++j) cols[j * THREADS + threadIdx.x] = f[j];
        __syncthreads();
        if (threadIdx.x < LPR)
#pragma unroll
          for (int j = 0; j < C::N; ++j) {
            f[j] = 0.f;
            for (int i = 0; i < RPB; ++i) f[j] += cols[j * THREADS + i * LPR + threadIdx.x];
          }
      }
      if (threadIdx.x < LPR) {
        const int64_t col = (int64_t)(lane + v * LPR) * C::N;
#pragma unroll
        for (int j = 0; j < C::N; ++j)
          if (col + j < a.cols) out[k * a.cols + col + j] = f[j];
      }
    }
}

// dw and db: 32 columns a workgroup, 32 threads a column.
template <typename T>
__global__ __launch_bounds__(1024) void norm_columns_kernel(NormArgs a) {
  __shared__ float red[32][33];
  const int c = threadIdx.x % 32, y = threadIdx.x / 32;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < 2 * a.cols)
#pragma unroll 8
    for (int p = y; p < a.n_parts; p += 32) s += a.part[(int64_t)p * 2 * a.cols + col];
  red[y][c] = s;
  __syncthreads();
  if (y != 0 || col >= 2 * a.cols) return;
  s = 0.f;
#pragma unroll
  for (int p = 0; p < 32; ++p) s += red[p][c];
  void* out = col < a.cols ? a.dw : a.db;
  if (out == nullptr) return;
  const int64_t at = col < a.cols ? col : col - a.cols;
  if (a.w_is_f32) reinterpret_cast<float*>(out)[at] = s;
  else reinterpret_cast<T*>(out)[at] = (T)s;
}

constexpr int64_t kNormCols = 16384;  // what 1024 threads' registers hold

// f.operator()<T, LPR, NV>() for rows of `cols` elements.
template <typename F>
int norm_dispatch(int dtype, int64_t cols, F&& f) {
  auto by_width = [&](auto t) {
    using T = decltype(t);
    const int64_t chunks = (cols + Chunk<T>::N - 1) / Chunk<T>::N;
    auto go = [&](auto lpr, auto nv) { return f(t, lpr, nv); };
#define TJ_NORM(L, N) return go(std::integral_constant<int, L>{}, std::integral_constant<int, N>{})
    if (chunks <= 8) TJ_NORM(8, 1);
    if (chunks <= 16) TJ_NORM(16, 1);
    if (chunks <= 32) TJ_NORM(32, 1);
    if (chunks <= 64) TJ_NORM(64, 1);
    if (chunks <= 128) TJ_NORM(64, 2);
    if (chunks <= 256) TJ_NORM(64, 4);
    if (chunks <= 512) TJ_NORM(256, 2);
    if (chunks <= 1024) TJ_NORM(256, 4);
    if constexpr (sizeof(T) == 4)
      if (chunks > 2048) TJ_NORM(1024, 4);
    TJ_NORM(1024, 2);
#undef TJ_NORM
  };
  if (dtype == TJ_F32) return by_width(float{});
  if (dtype == TJ_F16) return by_width(half_t{});
  return by_width(bf16_t{});
}

int norm_elem_bytes(int dtype) { return dtype == TJ_F32 ? 4 : (dtype == TJ_F16 || dtype == TJ_BF16 ? 2 : 0); }

// Workgroups: enough to fill the chip, no more rows' columns to add up than that.
int64_t norm_grid(int64_t rows, int rows_per_block, int64_t most) {
  const int64_t n = (rows + rows_per_block - 1) / rows_per_block;
  return n < most ? n : most;
}
constexpr int64_t kFwdGroups = 4096, kBwdGroups = 512;

int norm_checks(int dtype, int w_dtype, int64_t rows, int64_t cols, const void* w, const void* b) {
  if (norm_elem_bytes(dtype) == 0) return TJ_ERR_DTYPE;
  if ((w != nullptr || b != nullptr) && w_dtype != TJ_F32 && w_dtype != dtype) return TJ_ERR_DTYPE;
  if (rows < 0 || cols <= 0 || rows >= (int64_t(1) << 40)) return TJ_ERR_SHAPE;
  if (cols > kNormCols) return TJ_ERR_UNSUPPORTED;
  return TJ_OK;
}

bool element_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(norm_elem_bytes(dtype) - 1)) == 0;
}

}  // namespace
}  // namespace tj

using namespace tj;

extern "C" int tj_layer_norm_fwd(const void* x, const void* weight, const void* bias, void* y, int dtype, int w_dtype,
                                 int64_t rows, int64_t cols, int64_t x_stride, int64_t y_stride, float eps, float* mean,
                                 float* rstd, hipStream_t stream) {
  if (const int rc = norm_checks(dtype, w_dtype, rows, cols, weight, bias)) return rc;
  if ((mean == nullptr) != (rstd == nullptr) || !(eps >= 0.f)) return TJ_ERR_SHAPE;
  if (rows == 0) return TJ_OK;
  if (x == nullptr || y == nullptr) return TJ_ERR_SHAPE;
  if (!element_aligned(x, dtype) || !element_aligned(y, dtype) || !element_aligned(weight, w_dtype == TJ_F32 ? TJ_F32 : dtype) ||
      !element_aligned(bias, w_dtype == TJ_F32 ? TJ_F32 : dtype) || !element_aligned(mean, TJ_F32) || !element_aligned(rstd, TJ_F32))
    return TJ_ERR_ALIGN;
  NormArgs a{};
  a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd;
  a.rows = rows; a.cols = cols; a.x_stride = x_stride; a.y_stride = y_stride; a.eps = eps;
  a.w_is_f32 = w_dtype == TJ_F32;
  return norm_dispatch(dtype, cols, [&](auto t, auto lpr, auto nv) {
    constexpr int LPR = decltype(lpr)::value, THREADS = norm_threads<LPR>();
    const int64_t grid = norm_grid(rows, THREADS / LPR, kFwdGroups);
    hipLaunchKernelGGL((norm_fwd_kernel<decltype(t), LPR, decltype(nv)::value>), dim3(uint32_t(grid)), dim3(THREADS), 0,
                       stream, a);
    return tjh::launch_status();
  });
}

extern "C" size_t tj_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > kNormCols) return 0;
  return size_t(norm_grid(rows, 1, kBwdGroups)) * 2 * size_t(cols) * sizeof(float);
}

extern "C" int tj_layer_norm_bwd(const void* dy, const void* x, const void* weight, const float* mean, const float* rstd,
                                 void* dx, void* dweight, void* dbias, int dtype, int w_dtype, int64_t rows, int64_t cols,
                                 int64_t dy_stride, int64_t x_stride, int64_t dx_stride, void* workspace,
                                 size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = norm_checks(dtype, w_dtype, rows, cols, weight, dweight != nullptr ? dweight : dbias)) return rc;
  if (rows == 0) return TJ_OK;
  if (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr) return TJ_ERR_SHAPE;
  const int wd = w_dtype == TJ_F32 ? TJ_F32 : dtype;
  if (!element_aligned(dy, dtype) || !element_aligned(x, dtype) || !element_aligned(dx, dtype) ||
      !element_aligned(weight, wd) || !element_aligned(dweight, wd) || !element_aligned(dbias, wd) ||
      !element_aligned(mean, TJ_F32) || !element_aligned(rstd, TJ_F32) || !element_aligned(workspace, TJ_F32))
    return TJ_ERR_ALIGN;
  const bool columns = dweight != nullptr || dbias != nullptr;
  if (columns && (workspace == nullptr || workspace_bytes < tj_layer_norm_bwd_workspace_bytes(rows, cols)))
    return TJ_ERR_WORKSPACE;
  NormArgs a{};
  a.dy = dy; a.x = x; a.w = weight; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dx = dx; a.dw = dweight; a.db = dbias; a.part = columns ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows; a.cols = cols; a.dy_stride = dy_stride; a.x_stride = x_stride; a.dx_stride = dx_stride;
  a.w_is_f32 = w_dtype == TJ_F32;
  return norm_dispatch(dtype, cols, [&](auto t, auto lpr, auto nv) {
    using T = decltype(t);
    constexpr int LPR = decltype(lpr)::value, THREADS = norm_threads<LPR>();
    a.n_parts = (int)norm_grid(rows, THREADS / LPR, kBwdGroups);
    hipLaunchKernelGGL((norm_bwd_kernel<T, LPR, decltype(nv)::value>), dim3(uint32_t(a.n_parts)), dim3(THREADS), 0, stream, a);
    const int rc = tjh::launch_status();
    if (rc != TJ_OK || !columns) return rc;
    hipLaunchKernelGGL((norm_columns_kernel<T>), dim3(uint32_t((2 * cols + 31) / 32)), dim3(1024), 0, stream, a);
    return tjh::launch_status();
  });
}
