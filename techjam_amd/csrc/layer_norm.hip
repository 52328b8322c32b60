// Layer norm of rows, forward and backward, fp32 / fp16 / bf16:
//
//   xh = (x - mean) rstd,  y = xh w + b
//   g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Bound by memory: each pass reads its rows once. A row's values stay in the
// registers of `LPR` lanes (a part of a wave, a wave, or a whole workgroup), NV
// chunks of N elements each, through the sums and the output; mean and variance
// are two sums over those registers (no difference of squares). A workgroup
// walks over rows with the weights, and in the backward pass the columns' sums,
// in registers; the workgroups' column sums are added up by a second kernel in
// a fixed order. All sums are fp32. A chunk is 16 bytes where width, strides and
// bases are multiples of that, one element otherwise. Loads and stores go through
// bounds-checked buffers with an offset outside for what is not there, so that a
// row's accesses are all in flight at once (with a branch around each, 65536 rows
// of 2048 bf16 took 204 us forward and 226 us backward). Now 88 us forward, 6.1 TB/s,
// and 155 us backward, 5.2 TB/s (a copy of 1
// GiB: 5.1); 131072 rows of 128 fp16: 13 and 22 us.
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

constexpr uint32_t kOutside = 0x80000000u;

// The workgroup's rows r0 .. of a tensor: a buffer from row r0 on.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(p)) + bytes, (short)0, 0x7fffffff,
                                           0x00020000);
}

// N elements of T at byte offset `at`, as fp32; zeros outside.
template <typename T, int N>
__device__ __forceinline__ void load_n(float (&f)[N], __amdgpu_buffer_rsrc_t r, uint32_t at) {
  if constexpr (N * sizeof(T) >= 16) {
    constexpr int M = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(M)));
#pragma unroll
    for (int i = 0; i < N; i += M) {
      const vec v = __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b128(r, at + i * (uint32_t)sizeof(T), 0, 0));
#pragma unroll
      for (int j = 0; j < M; ++j) f[i + j] = (float)v[j];
    }
  } else if constexpr (sizeof(T) == 4) {
    f[0] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0));
  } else {
    f[0] = (float)__builtin_bit_cast(T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0));
  }
}
// The same stored, rounded to T; nothing outside.
template <typename T, int N>
__device__ __forceinline__ void store_n(const float (&f)[N], __amdgpu_buffer_rsrc_t r, uint32_t at) {
  if constexpr (N * sizeof(T) >= 16) {
    constexpr int M = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(M)));
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < N; i += M) {
      vec v;
#pragma unroll
      for (int j = 0; j < M; ++j) v[j] = (T)f[i + j];
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, at + i * (uint32_t)sizeof(T), 0, 0);
    }
  } else if constexpr (sizeof(T) == 4) {
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, f[0]), r, at, 0, 0);
  } else {
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (T)f[0]), r, at, 0, 0);
  }
}

// A chunk of the weight or bias (fp32 or T), `none` where there is none.
template <typename T, int N>
__device__ __forceinline__ void load_param(float (&f)[N], const void* p, int is_f32, int64_t col, int64_t cols, float none) {
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = none;
  if (p == nullptr) return;
  const auto r = rows_at(p, 0);
  if (is_f32) load_n<float, N>(f, r, col < cols ? (uint32_t)col * 4u : kOutside);
  else load_n<T, N>(f, r, col < cols ? (uint32_t)col * (uint32_t)sizeof(T) : kOutside);
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

// Y: the output's type, T or fp32.
template <typename T, typename Y, int N, int LPR, int NV>
__global__ __launch_bounds__(norm_threads<LPR>()) void norm_fwd_kernel(NormArgs a) {
  constexpr int THREADS = norm_threads<LPR>(), RPB = THREADS / LPR;
  __shared__ float red[4 * (LPR > kWave ? LPR / kWave : 1)];
  const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  int parity = 0;
  float w[NV][N], b[NV][N];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t col = (int64_t)(lane + v * LPR) * N;
    load_param<T, N>(w[v], a.w, a.w_is_f32, col, a.cols, 1.f);
    load_param<T, N>(b[v], a.b, a.w_is_f32, col, a.cols, 0.f);
  }
  const float inv_n = 1.f / (float)a.cols;
  const uint32_t x_row = sub * (uint32_t)(a.x_stride * (int64_t)sizeof(T)), y_row = sub * (uint32_t)(a.y_stride * (int64_t)sizeof(Y));
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
    const bool on = sub < a.rows - r0;
    const auto xr = rows_at(a.x, r0 * a.x_stride * (int64_t)sizeof(T));
    const auto yr = rows_at(a.y, r0 * a.y_stride * (int64_t)sizeof(Y));
    float x[NV][N], s[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (lane + v * LPR) * N;
      load_n<T, N>(x[v], xr, on && col < a.cols ? x_row + col * (int)sizeof(T) : kOutside);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < N; ++j) s[0] += x[v][j];
    row_sums<LPR, 1>(s, red, parity);
    const float mean = s[0] * inv_n;
    s[0] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const bool in = (lane + v * LPR) * N < a.cols;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x[v][j] -= mean;
        s[0] = fmaf(x[v][j], in ? x[v][j] : 0.f, s[0]);
      }
    }
    row_sums<LPR, 1>(s, red, parity);
    const float rstd = 1.f / sqrtf(s[0] * inv_n + a.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (lane + v * LPR) * N;
#pragma unroll
      for (int j = 0; j < N; ++j) x[v][j] = fmaf(x[v][j] * rstd, w[v][j], b[v][j]);
      store_n<Y, N>(x[v], yr, on && col < a.cols ? y_row + col * (int)sizeof(Y) : kOutside);
    }
    if (a.mean != nullptr && on && lane == 0) {
      a.mean[r0 + sub] = mean;
      a.rstd[r0 + sub] = rstd;
    }
  }
}

// Y: the type of the output and so of its gradient.
template <typename T, typename Y, int N, int LPR, int NV>
__global__ __launch_bounds__(norm_threads<LPR>()) void norm_bwd_kernel(NormArgs a) {
  constexpr int THREADS = norm_threads<LPR>(), RPB = THREADS / LPR;
  __shared__ float red[4 * (LPR > kWave ? LPR / kWave : 1)];
  __shared__ float cols[LPR < THREADS ? THREADS * N : 1];
  const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  int parity = 0;
  float w[NV][N], dw[NV][N], db[NV][N];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    load_param<T, N>(w[v], a.w, a.w_is_f32, (int64_t)(lane + v * LPR) * N, a.cols, 1.f);
#pragma unroll
    for (int j = 0; j < N; ++j) dw[v][j] = db[v][j] = 0.f;
  }
  const float inv_n = 1.f / (float)a.cols;
  const uint32_t x_row = sub * (uint32_t)(a.x_stride * (int64_t)sizeof(T)), g_row = sub * (uint32_t)(a.dy_stride * (int64_t)sizeof(Y)),
                 d_row = sub * (uint32_t)(a.dx_stride * (int64_t)sizeof(T));
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
    const bool on = sub < a.rows - r0;
    const auto xr = rows_at(a.x, r0 * a.x_stride * (int64_t)sizeof(T));
    const auto gr = rows_at(a.dy, r0 * a.dy_stride * (int64_t)sizeof(Y));
    float x[NV][N], g[NV][N], s[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (lane + v * LPR) * N;
      const bool in = on && col < a.cols;
      load_n<T, N>(x[v], xr, in ? x_row + col * (int)sizeof(T) : kOutside);
      load_n<Y, N>(g[v], gr, in ? g_row + col * (int)sizeof(Y) : kOutside);
    }
    const float mean = on ? a.mean[r0 + sub] : 0.f, rstd = on ? a.rstd[r0 + sub] : 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      // Past the row's end dy and x read as zero, and with no mean there xh is too:
      // -mean rstd may be an infinity, which times zero would spoil the row's sums.
      const float centre = (lane + v * LPR) * N < a.cols ? mean : 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x[v][j] = (x[v][j] - centre) * rstd;
        dw[v][j] = fmaf(g[v][j], x[v][j], dw[v][j]);
        db[v][j] += g[v][j];
        g[v][j] *= w[v][j];
        s[0] += g[v][j];
        s[1] = fmaf(g[v][j], x[v][j], s[1]);
      }
    }
    if (a.dx != nullptr) {
      row_sums<LPR, 2>(s, red, parity);
      const float c0 = s[0] * inv_n, c1 = s[1] * inv_n;
      const auto dr = rows_at(a.dx, r0 * a.dx_stride * (int64_t)sizeof(T));
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int col = (lane + v * LPR) * N;
#pragma unroll
        for (int j = 0; j < N; ++j) g[v][j] = rstd * (g[v][j] - fmaf(x[v][j], c1, c0));
        store_n<T, N>(g[v], dr, on && col < a.cols ? d_row + col * (int)sizeof(T) : kOutside);
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
      float(&f)[N] = k == 0 ? dw[v] : db[v];
      if constexpr (LPR < THREADS) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; ++j) cols[j * THREADS + threadIdx.x] = f[j];
        __syncthreads();
        if (threadIdx.x < LPR)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            f[j] = 0.f;
#pragma unroll 4
            for (int i = 0; i < RPB; ++i) f[j] += cols[j * THREADS + i * LPR + threadIdx.x];
          }
      }
      if (threadIdx.x < LPR) {
        const int64_t col = (int64_t)(lane + v * LPR) * N;
#pragma unroll
        for (int j = 0; j < N; ++j)
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

// f.operator()<T, Y, N, LPR, NV>() for rows of `cols` elements, whose chunks are
// 16 bytes (`whole`) or single elements; y_dtype is T's or fp32.
template <typename F>
int norm_dispatch(int dtype, int y_dtype, int64_t cols, bool whole, F&& f) {
  auto by_width = [&](auto t, auto y) {
    using T = decltype(t);
    constexpr int VEC = 16 / (int)sizeof(T);
#define TJ_NORM(N, L, V) \
  return f(t, y, std::integral_constant<int, N>{}, std::integral_constant<int, L>{}, std::integral_constant<int, V>{})
    if (!whole) {
      if (cols <= 256) TJ_NORM(1, 64, 4);
      if (cols <= 1024) TJ_NORM(1, 64, 16);
      if (cols <= 4096) TJ_NORM(1, 256, 16);
      TJ_NORM(1, 1024, 16);
    }
    const int64_t chunks = cols / VEC;
    if (chunks <= 8) TJ_NORM(VEC, 8, 1);
    if (chunks <= 16) TJ_NORM(VEC, 16, 1);
    if (chunks <= 32) TJ_NORM(VEC, 32, 1);
    if (chunks <= 64) TJ_NORM(VEC, 64, 1);
    if (chunks <= 128) TJ_NORM(VEC, 64, 2);
    if (chunks <= 256) TJ_NORM(VEC, 64, 4);
    if (chunks <= 512) TJ_NORM(VEC, 256, 2);
    if (chunks <= 1024) TJ_NORM(VEC, 256, 4);
    if constexpr (sizeof(T) == 4)
      if (chunks > 2048) TJ_NORM(VEC, 1024, 4);
    TJ_NORM(VEC, 1024, 2);
#undef TJ_NORM
  };
  if (dtype == TJ_F32) return by_width(float{}, float{});
  if (dtype == TJ_F16) return y_dtype == TJ_F32 ? by_width(half_t{}, float{}) : by_width(half_t{}, half_t{});
  return y_dtype == TJ_F32 ? by_width(bf16_t{}, float{}) : by_width(bf16_t{}, bf16_t{});
}

int norm_elem_bytes(int dtype) { return dtype == TJ_F32 ? 4 : (dtype == TJ_F16 || dtype == TJ_BF16 ? 2 : 0); }

// Workgroups: enough to fill the chip, but each has the weights to load first,
// and in the backward pass its column sums are to be added up. Forward 512 /
// 1024 / 2048 groups: 18 / 15 / 14 us on 131072 rows of 128 fp16, 87 / 92 / 89 on
// 65536 of 2048 bf16 (4096: 39 and 158 with the weights loaded one by one).
// Backward 512 / 1024 with the column kernel: 27.5 / 26 and 163 / 166 us.
int64_t norm_grid(int64_t rows, int rows_per_block, int64_t most) {
  const int64_t n = (rows + rows_per_block - 1) / rows_per_block;
  return n < most ? n : most;
}
constexpr int64_t kFwdGroups = 1024, kBwdGroupsNarrow = 1024, kBwdGroups = 512;  // narrow: rows of less than a wave

int norm_checks(int dtype, int y_dtype, int w_dtype, int64_t rows, int64_t cols, const void* w, const void* b) {
  if (norm_elem_bytes(dtype) == 0 || (y_dtype != TJ_F32 && y_dtype != dtype)) return TJ_ERR_DTYPE;
  if ((w != nullptr || b != nullptr) && w_dtype != TJ_F32 && w_dtype != dtype) return TJ_ERR_DTYPE;
  if (rows < 0 || cols <= 0 || rows >= (int64_t(1) << 40)) return TJ_ERR_SHAPE;
  if (cols > kNormCols) return TJ_ERR_UNSUPPORTED;
  return TJ_OK;
}

// Rows that a workgroup reaches by 31-bit byte offsets, 32 at a time.
bool row_stride_ok(int64_t stride, int dtype) {
  return stride >= 0 && stride < (int64_t(1) << 31) / (32 * norm_elem_bytes(dtype)) - kNormCols;
}

// 16-byte chunks: the tensor's base, rows and width (elements) are multiples of that.
bool whole_chunks(int dtype, int64_t cols, std::initializer_list<const void*> bases, std::initializer_list<int64_t> strides) {
  const int64_t vec = 16 / norm_elem_bytes(dtype);
  bool ok = cols % vec == 0;
  for (const void* p : bases) ok = ok && tjh::aligned16(p);
  for (int64_t s : strides) ok = ok && s % vec == 0;
  return ok;
}

bool element_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(norm_elem_bytes(dtype) - 1)) == 0;
}

}  // namespace
}  // namespace tj

using namespace tj;

extern "C" int tj_layer_norm_fwd(const void* x, const void* weight, const void* bias, void* y, int dtype, int y_dtype, int w_dtype,
                                 int64_t rows, int64_t cols, int64_t x_stride, int64_t y_stride, float eps, float* mean,
                                 float* rstd, hipStream_t stream) {
  if (const int rc = norm_checks(dtype, y_dtype, w_dtype, rows, cols, weight, bias)) return rc;
  if ((mean == nullptr) != (rstd == nullptr) || !(eps >= 0.f)) return TJ_ERR_SHAPE;
  if (rows == 0) return TJ_OK;
  if (x == nullptr || y == nullptr) return TJ_ERR_SHAPE;
  if (!element_aligned(x, dtype) || !element_aligned(y, y_dtype) || !element_aligned(weight, w_dtype == TJ_F32 ? TJ_F32 : dtype) ||
      !element_aligned(bias, w_dtype == TJ_F32 ? TJ_F32 : dtype) || !element_aligned(mean, TJ_F32) || !element_aligned(rstd, TJ_F32))
    return TJ_ERR_ALIGN;
  if (!row_stride_ok(x_stride, dtype) || !row_stride_ok(y_stride, y_dtype)) return TJ_ERR_UNSUPPORTED;
  NormArgs a{};
  a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd;
  a.rows = rows; a.cols = cols; a.x_stride = x_stride; a.y_stride = y_stride; a.eps = eps;
  a.w_is_f32 = w_dtype == TJ_F32;
  const bool whole = whole_chunks(dtype, cols, {x, y, weight, bias}, {x_stride, y_stride});
  return norm_dispatch(dtype, y_dtype, cols, whole, [&](auto t, auto y, auto n, auto lpr, auto nv) {
    constexpr int LPR = decltype(lpr)::value, THREADS = norm_threads<LPR>();
    const int64_t grid = norm_grid(rows, THREADS / LPR, kFwdGroups);
    hipLaunchKernelGGL((norm_fwd_kernel<decltype(t), decltype(y), decltype(n)::value, LPR, decltype(nv)::value>),
                       dim3(uint32_t(grid)), dim3(THREADS), 0, stream, a);
    return tjh::launch_status();
  });
}

extern "C" size_t tj_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > kNormCols) return 0;
  return size_t(norm_grid(rows, 1, kBwdGroupsNarrow)) * 2 * size_t(cols) * sizeof(float);
}

extern "C" int tj_layer_norm_bwd(const void* dy, const void* x, const void* weight, const float* mean, const float* rstd,
                                 void* dx, void* dweight, void* dbias, int dtype, int y_dtype, int w_dtype, int64_t rows, int64_t cols,
                                 int64_t dy_stride, int64_t x_stride, int64_t dx_stride, void* workspace,
                                 size_t workspace_bytes, hipStream_t stream) {
  if (const int rc = norm_checks(dtype, y_dtype, w_dtype, rows, cols, weight, dweight != nullptr ? dweight : dbias)) return rc;
  if (rows == 0) return TJ_OK;
  if (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr) return TJ_ERR_SHAPE;
  const int wd = w_dtype == TJ_F32 ? TJ_F32 : dtype;
  if (!element_aligned(dy, y_dtype) || !element_aligned(x, dtype) || !element_aligned(dx, dtype) ||
      !element_aligned(weight, wd) || !element_aligned(dweight, wd) || !element_aligned(dbias, wd) ||
      !element_aligned(mean, TJ_F32) || !element_aligned(rstd, TJ_F32) || !element_aligned(workspace, TJ_F32))
    return TJ_ERR_ALIGN;
  if (!row_stride_ok(x_stride, dtype) || !row_stride_ok(dy_stride, y_dtype) || (dx != nullptr && !row_stride_ok(dx_stride, dtype)))
    return TJ_ERR_UNSUPPORTED;
  const bool columns = dweight != nullptr || dbias != nullptr;
  if (columns && (workspace == nullptr || workspace_bytes < tj_layer_norm_bwd_workspace_bytes(rows, cols)))
    return TJ_ERR_WORKSPACE;
  NormArgs a{};
  a.dy = dy; a.x = x; a.w = weight; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dx = dx; a.dw = dweight; a.db = dbias; a.part = columns ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows; a.cols = cols; a.dy_stride = dy_stride; a.x_stride = x_stride; a.dx_stride = dx_stride;
  a.w_is_f32 = w_dtype == TJ_F32;
  const bool whole = whole_chunks(dtype, cols, {x, dy, dx, weight}, {x_stride, dy_stride, dx == nullptr ? 0 : dx_stride});
  return norm_dispatch(dtype, y_dtype, cols, whole, [&](auto t, auto y, auto n, auto lpr, auto nv) {
    using T = decltype(t);
    constexpr int LPR = decltype(lpr)::value, THREADS = norm_threads<LPR>();
    a.n_parts = (int)norm_grid(rows, THREADS / LPR, LPR < kWave ? kBwdGroupsNarrow : kBwdGroups);
    hipLaunchKernelGGL((norm_bwd_kernel<T, decltype(y), decltype(n)::value, LPR, decltype(nv)::value>),
                       dim3(uint32_t(a.n_parts)), dim3(THREADS), 0, stream, a);
    const int rc = tjh::launch_status();
    if (rc != TJ_OK || !columns) return rc;
    hipLaunchKernelGGL((norm_columns_kernel<T>), dim3(uint32_t((2 * cols + 31) / 32)), dim3(1024), 0, stream, a);
    return tjh::launch_status();
  });
}
