// Row operators of token blocks (include/sga_hip.h): layer norm forward and backward, counter-based dropout.
#include "token_common.h"

using namespace token;

namespace {

// the sum of v over the workgroup, for every lane (n = 256 threads); sh: 4 floats, free again on return
__device__ __forceinline__ float block_sum(float v, float* sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (sh[0] + sh[1]) + (sh[2] + sh[3]);
  __syncthreads();
  return v;
}

template <typename T, typename P>
__global__ __launch_bounds__(256) void layer_norm_fwd_kernel(const T* __restrict__ x, int64_t ld_x, const P* __restrict__ w, const P* __restrict__ b,
                                                             T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, int cols,
                                                             float eps) {
  __shared__ float sh[4];
  const int64_t m = blockIdx.x;
  const T* row = x + m * ld_x;
  float s = 0.f;
  for (int c = threadIdx.x; c < cols; c += 256) s += to_f32(row[c]);
  const float mu = block_sum(s, sh) / (float)cols;
  float q = 0.f;
  for (int c = threadIdx.x; c < cols; c += 256) { const float d = to_f32(row[c]) - mu; q = fmaf(d, d, q); }
  const float r = 1.f / sqrtf(block_sum(q, sh) / (float)cols + eps);
  for (int c = threadIdx.x; c < cols; c += 256) {
    const float h = (to_f32(row[c]) - mu) * r;
    y[m * cols + c] = from_f32<T>(fmaf(h, w ? to_f32(w[c]) : 1.f, b ? to_f32(b[c]) : 0.f));
  }
  if (threadIdx.x == 0) {
    if (mean) mean[m] = mu;
    if (rstd) rstd[m] = r;
  }
}

template <typename T, typename P>
__global__ __launch_bounds__(256) void layer_norm_gx_kernel(const T* __restrict__ x, int64_t ld_x, const P* __restrict__ w, const T* __restrict__ gy,
                                                            int64_t ld_gy, const T* __restrict__ add, int64_t ld_add, const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, T* __restrict__ gx, int cols) {
  __shared__ float sh[4];
  const int64_t m = blockIdx.x;
  const float mu = mean[m], r = rstd[m];
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < cols; c += 256) {
    const float g = to_f32(gy[m * ld_gy + c]) * (w ? to_f32(w[c]) : 1.f), h = (to_f32(x[m * ld_x + c]) - mu) * r;
    s1 += g;
    s2 = fmaf(g, h, s2);
  }
  const float c1 = block_sum(s1, sh) / (float)cols, c2 = block_sum(s2, sh) / (float)cols;
  for (int c = threadIdx.x; c < cols; c += 256) {
    const float g = to_f32(gy[m * ld_gy + c]) * (w ? to_f32(w[c]) : 1.f), h = (to_f32(x[m * ld_x + c]) - mu) * r;
    float v = r * (g - c1 - h * c2);
    if (add) v += to_f32(add[m * ld_add + c]);
    gx[m * cols + c] = from_f32<T>(v);
  }
}

// part[chunk][0][c] = sum of g_y h, part[chunk][1][c] = sum of g_y over the chunk's rows
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_parts_kernel(const T* __restrict__ x, int64_t ld_x, const T* __restrict__ gy, int64_t ld_gy,
                                                               const float* __restrict__ mean, const float* __restrict__ rstd,
                                                               float* __restrict__ part, int64_t rows, int cols, int64_t per) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  const int64_t m0 = (int64_t)blockIdx.y * per, m1 = m0 + per < rows ? m0 + per : rows;
  float sw = 0.f, sb = 0.f;
  for (int64_t m = m0; m < m1; ++m) {
    const float g = to_f32(gy[m * ld_gy + c]);
    sw = fmaf(g, (to_f32(x[m * ld_x + c]) - mean[m]) * rstd[m], sw);
    sb += g;
  }
  part[((int64_t)blockIdx.y * 2) * cols + c] = sw;
  part[((int64_t)blockIdx.y * 2 + 1) * cols + c] = sb;
}

template <typename P>
__global__ __launch_bounds__(256) void layer_norm_join_kernel(const float* __restrict__ part, int64_t nparts, P* __restrict__ gw, P* __restrict__ gb,
                                                              int cols) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float sw = 0.f, sb = 0.f;
  for (int64_t p = 0; p < nparts; ++p) { sw += part[2 * p * cols + c]; sb += part[(2 * p + 1) * cols + c]; }
  if (gw) gw[c] = from_f32<P>(sw);
  if (gb) gb[c] = from_f32<P>(sb);
}

template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, int64_t ld_x, const T* res, int64_t ld_res, T* y, int64_t rows, int64_t cols,
                                                      const Drop d) {
  uint64_t seed = 0, offset = 0;
  if (d.on) drop_key(d, seed, offset);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / cols, c = i - m * cols;
    float v = to_f32(x[m * ld_x + c]);
    if (d.on) v = drop_one(d, seed, offset, (uint64_t)i, v);
    if (res) v += to_f32(res[m * ld_res + c]);
    y[i] = from_f32<T>(v);
  }
}

constexpr int64_t kMaxRows = 0x7fffffff;
constexpr int kMaxCols = 1 << 20;

#define LAUNCHED() do { if (hipGetLastError() != hipSuccess) return SGA_ERR_HIP; } while (0)

bool ld_ok(const void* p, int64_t ld, int64_t cols) { return !p || ld == 0 || ld >= cols; }

int norm_check(const sga_layer_norm* a) {
  if (!a || a->rows < 0 || a->cols < 1 || !dtype_ok(a->dtype)) return SGA_ERR_BAD_ARG;
  if (a->param_dtype != a->dtype && a->param_dtype != SGA_DTYPE_F32) return SGA_ERR_BAD_ARG;
  if (a->rows > kMaxRows || a->cols > kMaxCols) return SGA_ERR_UNSUPPORTED;
  if (!at_ok(a->x, a->dtype) || !at_ok(a->w, a->param_dtype) || !at_ok(a->b, a->param_dtype) || !at_ok(a->mean, SGA_DTYPE_F32) ||
      !at_ok(a->rstd, SGA_DTYPE_F32) || !ld_ok(a->x, a->ld_x, a->cols))
    return SGA_ERR_BAD_ARG;
  return SGA_OK;
}
int norm_fwd_check(const sga_layer_norm* a) {
  const int st = norm_check(a);
  if (st != SGA_OK) return st;
  if (!(a->eps >= 0.f) || (a->rows > 0 && (!a->x || !a->y)) || !at_ok(a->y, a->dtype)) return SGA_ERR_BAD_ARG;
  return SGA_OK;
}
int norm_bwd_check(const sga_layer_norm* a) {
  const int st = norm_check(a);
  if (st != SGA_OK) return st;
  if (a->rows > 0 && (!a->x || !a->g_y || !a->mean || !a->rstd)) return SGA_ERR_BAD_ARG;
  if (!at_ok(a->g_y, a->dtype) || !at_ok(a->g_add, a->dtype) || !at_ok(a->g_x, a->dtype) || !at_ok(a->g_w, a->param_dtype) ||
      !at_ok(a->g_b, a->param_dtype) || !ld_ok(a->g_y, a->ld_g_y, a->cols) || !ld_ok(a->g_add, a->ld_g_add, a->cols))
    return SGA_ERR_BAD_ARG;
  return SGA_OK;
}
int64_t norm_per(const sga_layer_norm& a) { return ceil_div(a.rows, 1024) > 64 ? ceil_div(a.rows, 1024) : 64; }   // at most 1024 partial sums
int64_t norm_parts(const sga_layer_norm& a) { return ceil_div(a.rows, norm_per(a)); }
int64_t norm_bwd_bytes(const sga_layer_norm& a) {
  return (a.g_w || a.g_b) ? round_up(norm_parts(a) * 2 * a.cols * 4, 256) : 0;
}

template <typename T, typename P>
int norm_fwd(const sga_layer_norm& a, hipStream_t st) {
  hipLaunchKernelGGL((layer_norm_fwd_kernel<T, P>), dim3((unsigned)a.rows), dim3(256), 0, st, (const T*)a.x, a.ld_x, (const P*)a.w, (const P*)a.b,
                     (T*)a.y, a.mean, a.rstd, a.cols, a.eps);
  LAUNCHED();
  return SGA_OK;
}

template <typename T, typename P>
int norm_bwd(const sga_layer_norm& a, float* part, hipStream_t st) {
  if (a.g_x && a.rows > 0) {
    hipLaunchKernelGGL((layer_norm_gx_kernel<T, P>), dim3((unsigned)a.rows), dim3(256), 0, st, (const T*)a.x, a.ld_x, (const P*)a.w,
                       (const T*)a.g_y, a.ld_g_y, (const T*)a.g_add, a.ld_g_add, a.mean, a.rstd, (T*)a.g_x, a.cols);
    LAUNCHED();
  }
  if (a.g_w || a.g_b) {
    const int64_t np = norm_parts(a);
    const unsigned gx = (unsigned)ceil_div(a.cols, 256);
    if (np > 0) {
      hipLaunchKernelGGL((layer_norm_parts_kernel<T>), dim3(gx, (unsigned)np), dim3(256), 0, st, (const T*)a.x, a.ld_x, (const T*)a.g_y, a.ld_g_y,
                         a.mean, a.rstd, part, a.rows, a.cols, norm_per(a));
      LAUNCHED();
    }
    hipLaunchKernelGGL((layer_norm_join_kernel<P>), dim3(gx), dim3(256), 0, st, part, np, (P*)a.g_w, (P*)a.g_b, a.cols);
    LAUNCHED();
  }
  return SGA_OK;
}

template <typename T>
int dropout_run(const void* x, int64_t ld_x, const void* res, int64_t ld_res, void* y, int64_t rows, int64_t cols, const Drop& d, hipStream_t st) {
  const int64_t blocks = ceil_div(rows * cols, 256);
  hipLaunchKernelGGL((dropout_kernel<T>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st, (const T*)x, ld_x, (const T*)res, ld_res,
                     (T*)y, rows, cols, d);
  LAUNCHED();
  return SGA_OK;
}

}  // namespace

extern "C" {

int sga_op_layer_norm_workspace(const sga_layer_norm* a, int backward, int64_t* bytes) {
  if (!bytes) return SGA_ERR_BAD_ARG;
  const int st = backward ? norm_bwd_check(a) : norm_fwd_check(a);
  if (st != SGA_OK) return st;
  *bytes = backward ? norm_bwd_bytes(*a) : 0;
  return SGA_OK;
}

int sga_op_layer_norm_fwd(const sga_layer_norm* a, void* stream) {
  const int st = norm_fwd_check(a);
  if (st != SGA_OK || a->rows == 0) return st;
  hipStream_t s = (hipStream_t)stream;
  if (a->dtype == SGA_DTYPE_F32) return norm_fwd<float, float>(*a, s);
  if (a->dtype == SGA_DTYPE_BF16) return a->param_dtype == SGA_DTYPE_F32 ? norm_fwd<bf16, float>(*a, s) : norm_fwd<bf16, bf16>(*a, s);
  return a->param_dtype == SGA_DTYPE_F32 ? norm_fwd<f16, float>(*a, s) : norm_fwd<f16, f16>(*a, s);
}

int sga_op_layer_norm_bwd(const sga_layer_norm* a, void* workspace, int64_t workspace_bytes, void* stream) {
  const int st = norm_bwd_check(a);
  if (st != SGA_OK) return st;
  const int64_t need = norm_bwd_bytes(*a);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))) return SGA_ERR_BAD_ARG;
  hipStream_t s = (hipStream_t)stream;
  float* p = (float*)workspace;
  if (a->dtype == SGA_DTYPE_F32) return norm_bwd<float, float>(*a, p, s);
  if (a->dtype == SGA_DTYPE_BF16) return a->param_dtype == SGA_DTYPE_F32 ? norm_bwd<bf16, float>(*a, p, s) : norm_bwd<bf16, bf16>(*a, p, s);
  return a->param_dtype == SGA_DTYPE_F32 ? norm_bwd<f16, float>(*a, p, s) : norm_bwd<f16, f16>(*a, p, s);
}

int sga_op_dropout(const void* x, int64_t ld_x, const void* residual, int64_t ld_residual, void* y, int64_t rows, int64_t cols,
                   int dtype, const sga_dropout* dropout, void* stream) {
  if (rows < 0 || cols < 1 || !dtype_ok(dtype) || !dropout || !drop_ok(*dropout)) return SGA_ERR_BAD_ARG;
  if (rows > kMaxRows || cols > 0x7fffffff) return SGA_ERR_UNSUPPORTED;
  if ((rows > 0 && (!x || !y)) || !at_ok(x, dtype) || !at_ok(y, dtype) || !at_ok(residual, dtype)) return SGA_ERR_BAD_ARG;
  if (!ld_ok(x, ld_x, cols) || !ld_ok(residual, ld_residual, cols)) return SGA_ERR_BAD_ARG;
  if (rows == 0) return SGA_OK;
  const Drop d = make_drop(*dropout);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SGA_DTYPE_F32) return dropout_run<float>(x, ld_x, residual, ld_residual, y, rows, cols, d, s);
  if (dtype == SGA_DTYPE_BF16) return dropout_run<bf16>(x, ld_x, residual, ld_residual, y, rows, cols, d, s);
  return dropout_run<f16>(x, ld_x, residual, ld_residual, y, rows, cols, d, s);
}

}  // extern "C"
