// Matrix product with a fused epilogue, and its backward pass (include/sga_hip.h: sga_op_linear_*).
//   forward   C[m, n] = epi( sum_k x[m, k] w[n, k] ),  epi(v) = residual + D_p(act(v + bias)),  pre = v + bias
//   backward  dz = D_p(g_out) act'(pre);  g_x[m, k] = sum_n dz[m, n] w[n, k];  g_w[n, k] = sum_m dz[m, n] x[m, k];  g_bias = sum_m dz
#include "token_common.h"

using namespace token;

namespace {

struct Epilogue {
  const void* bias; const void* residual; int64_t ld_residual; void* out; int64_t ld_out; void* pre; int64_t cols; int act; Drop drop;
};

template <typename T>
__device__ __forceinline__ void epilogue_one(const Epilogue& e, uint64_t seed, uint64_t offset, int64_t m, int64_t n, float v) {
  if (e.bias) v += to_f32(((const T*)e.bias)[n]);
  if (e.pre) ((T*)e.pre)[m * e.cols + n] = from_f32<T>(v);
  v = act_value(v, e.act);
  if (e.drop.on) v = drop_one(e.drop, seed, offset, (uint64_t)(m * e.cols + n), v);
  if (e.residual) v += to_f32(((const T*)e.residual)[m * e.ld_residual + n]);
  ((T*)e.out)[m * e.ld_out + n] = from_f32<T>(v);
}

// C[m, n] = epi(sum_k A(m, k) B(n, k)), A(m, k) = A[m sam + k sak]: one 64 x 64 tile per workgroup, 4 x 4 results per lane
template <typename T>
__global__ __launch_bounds__(256) void token_product_kernel(const T* __restrict__ A, int64_t sam, int64_t sak, const T* __restrict__ B,
                                                            int64_t sbn, int64_t sbk, int64_t M, int64_t N, int64_t K, const Epilogue e) {
  __shared__ float As[16][65], Bs[16][65];
  const int64_t m0 = (int64_t)blockIdx.x * 64, n0 = (int64_t)blockIdx.y * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += 16) {
    for (int i = threadIdx.x; i < 1024; i += 256) {
      const int k = i & 15, r = i >> 4;
      const bool ink = k0 + k < K;
      As[k][r] = ink && m0 + r < M ? to_f32(A[(m0 + r) * sam + (k0 + k) * sak]) : 0.f;
      Bs[k][r] = ink && n0 + r < N ? to_f32(B[(n0 + r) * sbn + (k0 + k) * sbk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { a[i] = As[k][ty * 4 + i]; b[i] = Bs[k][tx * 4 + i]; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
  uint64_t seed = 0, offset = 0;
  if (e.drop.on) drop_key(e.drop, seed, offset);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m < M && n < N) epilogue_one<T>(e, seed, offset, m, n, acc[i][j]);
    }
}


// dz = D_p(g) act'(pre) (dz null: not wanted), part[chunk][n] = sum of the chunk's dz (part null: not wanted)
template <typename T>
__global__ __launch_bounds__(256) void token_dz_kernel(const T* __restrict__ g, int64_t ld_g, const T* __restrict__ pre, int act, const Drop d,
                                                       T* __restrict__ dz, float* __restrict__ part, int64_t rows, int64_t cols, int64_t per) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= cols) return;
  const int64_t m0 = (int64_t)blockIdx.y * per, m1 = m0 + per < rows ? m0 + per : rows;
  uint64_t seed = 0, offset = 0;
  if (d.on) drop_key(d, seed, offset);
  float sum = 0.f;
  for (int64_t m = m0; m < m1; ++m) {
    float v = to_f32(g[m * ld_g + n]);
    if (d.on) v = drop_one(d, seed, offset, (uint64_t)(m * cols + n), v);
    if (act != SGA_ACT_NONE) v *= act_slope(to_f32(pre[m * cols + n]), act);
    sum += v;
    if (dz) dz[m * cols + n] = from_f32<T>(v);
  }
  if (part) part[(int64_t)blockIdx.y * cols + n] = sum;
}

template <typename T>
__global__ __launch_bounds__(256) void token_sum_parts_kernel(const float* __restrict__ part, int64_t nparts, T* __restrict__ out, int64_t cols) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= cols) return;
  float s = 0.f;
  for (int64_t p = 0; p < nparts; ++p) s += part[p * cols + n];
  out[n] = from_f32<T>(s);
}

constexpr int kMaxFeatures = 1 << 20;
constexpr int64_t kMaxRows = 0x7fffffff;

// what the backward pass lays out in its workspace
struct BwdPlan {
  bool dz, part;             // dz differs from g_out; g_bias is wanted
  int64_t per, chunks, dz_off, part_off, bytes;
};
BwdPlan bwd_plan(const sga_linear& a) {
  BwdPlan p = {};
  p.dz = (a.act != SGA_ACT_NONE || a.dropout.p > 0.0) && (a.g_x || a.g_w);
  p.part = a.g_bias != nullptr;
  p.per = ceil_div(a.rows, 1024) > 64 ? ceil_div(a.rows, 1024) : 64;      // rows per partial sum of g_bias: at most 1024 of them
  p.chunks = ceil_div(a.rows, p.per);
  if (p.dz) { p.dz_off = p.bytes; p.bytes += round_up(a.rows * a.out_features * (int64_t)dtype_bytes(a.dtype), 256); }
  if (p.part) { p.part_off = p.bytes; p.bytes += round_up(p.chunks * a.out_features * 4, 256); }
  return p;
}

int common_check(const sga_linear* a) {
  if (!a || a->rows < 0 || a->in_features < 1 || a->out_features < 1) return SGA_ERR_BAD_ARG;
  if (!dtype_ok(a->dtype) || a->act < SGA_ACT_NONE || a->act > SGA_ACT_SILU || !drop_ok(a->dropout)) return SGA_ERR_BAD_ARG;
  if (a->in_features > kMaxFeatures || a->out_features > kMaxFeatures || a->rows > kMaxRows) return SGA_ERR_UNSUPPORTED;
  if (a->ld_w < a->in_features && !(a->ld_w == 0)) return SGA_ERR_BAD_ARG;
  if (a->ld_x < a->in_features && !(a->ld_x == 0)) return SGA_ERR_BAD_ARG;
  if (!at_ok(a->x, a->dtype) || !at_ok(a->w, a->dtype) || !at_ok(a->pre, a->dtype)) return SGA_ERR_BAD_ARG;
  return SGA_OK;
}
int fwd_check(const sga_linear* a) {
  const int st = common_check(a);
  if (st != SGA_OK) return st;
  if (a->rows > 0 && (!a->x || !a->w || !a->out)) return SGA_ERR_BAD_ARG;
  if (a->ld_out < a->out_features || (a->residual && a->ld_residual != 0 && a->ld_residual < a->out_features)) return SGA_ERR_BAD_ARG;
  if (!at_ok(a->bias, a->dtype) || !at_ok(a->residual, a->dtype) || !at_ok(a->out, a->dtype)) return SGA_ERR_BAD_ARG;
  return SGA_OK;
}
int bwd_check(const sga_linear* a) {
  const int st = common_check(a);
  if (st != SGA_OK) return st;
  if (a->rows > 0 && (!a->g_out || (a->act != SGA_ACT_NONE && !a->pre) || (a->g_x && !a->w) || (a->g_w && !a->x))) return SGA_ERR_BAD_ARG;
  if (a->ld_g_out != 0 && a->ld_g_out < a->out_features) return SGA_ERR_BAD_ARG;
  if (!at_ok(a->g_out, a->dtype) || !at_ok(a->g_x, a->dtype) || !at_ok(a->g_w, a->dtype) || !at_ok(a->g_bias, a->dtype)) return SGA_ERR_BAD_ARG;
  return SGA_OK;
}

#define LAUNCHED() do { if (hipGetLastError() != hipSuccess) return SGA_ERR_HIP; } while (0)

template <typename T>
int product(const void* A, int64_t sam, int64_t sak, const void* B, int64_t sbn, int64_t sbk, int64_t M, int64_t N, int64_t K, const Epilogue& e,
            hipStream_t st) {
  hipLaunchKernelGGL((token_product_kernel<T>), dim3((unsigned)ceil_div(M, 64), (unsigned)ceil_div(N, 64)), dim3(256), 0, st, (const T*)A, sam, sak,
                     (const T*)B, sbn, sbk, M, N, K, e);
  LAUNCHED();
  return SGA_OK;
}

template <typename T>
int linear_fwd(const sga_linear& a, hipStream_t st) {
  Epilogue e = {a.bias, a.residual, a.ld_residual, a.out, a.ld_out, a.pre, a.out_features, a.act, make_drop(a.dropout)};
  return product<T>(a.x, a.ld_x, 1, a.w, a.ld_w, 1, a.rows, a.out_features, a.in_features, e, st);
}

template <typename T>
int linear_bwd(const sga_linear& a, char* ws, hipStream_t st) {
  const BwdPlan p = bwd_plan(a);
  const T* dz = (const T*)a.g_out;
  int64_t ld_dz = a.ld_g_out;
  float* part = p.part ? (float*)(ws + p.part_off) : nullptr;
  if ((p.dz || p.part) && a.rows > 0) {
    T* to = p.dz ? (T*)(ws + p.dz_off) : nullptr;
    hipLaunchKernelGGL((token_dz_kernel<T>), dim3((unsigned)ceil_div(a.out_features, 256), (unsigned)p.chunks), dim3(256), 0, st, (const T*)a.g_out,
                       a.ld_g_out, (const T*)a.pre, a.act, make_drop(a.dropout), to, part, a.rows, (int64_t)a.out_features, p.per);
    LAUNCHED();
    if (p.dz) { dz = to; ld_dz = a.out_features; }
  }
  if (p.part) {
    hipLaunchKernelGGL((token_sum_parts_kernel<T>), dim3((unsigned)ceil_div(a.out_features, 256)), dim3(256), 0, st, part, p.chunks, (T*)a.g_bias,
                       (int64_t)a.out_features);
    LAUNCHED();
  }
  Epilogue e = {};
  if (a.g_x && a.rows > 0) {
    e.out = a.g_x; e.ld_out = e.cols = a.in_features;
    const int s = product<T>(dz, ld_dz, 1, a.w, 1, a.ld_w, a.rows, a.in_features, a.out_features, e, st);
    if (s != SGA_OK) return s;
  }
  if (a.g_w) {
    e.out = a.g_w; e.ld_out = e.cols = a.in_features;
    const int s = product<T>(dz, 1, ld_dz, a.x, 1, a.ld_x, a.out_features, a.in_features, a.rows, e, st);
    if (s != SGA_OK) return s;
  }
  return SGA_OK;
}

}  // namespace

extern "C" {

int sga_op_linear_workspace(const sga_linear* a, int backward, int64_t* bytes) {
  if (!bytes) return SGA_ERR_BAD_ARG;
  const int st = backward ? bwd_check(a) : fwd_check(a);
  if (st != SGA_OK) return st;
  *bytes = backward ? bwd_plan(*a).bytes : 0;
  return SGA_OK;
}

int sga_op_linear_fwd(const sga_linear* a, void* workspace, int64_t workspace_bytes, void* stream) {
  const int st = fwd_check(a);
  if (st != SGA_OK || a->rows == 0) return st;
  hipStream_t s = (hipStream_t)stream;
  (void)workspace; (void)workspace_bytes;
  return a->dtype == SGA_DTYPE_F32 ? linear_fwd<float>(*a, s) : a->dtype == SGA_DTYPE_BF16 ? linear_fwd<bf16>(*a, s) : linear_fwd<f16>(*a, s);
}

int sga_op_linear_bwd(const sga_linear* a, void* workspace, int64_t workspace_bytes, void* stream) {
  const int st = bwd_check(a);
  if (st != SGA_OK) return st;
  const int64_t need = bwd_plan(*a).bytes;
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))) return SGA_ERR_BAD_ARG;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  return a->dtype == SGA_DTYPE_F32 ? linear_bwd<float>(*a, ws, s) : a->dtype == SGA_DTYPE_BF16 ? linear_bwd<bf16>(*a, ws, s) : linear_bwd<f16>(*a, ws, s);
}

}  // extern "C"
