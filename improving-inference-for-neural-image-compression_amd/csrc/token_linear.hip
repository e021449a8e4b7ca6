// Matrix product with a fused epilogue, and its backward pass (include/sga_hip.h: sga_op_linear_*).
//   forward   C[m, n] = epi( sum_k x[m, k] w[n, k] ),  epi(v) = residual + D_p(act(v + bias)),  pre = v + bias
//   backward  dz = D_p(g_out) act'(pre);  g_x[m, k] = sum_n dz[m, n] w[n, k];  g_w[n, k] = sum_m dz[m, n] x[m, k];  g_bias = sum_m dz
#include "token_common.h"

using namespace token;

namespace {

// dz = D_p(g) act'(pre) (dz null: not wanted; its rows end in zeros up to ld_dz), part[chunk][n] = sum of the chunk's dz before the
// rounding (part null: not wanted).  32 pieces of 8 columns x 8 rows per workgroup; `vec`: all pieces whole and 16-byte aligned.
// dz is rounded to the type as the products' operand, for a product of 16-bit types takes no wider one: g_x and g_w of bf16 are then off by
// 0.0023 of their norm, where their own rounding alone makes 0.0017 (8192 x 2048 x 8192, gelu).  Two 16-bit terms would hold it, at twice
// the products' time, 454 of 523 us there.
// Bound by HBM: 8192 x 8192 bf16, gelu (403 MB) 81 us = 5.0 TB/s, a copy's rate.  Two passes (here and over dz in the products) instead
// of act' in the products' own fetches, which go past the registers.  The sums of a chunk stay in 32 bits, in a fixed order.
template <typename T>
__global__ __launch_bounds__(256) void token_dz_kernel(const T* __restrict__ g, int64_t ld_g, const T* __restrict__ pre, int act, const Drop d,
                                                       T* __restrict__ dz, int64_t ld_dz, float* __restrict__ part, int64_t rows, int64_t cols,
                                                       int64_t per, int vec) {
  __shared__ float sh[8][264];
  const int px = threadIdx.x & 31, py = threadIdx.x >> 5;
  const int64_t n = (int64_t)blockIdx.x * 256 + px * 8;
  const int64_t m0 = (int64_t)blockIdx.y * per, m1 = m0 + per < rows ? m0 + per : rows;
  const int live = cols - n >= 8 ? 8 : cols > n ? (int)(cols - n) : 0;
  uint64_t seed = 0, offset = 0;
  if (d.on) drop_key(d, seed, offset);
  float sum[8] = {};
  for (int64_t m = m0 + py; m < m1 && live > 0; m += 8) {
    float v[8], z[8] = {};
    if (vec) {
      load8(g + m * ld_g + n, v);
      if (act != SGA_ACT_NONE) load8(pre + m * cols + n, z);
      if (d.on) {
        uint32_t w[8];
        const uint64_t q = (uint64_t)(m * cols + n) >> 2;
        drop_words(seed, offset, q, w);
        drop_words(seed, offset, q + 1, w + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = drop_apply(d, w[j], v[j]);
      }
    } else {
      uint32_t w[12];
      const uint64_t i0 = (uint64_t)(m * cols + n);
      const int shift = (int)(i0 & 3);
      if (d.on) {
#pragma unroll
        for (int k = 0; k < 3; ++k) drop_words(seed, offset, (i0 >> 2) + k, w + 4 * k);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = j < live ? to_f32(g[m * ld_g + n + j]) : 0.f;
        z[j] = j < live && act != SGA_ACT_NONE ? to_f32(pre[m * cols + n + j]) : 0.f;
        if (d.on) v[j] = j < live ? drop_apply(d, shift == 0 ? w[j] : shift == 1 ? w[j + 1] : shift == 2 ? w[j + 2] : w[j + 3], v[j]) : 0.f;
      }
    }
    act_slopes<T, 8>(v, z, act);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] += v[j];
    if (dz) store8(dz + m * ld_dz + n, v);      // ld_dz is a multiple of 8: a ragged last piece ends in zeros
  }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) sh[py][px * 8 + j] = sum[j];
  __syncthreads();
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c < cols) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sh[k][threadIdx.x];
    part[(int64_t)blockIdx.y * cols + c] = s;
  }
}

// g_bias = the sum of the partial sums: 32 columns x 8 runs of them per workgroup.  Bound by latency, the
// parts lie in L2: 128 x 8192 in 5 us (a lane per column alone took 35)
template <typename T>
__global__ __launch_bounds__(256) void token_sum_parts_kernel(const float* __restrict__ part, int64_t nparts, T* __restrict__ out, int64_t cols) {
  __shared__ float sh[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t n = (int64_t)blockIdx.x * 32 + tx, per = (nparts + 7) / 8, p0 = ty * per, p1 = p0 + per < nparts ? p0 + per : nparts;
  float s = 0.f;
  if (n < cols) {
#pragma unroll 8
    for (int64_t p = p0; p < p1; ++p) s += part[p * cols + n];
  }
  sh[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && n < cols) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sh[k][tx];
    out[n] = from_f32<T>(s);
  }
}

// g_weight of no rows, the sum of no terms: a product has at least one k (its tiles read the last one again for their ends)
template <typename T>
__global__ __launch_bounds__(256) void token_zero_kernel(T* __restrict__ out, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = (T)0.f;
}

constexpr int kMaxFeatures = 1 << 20;
constexpr int64_t kMaxRows = 0x7fffff00;      // as many as 256-row tiles of 512 lanes fit into a launch of 2^32 lanes

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

Product forward_product(const sga_linear& a) {
  const int64_t E = (int64_t)dtype_bytes(a.dtype);
  Product p = {};
  p.x = {a.x, a.ld_x, 0};
  p.w = {a.w, a.ld_w, 0};
  p.M = a.rows; p.N = a.out_features; p.K = a.in_features;
  p.dtype = a.dtype;
  p.e = {a.bias, a.residual, a.ld_residual, a.out, a.ld_out, a.pre, a.out_features, a.act, 0, make_drop(a.dropout)};
  p.e.vec = a.out_features % 8 == 0 && aligned16(a.out) && a.ld_out * E % 16 == 0 && aligned16(a.bias) && aligned16(a.pre) &&
            (!a.residual || (aligned16(a.residual) && a.ld_residual * E % 16 == 0));
  return p;
}

// what the backward pass lays out in its workspace: [dz][parts of g_bias][the products' own], the two products one after the other
struct BwdPlan {
  bool dz, part;             // dz differs from g_out; g_bias is wanted
  int64_t ld_dz, per, chunks, dz_off, part_off, prod_off, bytes;
  Product gx, gw;
};
BwdPlan bwd_plan(const sga_linear& a, char* ws) {
  const int64_t E = (int64_t)dtype_bytes(a.dtype);
  BwdPlan p = {};
  p.dz = (a.act != SGA_ACT_NONE || a.dropout.p > 0.0) && (a.g_x || a.g_w);
  p.part = a.g_bias != nullptr;
  p.ld_dz = round_up(a.out_features, 8);
  // rows per workgroup of the dz pass, a partial sum of g_bias each: 64, or as few as 8 where that would leave CUs idle, and at
  // most 1024 partial sums
  const int64_t floor = ceil_div(a.rows, 1024), few = a.rows * ceil_div(a.out_features, 256) / 1024 / 8 * 8;
  p.per = few < 8 ? 8 : few > 64 ? 64 : few;
  p.per = p.per > floor ? p.per : floor;
  p.chunks = ceil_div(a.rows, p.per);
  if (p.dz) { p.dz_off = p.bytes; p.bytes += round_up(a.rows * p.ld_dz * E, 256); }
  if (p.part) { p.part_off = p.bytes; p.bytes += round_up(p.chunks * a.out_features * 4, 256); }
  p.prod_off = p.bytes;
  Operand dz = {a.g_out, a.ld_g_out, 0};
  if (p.dz) dz = {ws + p.dz_off, p.ld_dz, 0};
  Epilogue e = {};
  e.cols = e.ld_out = a.in_features;
  int64_t most = 0;
  if (a.g_x && a.rows > 0) {
    e.out = a.g_x;
    e.vec = a.in_features % 8 == 0 && aligned16(a.g_x);
    p.gx = {dz, {a.w, a.ld_w, 1}, a.rows, a.in_features, a.out_features, a.dtype, e};
    most = product_workspace(p.gx);
  }
  if (a.g_w && a.rows > 0) {
    e.out = a.g_w;
    e.vec = a.in_features % 8 == 0 && aligned16(a.g_w);
    dz.strided = 1;
    p.gw = {dz, {a.x, a.ld_x, 1}, a.out_features, a.in_features, a.rows, a.dtype, e};
    const int64_t b = product_workspace(p.gw);
    most = most > b ? most : b;
  }
  p.bytes += most;
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
int linear_bwd(const sga_linear& a, char* ws, hipStream_t st) {
  const BwdPlan p = bwd_plan(a, ws);
  const int64_t E = sizeof(T);
  float* part = p.part ? (float*)(ws + p.part_off) : nullptr;
  if ((p.dz || p.part) && a.rows > 0) {
    const int vec = a.out_features % 8 == 0 && aligned16(a.g_out) && a.ld_g_out * E % 16 == 0 && (a.act == SGA_ACT_NONE || aligned16(a.pre));
    hipLaunchKernelGGL((token_dz_kernel<T>), dim3((unsigned)ceil_div(a.out_features, 256), (unsigned)p.chunks), dim3(256), 0, st, (const T*)a.g_out,
                       a.ld_g_out, (const T*)a.pre, a.act, make_drop(a.dropout), p.dz ? (T*)(ws + p.dz_off) : nullptr, p.ld_dz, part, a.rows,
                       (int64_t)a.out_features, p.per, vec);
    LAUNCHED();
  }
  if (p.part) {
    hipLaunchKernelGGL((token_sum_parts_kernel<T>), dim3((unsigned)ceil_div(a.out_features, 32)), dim3(256), 0, st, part, p.chunks, (T*)a.g_bias,
                       (int64_t)a.out_features);
    LAUNCHED();
  }
  if (a.g_x && a.rows > 0) {
    const int s = launch_product(p.gx, ws + p.prod_off, st);
    if (s != SGA_OK) return s;
  }
  if (a.g_w && a.rows > 0) return launch_product(p.gw, ws + p.prod_off, st);
  if (a.g_w) {
    const int64_t n = (int64_t)a.out_features * a.in_features, blocks = ceil_div(n, 256);
    hipLaunchKernelGGL((token_zero_kernel<T>), dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, st, (T*)a.g_w, n);
    LAUNCHED();
  }
  return SGA_OK;
}

}  // namespace

extern "C" {

int sga_op_linear_workspace(const sga_linear* a, int backward, int64_t* bytes) {
  if (!bytes) return SGA_ERR_BAD_ARG;
  const int st = backward ? bwd_check(a) : fwd_check(a);
  if (st != SGA_OK) return st;
  *bytes = backward ? bwd_plan(*a, nullptr).bytes : a->rows > 0 ? product_workspace(forward_product(*a)) : 0;
  return SGA_OK;
}

int sga_op_linear_fwd(const sga_linear* a, void* workspace, int64_t workspace_bytes, void* stream) {
  const int st = fwd_check(a);
  if (st != SGA_OK || a->rows == 0) return st;
  const Product p = forward_product(*a);
  const int64_t need = product_workspace(p);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))) return SGA_ERR_NOMEM;
  return launch_product(p, (char*)workspace, (hipStream_t)stream);
}

int sga_op_linear_bwd(const sga_linear* a, void* workspace, int64_t workspace_bytes, void* stream) {
  const int st = bwd_check(a);
  if (st != SGA_OK) return st;
  const int64_t need = bwd_plan(*a, nullptr).bytes;
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))) return SGA_ERR_NOMEM;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  return a->dtype == SGA_DTYPE_F32 ? linear_bwd<float>(*a, ws, s) : a->dtype == SGA_DTYPE_BF16 ? linear_bwd<bf16>(*a, ws, s) : linear_bwd<f16>(*a, ws, s);
}

}  // extern "C"
