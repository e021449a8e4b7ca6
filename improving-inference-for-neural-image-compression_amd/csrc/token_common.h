// Shared device code of the token-block operators (token_linear.hip, token_rows.hip): element types, activations, dropout words.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "../../include/sga_hip.h"
#include "sga_common.h"

namespace token {

typedef __bf16 bf16;
typedef _Float16 f16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(f16 v) { return (float)v; }
// the one rounding of a result: to nearest, ties to even
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

// e^x to 2 units in the last place: 2^(x log2 e) by the hardware's exp2, and the part of x log2 e that float32 cannot hold as a
// factor.  The clamp keeps infinities out of that part; a NaN becomes some number, every use multiplies by x again.
// SHORT (results of 16 bits, whose half step is 2^-12 at the least): without that part, off by |x| 2^-24.
template <bool SHORT> __device__ __forceinline__ float exp_f(float x) {
  if constexpr (SHORT) return __builtin_amdgcn_exp2f(x * 1.44269504f);
  x = fminf(fmaxf(x, -1000.f), 1000.f);
  const float t = x * 1.44269504f;
  const float e = fmaf(x, 1.925963033e-8f, fmaf(x, 1.44269504f, -t));
  return __builtin_amdgcn_exp2f(t) * fmaf(e, 0.69314718f, 1.f);
}

// Phi(-|z|) = erfc(|z| / sqrt 2) / 2 = g(|z|) e^(-z^2 / 2) with g smooth and slowly varying: g as a polynomial in t = 1 / (1 + 0.3 |z|),
// fitted on 0 <= |z| <= 14 for the least maximum of the relative error (beyond, the exponential is 0): degree 8, with its constants as
// float32 holds them, is off by 1.1e-7 in exact arithmetic, 4e-7 with float32 steps; degree 6, for SHORT results, by 1.9e-6 and 2.2e-6.  Relative accuracy in the tail is what
// 1 + erf(z) cannot give, and the backward pass shares the exponential: about 25 (SHORT: 18) instructions where the
// library's erf and exp take about 60.
template <bool SHORT> __device__ __forceinline__ float normal_tail(float z, float gauss) {
  const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.3f, 1.f));
  float p;
  if constexpr (SHORT) {
    p = -0.08459318429231644f;
    p = fmaf(p, t, 0.24057263135910034f);
    p = fmaf(p, t, -0.04864419996738434f);
    p = fmaf(p, t, 0.16476432979106903f);
    p = fmaf(p, t, 0.10670459270477295f);
    p = fmaf(p, t, 0.1212746873497963f);
    p = fmaf(p, t, -7.978831126820296e-05f);
  } else {
    p = 0.038378264755010605f;
    p = fmaf(p, t, -0.16916599869728088f);
    p = fmaf(p, t, 0.22865986824035645f);
    p = fmaf(p, t, -0.07650627195835114f);
    p = fmaf(p, t, 0.14253540337085724f);
    p = fmaf(p, t, 0.09468357264995575f);
    p = fmaf(p, t, 0.12192033231258392f);
    p = fmaf(p, t, 0.1194876879453659f);
    p = fmaf(p, t, 7.168815500335768e-06f);
  }
  return p * gauss;
}

template <int ACT, bool SHORT> __device__ __forceinline__ float act_value_of(float z) {
  if constexpr (ACT == SGA_ACT_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
  if constexpr (ACT == SGA_ACT_GELU) {
    const float q = normal_tail<SHORT>(z, exp_f<SHORT>(-0.5f * z * z));
    return z * (z > 0.f ? 1.f - q : q);
  }
  if constexpr (ACT == SGA_ACT_GELU_TANH)
    return z * __builtin_amdgcn_rcpf(1.f + exp_f<SHORT>(-1.59576912f * fmaf(0.044715f * z * z, z, z)));
  if constexpr (ACT == SGA_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + exp_f<SHORT>(-z));
  return z;
}
template <int ACT, bool SHORT> __device__ __forceinline__ float act_slope_of(float z) {
  if constexpr (ACT == SGA_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == SGA_ACT_GELU) {
    const float gauss = exp_f<SHORT>(-0.5f * z * z), q = normal_tail<SHORT>(z, gauss);
    return fmaf(z * 0.39894228040143268f, gauss, z > 0.f ? 1.f - q : q);
  }
  if constexpr (ACT == SGA_ACT_GELU_TANH) {
    const float e = exp_f<SHORT>(-1.59576912f * fmaf(0.044715f * z * z, z, z)), s = __builtin_amdgcn_rcpf(1.f + e);
    const float c = fminf(fmaxf(z, -16.f), 16.f);      // s (1 - s) is 0 beyond, and the polynomial must not be inf
    const float d = s * (s > 0.f ? e * s : 0.f);       // s (1 - s) without the difference
    return fmaf(c * d, 1.59576912f * fmaf(0.134145f * c, c, 1.f), s) + (z - z);
  }
  if constexpr (ACT == SGA_ACT_SILU) {
    const float e = exp_f<SHORT>(-z), s = __builtin_amdgcn_rcpf(1.f + e);
    return s > 0.f ? s * fmaf(z, e * s, 1.f) : (z - z);
  }
  return 1.f;
}
// v[j] = act(v[j]); g[j] *= act'(v[j]);  T: the type of the result
template <typename T, int N> __device__ __forceinline__ void act_values(float v[N], int act) {
#define EACH(A) case A: _Pragma("unroll") for (int j = 0; j < N; ++j) v[j] = act_value_of<A, sizeof(T) == 2>(v[j]); break
  switch (act) { EACH(SGA_ACT_RELU); EACH(SGA_ACT_GELU); EACH(SGA_ACT_GELU_TANH); EACH(SGA_ACT_SILU); default: break; }
#undef EACH
}
template <typename T, int N> __device__ __forceinline__ void act_slopes(float g[N], const float v[N], int act) {
#define EACH(A) case A: _Pragma("unroll") for (int j = 0; j < N; ++j) g[j] *= act_slope_of<A, sizeof(T) == 2>(v[j]); break
  switch (act) { EACH(SGA_ACT_RELU); EACH(SGA_ACT_GELU); EACH(SGA_ACT_GELU_TANH); EACH(SGA_ACT_SILU); default: break; }
#undef EACH
}

// Dropout as the kernels take it.  keep: word >= thr (thr = round(p 2^32), up to 2^32: nothing is kept); on = 0: no dropout.
struct Drop {
  int on;
  uint32_t thr_lo, thr_all;      // thr_all = 1: p rounds to 1
  float scale;
  uint64_t seed, offset;
  const uint64_t* state;
};

inline Drop make_drop(const sga_dropout& d) {
  Drop o = {};
  if (d.p <= 0.0) return o;
  o.on = 1;
  const double t = d.p * 4294967296.0;
  const uint64_t thr = t >= 4294967295.5 ? (1ull << 32) : (uint64_t)__builtin_rint(t);
  o.thr_lo = (uint32_t)thr;
  o.thr_all = thr >> 32 ? 1u : 0u;
  o.scale = o.thr_all ? 0.f : (float)(1.0 / (1.0 - d.p));
  o.seed = d.seed;
  o.offset = d.offset;
  o.state = d.state;
  return o;
}
inline bool drop_ok(const sga_dropout& d) { return d.p >= 0.0 && d.p <= 1.0 && ((uintptr_t)d.state & 7) == 0; }

__device__ __forceinline__ void drop_key(const Drop& d, uint64_t& seed, uint64_t& offset) {
  seed = d.state ? d.state[0] : d.seed;
  offset = d.state ? d.state[1] : d.offset;
}
// the four words of elements 4 g .. 4 g + 3
__device__ __forceinline__ void drop_words(uint64_t seed, uint64_t offset, uint64_t g, uint32_t w[4]) {
  philox4x32_10((uint32_t)g, (uint32_t)(g >> 32), (uint32_t)offset, (uint32_t)(offset >> 32), (uint32_t)seed, (uint32_t)(seed >> 32), w);
}
// a dropped element is 0 whatever it held: select, do not multiply
__device__ __forceinline__ float drop_apply(const Drop& d, uint32_t word, float v) {
  return (word >= d.thr_lo && !d.thr_all) ? v * d.scale : 0.f;
}
__device__ __forceinline__ float drop_one(const Drop& d, uint64_t seed, uint64_t offset, uint64_t i, float v) {
  uint32_t w[4];
  drop_words(seed, offset, i >> 2, w);
  const int j = (int)(i & 3);
  return drop_apply(d, j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3], v);
}

inline size_t dtype_bytes(int t) { return t == SGA_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int t) { return t == SGA_DTYPE_F32 || t == SGA_DTYPE_BF16 || t == SGA_DTYPE_F16; }
// a pointer that its element type allows
inline bool at_ok(const void* p, int dtype) { return ((uintptr_t)p & (dtype_bytes(dtype) - 1)) == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }


// ---- epilogue of a product: 8 adjacent columns of one row ----------------------------------------------------------------
struct Epilogue {
  const void* bias; const void* residual; int64_t ld_residual; void* out; int64_t ld_out; void* pre; int64_t cols; int act;
  int vec;       // every row piece of 8 columns is whole and 16-byte aligned in every tensor
  Drop drop;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// 8 adjacent elements, 16-byte aligned
__device__ __forceinline__ void load8(const float* p, float v[8]) {
  const f32x4 a = ((const f32x4*)p)[0], b = ((const f32x4*)p)[1];
#pragma unroll
  for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
}
template <typename T> __device__ __forceinline__ void load8(const T* p, float v[8]) {
  typedef T t8 __attribute__((ext_vector_type(8)));
  const t8 a = *(const t8*)p;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)a[j];
}
__device__ __forceinline__ void store8(float* p, const float v[8]) {
  ((f32x4*)p)[0] = f32x4{v[0], v[1], v[2], v[3]};
  ((f32x4*)p)[1] = f32x4{v[4], v[5], v[6], v[7]};
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float v[8]) {
  typedef T t8 __attribute__((ext_vector_type(8)));
  t8 a;
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = from_f32<T>(v[j]);
  *(t8*)p = a;
}

// the same past the caches, for streams that nothing on this XCD reads again soon
template <typename T> __device__ __forceinline__ void load8_once(const T* p, float v[8]) {
  constexpr int Q = sizeof(T) / 2;
  u32x4 q[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) q[i] = __builtin_nontemporal_load((const u32x4*)p + i);
  T t[8];
  __builtin_memcpy(t, q, sizeof(t));
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = to_f32(t[j]);
}
template <typename T> __device__ __forceinline__ void store8_once(T* p, const float v[8]) {
  constexpr int Q = sizeof(T) / 2;
  T t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = from_f32<T>(v[j]);
  u32x4 q[Q];
  __builtin_memcpy(q, t, sizeof(t));
#pragma unroll
  for (int i = 0; i < Q; ++i) __builtin_nontemporal_store(q[i], (u32x4*)p + i);
}

// The residual is loaded apart from the rest (residual8), so that a lane can have several rows' on their way: the
// compiler may not move a load before a store to `out`, which may be the same tensor.
template <typename T> struct Raw8 { u32x4 q[sizeof(T) / 2]; };      // 8 elements as they lie
template <typename T> __device__ __forceinline__ Raw8<T> raw_once(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.q[i] = __builtin_nontemporal_load((const u32x4*)p + i);
  return r;
}
template <typename T>
__device__ __forceinline__ Raw8<T> residual8(const Epilogue& e, int64_t m, int64_t n) {
  Raw8<T> r = {};
  if (e.residual) r = *(const Raw8<T>*)((const T*)e.residual + m * e.ld_residual + n);
  return r;
}
template <typename T> __device__ __forceinline__ void bias8(const Epilogue& e, int64_t n, float b[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) b[j] = 0.f;
  if (e.bias) load8((const T*)e.bias + n, b);
}
// columns n .. n + 7 of row m, all of them there and aligned (e.vec); seed / offset: drop_key's.  ONCE: the results bypass the caches
template <typename T, bool ONCE = false>
__device__ __forceinline__ void epilogue8(const Epilogue& e, uint64_t seed, uint64_t offset, int64_t m, int64_t n, float v[8], const float b[8],
                                          const Raw8<T>& res) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] += b[j];
  if (e.pre) {
    if constexpr (ONCE) store8_once((T*)e.pre + m * e.cols + n, v);
    else store8((T*)e.pre + m * e.cols + n, v);
  }
  act_values<T, 8>(v, e.act);
  if (e.drop.on) {
    const uint64_t g = (uint64_t)(m * e.cols + n) >> 2;      // cols and n are multiples of 8 here
    uint32_t w[8];
    drop_words(seed, offset, g, w);
    drop_words(seed, offset, g + 1, w + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = drop_apply(e.drop, w[j], v[j]);
  }
  if (e.residual) {
    T r[8];
    __builtin_memcpy(r, &res, sizeof(r));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += to_f32(r[j]);
  }
  if constexpr (ONCE) store8_once((T*)e.out + m * e.ld_out + n, v);
  else store8((T*)e.out + m * e.ld_out + n, v);
}
// N elements (m[j], n[j]) of any row length and alignment: lanes take neighbouring columns.  live: bit j = it exists
__device__ __noinline__ inline uint32_t drop_word(uint64_t seed, uint64_t offset, uint64_t i) {
  uint32_t w[4];
  drop_words(seed, offset, i >> 2, w);
  const int j = (int)(i & 3);
  return j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3];
}
template <typename T, int N>
__device__ __forceinline__ void epilogue1(const Epilogue& e, uint64_t seed, uint64_t offset, const int64_t m[N], const int64_t n[N], unsigned live,
                                          float u[N]) {
  float res[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    res[j] = 0.f;
    if (live >> j & 1) {
      if (e.residual) res[j] = to_f32(((const T*)e.residual)[m[j] * e.ld_residual + n[j]]);
      if (e.bias) u[j] += to_f32(((const T*)e.bias)[n[j]]);
    }
  }
  if (e.pre) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (live >> j & 1) ((T*)e.pre)[m[j] * e.cols + n[j]] = from_f32<T>(u[j]);
  }
  act_values<T, N>(u, e.act);
  if (e.drop.on) {
#pragma unroll
    for (int j = 0; j < N; ++j) u[j] = drop_apply(e.drop, drop_word(seed, offset, (uint64_t)(m[j] * e.cols + n[j])), u[j]);
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (live >> j & 1) ((T*)e.out)[m[j] * e.ld_out + n[j]] = from_f32<T>(e.residual ? u[j] + res[j] : u[j]);
}

// ---- C[m, n] = epilogue(sum_k X(m, k) W(n, k)) (token_product.hip) -------------------------------------------------------
// strided = 0: operand(r, k) = p[r ld + k]; strided = 1: operand(r, k) = p[k ld + r]
struct Operand { const void* p; int64_t ld; int strided; };
struct Product {
  Operand x, w;
  int64_t M, N, K;               // at least 1 each
  int dtype;
  Epilogue e;
};
// device workspace (bytes) of launch_product with these members, and the launch itself: 0 or an sga_status
int64_t product_workspace(const Product& p);
int launch_product(const Product& p, char* ws, hipStream_t st);

}  // namespace token
