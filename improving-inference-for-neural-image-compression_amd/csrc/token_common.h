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

__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case SGA_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
    case SGA_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case SGA_ACT_GELU_TANH: return 0.5f * z * (1.f + tanhf(0.79788456080286536f * fmaf(0.044715f * z * z, z, z)));
    case SGA_ACT_SILU: return z / (1.f + expf(-z));
    default: return z;
  }
}

__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case SGA_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case SGA_ACT_GELU:
      return fmaf(z * 0.39894228040143268f, expf(-0.5f * z * z), 0.5f * (1.f + erff(z * 0.70710678118654752f)));
    case SGA_ACT_GELU_TANH: {
      const float t = tanhf(0.79788456080286536f * fmaf(0.044715f * z * z, z, z));
      const float c = fminf(fmaxf(z, -16.f), 16.f);      // beyond, 1 - t^2 is 0 and the polynomial must not be inf
      return 0.5f * (1.f + t) + 0.5f * c * (1.f - t * t) * 0.79788456080286536f * fmaf(0.134145f * c, c, 1.f);
    }
    case SGA_ACT_SILU: {
      const float s = 1.f / (1.f + expf(-z));
      return s * fmaf(z, 1.f - s, 1.f);
    }
    default: return 1.f;
  }
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

}  // namespace token
