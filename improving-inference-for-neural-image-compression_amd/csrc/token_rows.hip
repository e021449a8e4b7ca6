// Row operators of token blocks (include/sga_hip.h): layer norm forward and backward, counter-based dropout.
#include "token_common.h"

using namespace token;

namespace {

// ---- rows held in registers ------------------------------------------------------------------------------------------------
// A row of up to 8 V L columns is held by L lanes (one wave, or several waves of a workgroup), V pieces of 8 columns each.  VEC:
// a piece is 16 (32) adjacent bytes; otherwise (odd widths, starts, strides) the lanes take single elements, L apart, so that
// neighbouring lanes still read neighbouring addresses.
template <int L, int V, bool VEC> struct Cols {
  // column of element j of piece v of this lane
  static __device__ __forceinline__ int at(int lane, int v, int j) { return VEC ? (v * L + lane) * 8 + j : (v * 8 + j) * L + lane; }
  template <typename T> static __device__ __forceinline__ void load(const T* row, int lane, int cols, float (*x)[8]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if constexpr (VEC) {
        const int c = at(lane, v, 0);
        if (c < cols) load8(row + c, x[v]);
        else {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[v][j] = 0.f;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) { const int c = at(lane, v, j); x[v][j] = c < cols ? to_f32(row[c]) : 0.f; }
      }
    }
  }
  template <typename T> static __device__ __forceinline__ void store(T* row, int lane, int cols, const float (*x)[8]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if constexpr (VEC) {
        const int c = at(lane, v, 0);
        if (c < cols) store8(row + c, x[v]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) { const int c = at(lane, v, j); if (c < cols) row[c] = from_f32<T>(x[v][j]); }
      }
    }
  }
};

// sums of N values over the L lanes of a row, for each of them; sh: [waves of the workgroup][N], not used again before the
// next barrier of another buffer (callers alternate two)
template <int L, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], float* sh) {
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s[k] += __shfl_xor(s[k], o);
  if constexpr (L > 64) {
    constexpr int W = L / 64;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) sh[wave * N + k] = s[k];
    }
    __syncthreads();
    const int w0 = wave / W * W;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float t = sh[w0 * N + k];
#pragma unroll
      for (int w = 1; w < W; ++w) t += sh[(w0 + w) * N + k];
      s[k] = t;
    }
  }
}

// y = (x - mean) rstd w + b, mean and variance in two passes over the registers.  Bound by HBM.  Workgroups stay and walk the rows:
// weights are loaded once, the next row is on its way while this one is summed.  One piece per lane: 16384 x 4096 bf16 (268 MB)
// 55 us = 4.85 TB/s, against 57 with two pieces on half the lanes and 170 with a workgroup of 256 that reads its row three times.
template <typename T, typename P, int NT, int L, int V, bool VEC>
__global__ __launch_bounds__(NT) void layer_norm_fwd_kernel(const T* __restrict__ x, int64_t ld_x, const P* __restrict__ w, const P* __restrict__ b,
                                                            T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, int64_t rows,
                                                            int cols, float eps) {
  typedef Cols<L, V, VEC> C;
  constexpr int G = NT / L;
  __shared__ float sh[2][NT / 64];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const float n = (float)cols;
  float ww[V][8], bb[V][8], cur[V][8], nxt[V][8];
  if (w) C::load(w, lane, cols, ww);
  else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) ww[v][j] = 1.f;
  }
  if (b) C::load(b, lane, cols, bb);
  else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) bb[v][j] = 0.f;
  }
  const int64_t stride = (int64_t)gridDim.x * G, first = (int64_t)blockIdx.x * G;
  C::load(x + (first + group < rows ? first + group : rows - 1) * ld_x, lane, cols, cur);
  for (int64_t m0 = first; m0 < rows; m0 += stride) {      // the same number of turns for every row group of a workgroup
    const int64_t m = m0 + group, mn = m + stride;
    if (m0 + stride < rows) C::load(x + (mn < rows ? mn : rows - 1) * ld_x, lane, cols, nxt);
    float s[1] = {0.f};
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] += cur[v][j];
    row_sum<L, 1>(s, sh[0]);
    const float mu = s[0] / n;      // divided, not multiplied by 1 / n: the mean of equal values is that value
    float q[1] = {0.f};
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = C::at(lane, v, j) < cols ? cur[v][j] - mu : 0.f;
        cur[v][j] = d;
        q[0] = fmaf(d, d, q[0]);
      }
    row_sum<L, 1>(q, sh[1]);
    const float r = 1.f / sqrtf(q[0] / n + eps);
    if (m < rows) {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) cur[v][j] = fmaf(cur[v][j] * r, ww[v][j], bb[v][j]);
      C::store(y + m * cols, lane, cols, cur);
      if (lane == 0) {
        if (mean) mean[m] = mu;
        if (rstd) rstd[m] = r;
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) cur[v][j] = nxt[v][j];
  }
}

// g_x, and this workgroup's share of g_w and g_b: part[block][0][c] = sum of g_y h, part[block][1][c] = sum of g_y over the rows
// it walks.  Bound by HBM: every tensor once.  The lanes keep their columns' two sums and weights in registers from row to row; the
// row groups of a workgroup add theirs up in LDS at the end, in a fixed order.  8192 x 4096 bf16 with g_add (268 MB): 55 us with the
// join = 4.9 TB/s; 65 without the weights kept and the streams past the caches (they push the weights out), 70 with 512
// workgroups (twice the partial sums), 188 as two kernels that read x and g_y twice.
template <typename T, typename P, int L, int V, bool VEC>
__global__ __launch_bounds__(1024) void layer_norm_bwd_kernel(const T* __restrict__ x, int64_t ld_x, const P* __restrict__ w,
                                                              const T* __restrict__ gy, int64_t ld_gy, const T* __restrict__ add, int64_t ld_add,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ gx,
                                                              float* __restrict__ part, int64_t rows, int cols) {
  typedef Cols<L, V, VEC> C;
  constexpr int G = 1024 / L;
  __shared__ float sh[2][32];
  __shared__ float joint[G > 1 ? 8 * V * L : 1];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const float inv = 1.f / (float)cols;
  float sw[V][8], sb[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int j = 0; j < 8; ++j) sw[v][j] = sb[v][j] = 0.f;
  const int64_t stride = (int64_t)gridDim.x * G, first = (int64_t)blockIdx.x * G;
  // The next row's pieces are on their way while this row is summed; not so single elements, for odd layouts, and two pieces a
  // lane, for which the 128 registers of a lane would not do
  constexpr bool AHEAD = VEC && V == 1;
  Raw8<T> rx[V] = {}, rg[V] = {}, ra[V] = {};
  float rmu = 0.f, rr = 0.f;
  auto ahead = [&](int64_t m) {
    const int64_t at = m < rows ? m : rows - 1;
    rmu = mean[at];
    rr = rstd[at];
    if constexpr (AHEAD) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = C::at(lane, v, 0);
        if (c < cols) {
          rx[v] = raw_once(x + at * ld_x + c);
          rg[v] = raw_once(gy + at * ld_gy + c);
          if (add && gx) ra[v] = raw_once(add + at * ld_add + c);
        }
      }
    }
  };
  auto weights = [&](int v, float ww[8]) {
    if constexpr (VEC) {
      const int c = C::at(lane, v, 0);
      if (w && c < cols) load8(w + c, ww);
      else {
#pragma unroll
        for (int j = 0; j < 8; ++j) ww[j] = 1.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) { const int c = C::at(lane, v, j); ww[j] = w && c < cols ? to_f32(w[c]) : 1.f; }
    }
  };
  float wkept[AHEAD ? V : 1][8];
  if constexpr (AHEAD) weights(0, wkept[0]);
  auto open = [](const Raw8<T> (&raw)[V], float (*f)[8]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      T t[8];
      __builtin_memcpy(t, &raw[v], sizeof(t));
#pragma unroll
      for (int j = 0; j < 8; ++j) f[v][j] = to_f32(t[j]);
    }
  };
  ahead(first + group);
  int turn = 0;
  for (int64_t m0 = first; m0 < rows; m0 += stride, turn ^= 1) {
    const int64_t m = m0 + group, mr = m < rows ? m : rows - 1;
    const bool live = m < rows;
    float h[V][8], g[V][8], a[V][8];
    const float mu = rmu, r = rr;
    if constexpr (AHEAD) {
      open(rx, h);
      open(rg, g);
      open(ra, a);
    } else {
      C::load(x + mr * ld_x, lane, cols, h);
      C::load(gy + mr * ld_gy, lane, cols, g);
    }
    if (m0 + stride < rows) ahead(m + stride);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float ww[8];
      if constexpr (AHEAD) {
#pragma unroll
        for (int j = 0; j < 8; ++j) ww[j] = wkept[v][j];
      } else weights(v, ww);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[v][j] = C::at(lane, v, j) < cols ? (h[v][j] - mu) * r : 0.f;
        if (live) {
          sw[v][j] = fmaf(g[v][j], h[v][j], sw[v][j]);
          sb[v][j] += g[v][j];
        }
        g[v][j] *= ww[j];
        s[0] += g[v][j];
        s[1] = fmaf(g[v][j], h[v][j], s[1]);
      }
    }
    if (!gx) continue;
    row_sum<L, 2>(s, sh[turn]);
    const float c1 = s[0] * inv, c2 = s[1] * inv;
    if (!live) continue;
    if constexpr (!AHEAD) {
      if (add) C::load(add + m * ld_add, lane, cols, a);
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = r * (g[v][j] - c1 - h[v][j] * c2);
        g[v][j] = add ? d + a[v][j] : d;
      }
    C::store(gx + m * cols, lane, cols, g);
  }
  if (!part) return;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    if constexpr (G > 1) {
#pragma unroll 1
      for (int k = 1; k < G; ++k) {      // group k hands its sums to group 0
        __syncthreads();
        if (group == k) {
#pragma unroll
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j) joint[(v * 8 + j) * L + lane] = which ? sb[v][j] : sw[v][j];
        }
        __syncthreads();
        if (group == 0) {
#pragma unroll
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float t = joint[(v * 8 + j) * L + lane];
              if (which) sb[v][j] += t;
              else sw[v][j] += t;
            }
        }
      }
    }
    if (group == 0) {
      float* to = part + ((int64_t)blockIdx.x * 2 + which) * cols;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) { const int c = C::at(lane, v, j); if (c < cols) to[c] = which ? sb[v][j] : sw[v][j]; }
    }
  }
}

// the sum of v over the workgroup of 256, for every lane; sh: 4 floats, free again on return
__device__ __forceinline__ float block_sum(float v, float* sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (sh[0] + sh[1]) + (sh[2] + sh[3]);
  __syncthreads();
  return v;
}

// ---- rows too long for registers: read again for each pass (the second and third time from L2) ------------------------------
// For widths past 16384, kept simple: bound by HBM and L2, a workgroup of 256 per row, single elements a lane, so any
// alignment.  4096 x 20000 bf16 (328 MB) 250 us = 1.3 TB/s with inputs that change (184 with one that stays in the last-level cache); its
// gradients with g_add (656 MB) 516 us.
template <typename T, typename P>
__global__ __launch_bounds__(256) void layer_norm_fwd_long_kernel(const T* __restrict__ x, int64_t ld_x, const P* __restrict__ w,
                                                                  const P* __restrict__ b, T* __restrict__ y, float* __restrict__ mean,
                                                                  float* __restrict__ rstd, int cols, float eps) {
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
__global__ __launch_bounds__(256) void layer_norm_gx_long_kernel(const T* __restrict__ x, int64_t ld_x, const P* __restrict__ w,
                                                                 const T* __restrict__ gy, int64_t ld_gy, const T* __restrict__ add,
                                                                 int64_t ld_add, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                 T* __restrict__ gx, int cols) {
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

// part as in layer_norm_bwd_kernel, block y walks rows y, y + gridDim.y, ...
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_parts_long_kernel(const T* __restrict__ x, int64_t ld_x, const T* __restrict__ gy, int64_t ld_gy,
                                                                    const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                    float* __restrict__ part, int64_t rows, int cols) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float sw = 0.f, sb = 0.f;
  for (int64_t m = blockIdx.y; m < rows; m += gridDim.y) {
    const float g = to_f32(gy[m * ld_gy + c]);
    sw = fmaf(g, (to_f32(x[m * ld_x + c]) - mean[m]) * rstd[m], sw);
    sb += g;
  }
  part[((int64_t)blockIdx.y * 2) * cols + c] = sw;
  part[((int64_t)blockIdx.y * 2 + 1) * cols + c] = sb;
}

// g_w, g_b = the sums of nparts partial sums, in a fixed order: 32 columns (of the 2 cols) x 8 runs of partial sums per workgroup.
// Bound by latency: 256 parts of 2 x 4096 (8 MB, from L2) 4.9 us.
template <typename P>
__global__ __launch_bounds__(256) void layer_norm_join_kernel(const float* __restrict__ part, int nparts, P* __restrict__ gw, P* __restrict__ gb,
                                                              int cols) {
  __shared__ float sh[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + tx;
  const int per = (nparts + 7) / 8, p0 = ty * per, p1 = p0 + per < nparts ? p0 + per : nparts;
  float s = 0.f;
  if (c < 2 * (int64_t)cols) {
#pragma unroll 8
    for (int p = p0; p < p1; ++p) s += part[(int64_t)p * 2 * cols + c];
  }
  sh[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < 2 * (int64_t)cols) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sh[k][tx];
    P* to = c < cols ? gw : gb;
    if (to) to[c < cols ? c : c - cols] = from_f32<P>(s);
  }
}

// ---- dropout ---------------------------------------------------------------------------------------------------------------
// Tensors without gaps, 16-byte aligned: 8 adjacent elements per lane, whatever the row length -- the counter runs over the
// whole matrix.  The last piece may be short.  Bound by HBM, with the 20 Philox rounds a piece under the loads: 8192 x 8192 bf16 with
// residual (403 MB) 64 us = 6.3 TB/s (72 through the caches).
template <typename T, bool RES>
__global__ __launch_bounds__(256) void dropout_flat_kernel(const T* x, const T* res, T* y, int64_t n, const Drop d) {
  uint64_t seed = 0, offset = 0;
  if (d.on) drop_key(d, seed, offset);
  const int64_t pieces = n >> 3;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i <= pieces; i += (int64_t)gridDim.x * 256) {
    uint32_t w[8];
    float v[8], r[8];
    if (i < pieces) {
      load8_once(x + i * 8, v);
      if constexpr (RES) load8_once(res + i * 8, r);
    }
    if (d.on) {
      drop_words(seed, offset, (uint64_t)i * 2, w);
      drop_words(seed, offset, (uint64_t)i * 2 + 1, w + 4);
    }
    if (i < pieces) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (d.on) v[j] = drop_apply(d, w[j], v[j]);
        if constexpr (RES) v[j] += r[j];
      }
      store8_once(y + i * 8, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i * 8 + j < n) {
          float u = to_f32(x[i * 8 + j]);
          if (d.on) u = drop_apply(d, w[j], u);
          if constexpr (RES) u += to_f32(res[i * 8 + j]);
          y[i * 8 + j] = from_f32<T>(u);
        }
    }
  }
}

// rows with gaps, any alignment: the 4 elements of one counter per lane, which may lie in several rows.  Bound by the element loads:
// 8192 x 8190 bf16 of stride 8196 with residual 181 us, without gaps 64.
template <typename T>
__global__ __launch_bounds__(256) void dropout_rows_kernel(const T* x, int64_t ld_x, const T* res, int64_t ld_res, T* y, int64_t rows, int64_t cols,
                                                           const Drop d) {
  uint64_t seed = 0, offset = 0;
  if (d.on) drop_key(d, seed, offset);
  const int64_t n = rows * cols, groups = (n + 3) >> 2;
  for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < groups; g += (int64_t)gridDim.x * 256) {
    uint32_t w[4];
    if (d.on) drop_words(seed, offset, (uint64_t)g, w);
    int64_t m = g * 4 / cols, c = g * 4 - m * cols;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (g * 4 + j < n) {
        float u = to_f32(x[m * ld_x + c]);
        if (d.on) u = drop_apply(d, w[j], u);
        if (res) u += to_f32(res[m * ld_res + c]);
        y[g * 4 + j] = from_f32<T>(u);
      }
      if (++c == cols) { c = 0; ++m; }
    }
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

constexpr int kHeld = 16384;      // the widest row that is held in registers

// Rows of the backward pass are dealt to at most 256 workgroups of 1024 lanes (one per CU): its partial sums of g_w, g_b are 256 x 2
// rows of float32 then, 3 % of the traffic at 8192 rows.  Long rows: 64 runs of rows.
int bwd_lanes(int cols) { return cols <= 512 ? 64 : cols <= 1024 ? 128 : cols <= 2048 ? 256 : cols <= 4096 ? 512 : 1024; }
int norm_parts(const sga_layer_norm& a) {
  if (a.rows == 0) return 0;
  const int64_t n = a.cols > kHeld ? a.rows : ceil_div(a.rows, 1024 / bwd_lanes(a.cols));
  const int64_t most = a.cols > kHeld ? 64 : 256;
  return (int)(n < most ? n : most);
}
int64_t norm_bwd_bytes(const sga_layer_norm& a) {
  return (a.g_w || a.g_b) ? round_up((int64_t)norm_parts(a) * 2 * a.cols * 4, 256) : 0;
}

bool piece_ok(const void* p, int64_t ld, int64_t cols, int dtype) {
  return ((uintptr_t)p & 15) == 0 && (ld * (int64_t)dtype_bytes(dtype)) % 16 == 0 && cols % 8 == 0;
}

template <typename T, typename P, int NT, int L, int V>
int norm_fwd_held(const sga_layer_norm& a, bool vec, hipStream_t st) {
  const int64_t groups = ceil_div(a.rows, NT / L);
  const dim3 grid((unsigned)(groups < 2048 ? groups : 2048));
  if (vec)
    hipLaunchKernelGGL((layer_norm_fwd_kernel<T, P, NT, L, V, true>), grid, dim3(NT), 0, st, (const T*)a.x, a.ld_x, (const P*)a.w, (const P*)a.b, (T*)a.y,
                       a.mean, a.rstd, a.rows, a.cols, a.eps);
  else
    hipLaunchKernelGGL((layer_norm_fwd_kernel<T, P, NT, L, V, false>), grid, dim3(NT), 0, st, (const T*)a.x, a.ld_x, (const P*)a.w, (const P*)a.b, (T*)a.y,
                       a.mean, a.rstd, a.rows, a.cols, a.eps);
  LAUNCHED();
  return SGA_OK;
}

template <typename T, typename P>
int norm_fwd(const sga_layer_norm& a, hipStream_t st) {
  const bool vec = piece_ok(a.x, a.ld_x, a.cols, a.dtype) && piece_ok(a.y, a.cols, a.cols, a.dtype) && piece_ok(a.w, 0, a.cols, a.param_dtype) &&
                   piece_ok(a.b, 0, a.cols, a.param_dtype);
  if (a.cols <= 512) return norm_fwd_held<T, P, 256, 64, 1>(a, vec, st);
  if (a.cols <= 1024) return norm_fwd_held<T, P, 256, 128, 1>(a, vec, st);
  if (a.cols <= 2048) return norm_fwd_held<T, P, 256, 256, 1>(a, vec, st);
  if (a.cols <= 4096) return norm_fwd_held<T, P, 512, 512, 1>(a, vec, st);
  if (a.cols <= 8192) return norm_fwd_held<T, P, 1024, 1024, 1>(a, vec, st);
  if (a.cols <= kHeld) return norm_fwd_held<T, P, 1024, 1024, 2>(a, vec, st);
  hipLaunchKernelGGL((layer_norm_fwd_long_kernel<T, P>), dim3((unsigned)a.rows), dim3(256), 0, st, (const T*)a.x, a.ld_x, (const P*)a.w, (const P*)a.b,
                     (T*)a.y, a.mean, a.rstd, a.cols, a.eps);
  LAUNCHED();
  return SGA_OK;
}

template <typename T, typename P, int L, int V>
int norm_bwd_held(const sga_layer_norm& a, bool vec, float* part, int nparts, hipStream_t st) {
  if (vec)
    hipLaunchKernelGGL((layer_norm_bwd_kernel<T, P, L, V, true>), dim3(nparts), dim3(1024), 0, st, (const T*)a.x, a.ld_x, (const P*)a.w, (const T*)a.g_y,
                       a.ld_g_y, (const T*)a.g_add, a.ld_g_add, a.mean, a.rstd, (T*)a.g_x, part, a.rows, a.cols);
  else
    hipLaunchKernelGGL((layer_norm_bwd_kernel<T, P, L, V, false>), dim3(nparts), dim3(1024), 0, st, (const T*)a.x, a.ld_x, (const P*)a.w, (const T*)a.g_y,
                       a.ld_g_y, (const T*)a.g_add, a.ld_g_add, a.mean, a.rstd, (T*)a.g_x, part, a.rows, a.cols);
  LAUNCHED();
  return SGA_OK;
}

template <typename T, typename P>
int norm_bwd(const sga_layer_norm& a, float* ws, hipStream_t st) {
  const int np = norm_parts(a);
  float* part = (a.g_w || a.g_b) ? ws : nullptr;
  if (a.rows > 0 && (a.g_x || part)) {
    int s = SGA_OK;
    if (a.cols <= kHeld) {
      const bool vec = piece_ok(a.x, a.ld_x, a.cols, a.dtype) && piece_ok(a.g_y, a.ld_g_y, a.cols, a.dtype) &&
                       piece_ok(a.g_add, a.g_add ? a.ld_g_add : 0, a.cols, a.dtype) && piece_ok(a.g_x, a.cols, a.cols, a.dtype) &&
                       piece_ok(a.w, 0, a.cols, a.param_dtype);
      if (a.cols <= 512) s = norm_bwd_held<T, P, 64, 1>(a, vec, part, np, st);
      else if (a.cols <= 1024) s = norm_bwd_held<T, P, 128, 1>(a, vec, part, np, st);
      else if (a.cols <= 2048) s = norm_bwd_held<T, P, 256, 1>(a, vec, part, np, st);
      else if (a.cols <= 4096) s = norm_bwd_held<T, P, 512, 1>(a, vec, part, np, st);
      else if (a.cols <= 8192) s = norm_bwd_held<T, P, 1024, 1>(a, vec, part, np, st);
      else s = norm_bwd_held<T, P, 1024, 2>(a, vec, part, np, st);
    } else {
      if (a.g_x) {
        hipLaunchKernelGGL((layer_norm_gx_long_kernel<T, P>), dim3((unsigned)a.rows), dim3(256), 0, st, (const T*)a.x, a.ld_x, (const P*)a.w,
                           (const T*)a.g_y, a.ld_g_y, (const T*)a.g_add, a.ld_g_add, a.mean, a.rstd, (T*)a.g_x, a.cols);
        LAUNCHED();
      }
      if (part) {
        hipLaunchKernelGGL((layer_norm_parts_long_kernel<T>), dim3((unsigned)ceil_div(a.cols, 256), (unsigned)np), dim3(256), 0, st, (const T*)a.x,
                           a.ld_x, (const T*)a.g_y, a.ld_g_y, a.mean, a.rstd, part, a.rows, a.cols);
        LAUNCHED();
      }
    }
    if (s != SGA_OK) return s;
  }
  if (part || a.g_w || a.g_b) {
    hipLaunchKernelGGL((layer_norm_join_kernel<P>), dim3((unsigned)ceil_div(2 * (int64_t)a.cols, 32)), dim3(256), 0, st, part, np, (P*)a.g_w, (P*)a.g_b,
                       a.cols);
    LAUNCHED();
  }
  return SGA_OK;
}

template <typename T>
int dropout_run(const void* x, int64_t ld_x, const void* res, int64_t ld_res, void* y, int64_t rows, int64_t cols, const Drop& d, hipStream_t st) {
  const bool flat = ((uintptr_t)x & 15) == 0 && ((uintptr_t)y & 15) == 0 && ((uintptr_t)res & 15) == 0 && (rows == 1 || ld_x == cols) &&
                    (!res || rows == 1 || ld_res == cols);
  const int64_t n = rows * cols, blocks = ceil_div(flat ? (n >> 3) + 1 : (n + 3) >> 2, 256);
  const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
  if (flat && res) hipLaunchKernelGGL((dropout_flat_kernel<T, true>), grid, dim3(256), 0, st, (const T*)x, (const T*)res, (T*)y, n, d);
  else if (flat) hipLaunchKernelGGL((dropout_flat_kernel<T, false>), grid, dim3(256), 0, st, (const T*)x, (const T*)res, (T*)y, n, d);
  else hipLaunchKernelGGL((dropout_rows_kernel<T>), grid, dim3(256), 0, st, (const T*)x, ld_x, (const T*)res, ld_res, (T*)y, rows, cols, d);
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
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))) return SGA_ERR_NOMEM;
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
