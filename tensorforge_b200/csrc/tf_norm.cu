// tf_norm.cu -- root-mean-square norm with the residual's addition (f32, bf16 or 8-bit output with
// a scale a row), its gradient, and the row quantizer the 8-bit linear layer's operands come from.
//
// Forward, row by row, in f32:
//   s = x + residual;  rstd = (mean(s^2) + eps)^-1/2;  y = (s w) rstd
//   8-bit output: scale = max(max|y| / 448, 2^-126), q = e4m3(y / scale)
// The row stays in registers between its one read and its one write: t = s w is kept, and because
// rounding is monotone max|y| is fl(max|t| * rstd), so the sum of squares and the maximum come out
// of the same block reduction.  The maximum is taken over bit patterns, in which a NaN is larger
// than every number: a NaN anywhere in the row makes its scale, and so all its 8-bit values, NaN.
//
// Gradient, with hat = s rstd and g = dy w:
//   dx = rstd (g - hat mean(g hat)) + ds;   dweight[n] = sum_m dy[m, n] hat[m, n]
// Blocks walk over rows with the columns' sums in registers; each block stores its sums as one row
// of a scratch array, and a second kernel adds those rows in order (no atomics: the same bits every
// time).
//
// Both are bound by HBM: x, residual, sum and out (or dy, s, ds and dx) cross it once each.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "tf_internal.h"
#include "tf_ptx.cuh"

namespace tf {

namespace {

enum NormOut : int { OUT_F32 = 0, OUT_BF16 = 1, OUT_E4M3 = 2 };

constexpr float kE4m3Max = 448.0f;
constexpr float kTinyScale = 1.17549435e-38f;  // 2^-126: a row of zeros keeps a finite inverse

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// Eight consecutive elements at a 16-byte boundary.  Plain loads: sum_out may be x or the residual,
// dx may be ds (every element is read by the thread that then writes it).
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
  reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&v)[8]) {
  *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                             pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store1(float *p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// Two values rounded to e4m3 (nearest even, saturating, NaN kept): lo in bits [0, 8).
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}

// Sum of `a` and maximum of `b` over the T threads of one row.  `sm`: 2 x 32 words of shared memory
// of the row's own (T > 32).  Every thread gets the same bits.
template <int T>
__device__ __forceinline__ void row_reduce(float &a, uint32_t &b, uint32_t *sm) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
    b = max(b, __shfl_xor_sync(0xFFFFFFFFu, b, o));
  }
  if constexpr (T > 32) {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) {
      sm[w] = __float_as_uint(a);
      sm[32 + w] = b;
    }
    __syncthreads();
    constexpr int W = T / 32;
    a = lane < W ? __uint_as_float(sm[lane]) : 0.f;
    b = lane < W ? sm[32 + lane] : 0u;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
      b = max(b, __shfl_xor_sync(0xFFFFFFFFu, b, o));
    }
  }
}

__device__ __forceinline__ float weight_at(const NormArgs &p, int64_t c) {
  if (!p.weight) return 1.f;
  return p.w_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p.weight)[c])
                  : static_cast<const float *>(p.weight)[c];
}
__device__ __forceinline__ void weight8(const NormArgs &p, int64_t c, float (&w)[8]) {
  if (!p.weight) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.f;
  } else if (p.w_bf16) {
    load8(static_cast<const __nv_bfloat16 *>(p.weight) + c, w);
  } else {
    load8(static_cast<const float *>(p.weight) + c, w);
  }
}

template <int OUT>
__device__ __forceinline__ void out8(const NormArgs &p, int64_t m, int64_t c, const float (&y)[8]) {
  if constexpr (OUT == OUT_F32) store8(static_cast<float *>(p.out) + m * p.ldo + c, y);
  else if constexpr (OUT == OUT_BF16) store8(static_cast<__nv_bfloat16 *>(p.out) + m * p.ldo + c, y);
  else
    *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(p.out) + m * p.ldo + c) =
        make_uint2(pack_e4m3x2(y[0], y[1]) | pack_e4m3x2(y[2], y[3]) << 16,
                   pack_e4m3x2(y[4], y[5]) | pack_e4m3x2(y[6], y[7]) << 16);
}
template <int OUT>
__device__ __forceinline__ void out1(const NormArgs &p, int64_t m, int64_t c, float y) {
  if constexpr (OUT == OUT_F32) static_cast<float *>(p.out)[m * p.ldo + c] = y;
  else if constexpr (OUT == OUT_BF16) static_cast<__nv_bfloat16 *>(p.out)[m * p.ldo + c] = __float2bfloat16_rn(y);
  else static_cast<uint8_t *>(p.out)[m * p.ldo + c] = (uint8_t)pack_e4m3x2(y, 0.f);
}

// The factor from t to what the output type holds, and the row's scale and rstd written by one thread.
template <int OUT, bool NORM>
__device__ __forceinline__ float finish_row(const NormArgs &p, int64_t m, float sumsq, uint32_t amax_bits, bool writer) {
  float f = 1.f;
  if constexpr (NORM) {
    f = __frsqrt_rn(__fadd_rn(__fdiv_rn(sumsq, (float)p.N), p.eps));
    if (writer && p.rstd) p.rstd[m] = f;
  }
  if constexpr (OUT == OUT_E4M3) {
    float scale = __fdiv_rn(__uint_as_float(amax_bits) * f, kE4m3Max);
    scale = scale < kTinyScale ? kTinyScale : scale;  // keeps a NaN
    if (writer) p.scale[m] = scale;
    return scale;
  }
  return f;
}

// One row on T threads, E elements a thread in registers; 32-thread rows share a block of eight.
// VEC: groups of eight consecutive elements (all rows on 16-byte boundaries, N a multiple of 8);
// else single elements, T apart.  NORM false: the quantizer (y = x).
template <typename X, int OUT, bool VEC, int T, int E, bool NORM>
__global__ void __launch_bounds__(T == 32 ? 256 : T) norm_row_kernel(const NormArgs p) {
  grid_dependency_wait();
  grid_launch_dependents();
  constexpr int kRows = T == 32 ? 8 : 1;
  __shared__ uint32_t sm[64];
  const int t = T == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t m = (int64_t)blockIdx.x * kRows + (T == 32 ? threadIdx.x >> 5 : 0);
  if (kRows > 1 && m >= p.M) return;  // whole warps: nothing below waits for them
  const int N = (int)p.N;
  const X *x = static_cast<const X *>(p.x) + m * p.ldx;
  const X *r = p.residual ? static_cast<const X *>(p.residual) + m * p.ldr : nullptr;
  X *so = p.sum_out ? static_cast<X *>(p.sum_out) + m * p.lds : nullptr;
  float v[E];
  float sumsq = 0.f;
  uint32_t amax = 0u;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
      const int c = (i * T + t) * 8;
      float (&s)[8] = *reinterpret_cast<float (*)[8]>(&v[8 * i]);
      if (c < N) {
        load8(x + c, s);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = 0.f;
      }
    }
    if (r) {
#pragma unroll
      for (int i = 0; i < E / 8; ++i) {
        const int c = (i * T + t) * 8;
        if (c < N) {
          float q[8];
          load8(r + c, q);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[8 * i + j] = __fadd_rn(v[8 * i + j], q[j]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
      const int c = (i * T + t) * 8;
      float (&s)[8] = *reinterpret_cast<float (*)[8]>(&v[8 * i]);
      if (c < N) {
        if (so) store8(so + c, s);
        if constexpr (NORM) {
          float w[8];
          weight8(p, c, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sumsq = fmaf(s[j], s[j], sumsq);
            s[j] *= w[j];
          }
        }
        if constexpr (OUT == OUT_E4M3) {
#pragma unroll
          for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(s[j]) & 0x7FFFFFFFu);
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = i * T + t;
      v[i] = c < N ? to_f32(x[c]) : 0.f;
    }
    if (r) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = i * T + t;
        if (c < N) v[i] = __fadd_rn(v[i], to_f32(r[c]));
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = i * T + t;
      if (c < N) {
        if (so) store1(so + c, v[i]);
        if constexpr (NORM) {
          sumsq = fmaf(v[i], v[i], sumsq);
          v[i] *= weight_at(p, c);
        }
        if constexpr (OUT == OUT_E4M3) amax = max(amax, __float_as_uint(v[i]) & 0x7FFFFFFFu);
      }
    }
  }
  row_reduce<T>(sumsq, amax, sm);
  const float f = finish_row<OUT, NORM>(p, m, sumsq, amax, t == 0);
  // 8 bits: y / scale with y = t rstd, as y times the scale's inverse.
  const float rs = OUT == OUT_E4M3 && NORM ? __frsqrt_rn(__fadd_rn(__fdiv_rn(sumsq, (float)p.N), p.eps)) : 1.f;
  const float inv = OUT == OUT_E4M3 ? __frcp_rn(f) : f;
  auto value = [&](float a) { return OUT == OUT_E4M3 && NORM ? (a * rs) * inv : a * inv; };
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
      const int c = (i * T + t) * 8;
      if (c < N) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = value(v[8 * i + j]);
        out8<OUT>(p, m, c, y);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = i * T + t;
      if (c < N) out1<OUT>(p, m, c, value(v[i]));
    }
  }
}

// Rows longer than the register kernels hold: two passes over the row, the second mostly from L2.
// The first pass only reads (sum_out may be the residual's or x's own rows), the second writes.
template <typename X, int OUT, bool NORM>
__global__ void __launch_bounds__(1024) norm_long_kernel(const NormArgs p) {
  grid_dependency_wait();
  grid_launch_dependents();
  __shared__ uint32_t sm[64];
  const int64_t m = blockIdx.x;
  const X *x = static_cast<const X *>(p.x) + m * p.ldx;
  const X *r = p.residual ? static_cast<const X *>(p.residual) + m * p.ldr : nullptr;
  X *so = p.sum_out ? static_cast<X *>(p.sum_out) + m * p.lds : nullptr;
  float sumsq = 0.f;
  uint32_t amax = 0u;
#pragma unroll 4
  for (int64_t c = threadIdx.x; c < p.N; c += 1024) {
    float s = to_f32(x[c]);
    if (r) s = __fadd_rn(s, to_f32(r[c]));
    if constexpr (NORM) {
      sumsq = fmaf(s, s, sumsq);
      s *= weight_at(p, c);
    }
    if constexpr (OUT == OUT_E4M3) amax = max(amax, __float_as_uint(s) & 0x7FFFFFFFu);
  }
  row_reduce<1024>(sumsq, amax, sm);
  const float f = finish_row<OUT, NORM>(p, m, sumsq, amax, threadIdx.x == 0);
  const float rs = OUT == OUT_E4M3 && NORM ? __frsqrt_rn(__fadd_rn(__fdiv_rn(sumsq, (float)p.N), p.eps)) : 1.f;
  const float inv = OUT == OUT_E4M3 ? __frcp_rn(f) : f;
#pragma unroll 4
  for (int64_t c = threadIdx.x; c < p.N; c += 1024) {
    float s = to_f32(x[c]);
    if (r) s = __fadd_rn(s, to_f32(r[c]));
    if (so) store1(so + c, s);
    if constexpr (NORM) s *= weight_at(p, c);
    out1<OUT>(p, m, c, OUT == OUT_E4M3 && NORM ? (s * rs) * inv : s * inv);
  }
}

// ---- gradient ------------------------------------------------------------------------------------

// Blocks of kRows rows at a time (kRows = 8 for 32-thread rows); row group b, b + gridDim.x, ...
// part: gridDim.x rows of N f32, this block's column sums (null: no dweight).
template <typename X, bool VEC, int T, int E>
__global__ void __launch_bounds__(T == 32 ? 256 : T) norm_bwd_kernel(const NormBwdArgs p, float *__restrict__ part) {
  grid_dependency_wait();
  grid_launch_dependents();
  constexpr int kRows = T == 32 ? 8 : 1;
  __shared__ uint32_t sm[2][64];
  __shared__ float comb[kRows > 1 ? kRows * T * E : 1];
  const int t = T == 32 ? (threadIdx.x & 31) : threadIdx.x, sub = T == 32 ? threadIdx.x >> 5 : 0;
  const int N = (int)p.N;
  auto col = [&](int e) { return VEC ? ((e / 8) * T + t) * 8 + e % 8 : e * T + t; };
  NormArgs wa{};
  wa.weight = p.weight;
  wa.w_bf16 = p.w_bf16;
  float w[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    w[e] = col(e) < N ? weight_at(wa, col(e)) : 0.f;
    acc[e] = 0.f;
  }
  int par = 0;
  for (int64_t m = (int64_t)blockIdx.x * kRows + sub; m < p.M; m += (int64_t)gridDim.x * kRows, par ^= 1) {
    const X *dy = static_cast<const X *>(p.dy) + m * p.lddy;
    const X *s = static_cast<const X *>(p.s) + m * p.lds;
    const X *ds = p.ds ? static_cast<const X *>(p.ds) + m * p.ldds : nullptr;
    X *dx = static_cast<X *>(p.dx) + m * p.lddx;
    const float rstd = __ldg(p.rstd + m);
    float g[E], h[E], d[E];
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < E / 8; ++i) {
        float (&gg)[8] = *reinterpret_cast<float (*)[8]>(&g[8 * i]);
        float (&hh)[8] = *reinterpret_cast<float (*)[8]>(&h[8 * i]);
        float (&dd)[8] = *reinterpret_cast<float (*)[8]>(&d[8 * i]);
        const int c = (i * T + t) * 8;
        if (c < N) {
          load8(dy + c, gg);
          load8(s + c, hh);
          if (ds) load8(ds + c, dd);
        }
        if (c >= N || !ds) {
#pragma unroll
          for (int j = 0; j < 8; ++j) dd[j] = 0.f;
        }
        if (c >= N) {
#pragma unroll
          for (int j = 0; j < 8; ++j) gg[j] = hh[j] = 0.f;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = e * T + t;
        g[e] = c < N ? to_f32(dy[c]) : 0.f;
        h[e] = c < N ? to_f32(s[c]) : 0.f;
        d[e] = c < N && ds ? to_f32(ds[c]) : 0.f;
      }
    }
    float dot = 0.f;
    uint32_t none = 0u;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      h[e] *= rstd;
      acc[e] = fmaf(g[e], h[e], acc[e]);
      g[e] *= w[e];
      dot = fmaf(g[e], h[e], dot);
    }
    row_reduce<T>(dot, none, sm[par]);  // two buffers: the next row's may be written while this one is read
    const float c1 = __fdiv_rn(dot, (float)N);
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] = fmaf(rstd, fmaf(-h[e], c1, g[e]), d[e]);
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < E / 8; ++i) {
        const int c = (i * T + t) * 8;
        if (c < N) store8(dx + c, *reinterpret_cast<const float (*)[8]>(&g[8 * i]));
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * T + t < N) store1(dx + e * T + t, g[e]);
    }
  }
  if (!part) return;
  float *row = part + (int64_t)blockIdx.x * N;
  if constexpr (kRows > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) comb[(sub * E + e) * T + t] = acc[e];
    __syncthreads();
    if (sub == 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float v = acc[e];
#pragma unroll
        for (int r = 1; r < kRows; ++r) v += comb[(r * E + e) * T + t];
        if (col(e) < N) row[col(e)] = v;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (col(e) < N) row[col(e)] = acc[e];
  }
}

// Rows longer than the register kernel holds: two passes; the column sums are kept in this block's
// row of `part`, each element read and written by one thread.
template <typename X>
__global__ void __launch_bounds__(1024) norm_bwd_long_kernel(const NormBwdArgs p, float *__restrict__ part) {
  grid_dependency_wait();
  grid_launch_dependents();
  __shared__ uint32_t sm[2][64];
  NormArgs wa{};
  wa.weight = p.weight;
  wa.w_bf16 = p.w_bf16;
  float *row = part ? part + (int64_t)blockIdx.x * p.N : nullptr;
  int par = 0;
  bool first = true;
  for (int64_t m = blockIdx.x; m < p.M; m += gridDim.x, par ^= 1, first = false) {
    const X *dy = static_cast<const X *>(p.dy) + m * p.lddy;
    const X *s = static_cast<const X *>(p.s) + m * p.lds;
    const X *ds = p.ds ? static_cast<const X *>(p.ds) + m * p.ldds : nullptr;
    X *dx = static_cast<X *>(p.dx) + m * p.lddx;
    const float rstd = __ldg(p.rstd + m);
    float dot = 0.f;
    uint32_t none = 0u;
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < p.N; c += 1024)
      dot = fmaf(to_f32(dy[c]) * weight_at(wa, c), to_f32(s[c]) * rstd, dot);
    row_reduce<1024>(dot, none, sm[par]);
    const float c1 = __fdiv_rn(dot, (float)p.N);
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < p.N; c += 1024) {
      const float y = to_f32(dy[c]), h = to_f32(s[c]) * rstd, d = ds ? to_f32(ds[c]) : 0.f;
      if (row) row[c] = first ? y * h : fmaf(y, h, row[c]);
      store1(dx + c, fmaf(rstd, fmaf(-h, c1, y * weight_at(wa, c)), d));
    }
  }
}

// out[c] = sum over r = 0 .. rows - 1, in a fixed order, of part[r * N + c]: 32 columns a block, 32
// threads share a column's rows.
__global__ void __launch_bounds__(1024) column_sum_kernel(const float *__restrict__ part, int rows, int64_t N,
                                                          float *__restrict__ out) {
  grid_dependency_wait();
  grid_launch_dependents();
  __shared__ float sm[32][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (c < N) {
#pragma unroll 4
    for (int r = threadIdx.y; r < rows; r += 32) v += part[(int64_t)r * N + c];
  }
  sm[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = sm[threadIdx.x][threadIdx.y];  // thread (x, y): partial x of column y
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  const int64_t cc = (int64_t)blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && cc < N) out[cc] = v;
}

bool at16(const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

template <typename X, int OUT, bool VEC, bool NORM>
cudaError_t launch_norm_rows(const NormArgs &p, cudaStream_t st) {
  const unsigned g = (unsigned)p.M;
  if (p.N <= 256) return launch_dependent(norm_row_kernel<X, OUT, VEC, 32, 8, NORM>, dim3((unsigned)((p.M + 7) / 8)), dim3(256), st, p);
  if (p.N <= 1024) return launch_dependent(norm_row_kernel<X, OUT, VEC, 128, 8, NORM>, dim3(g), dim3(128), st, p);
  if (p.N <= 2048) return launch_dependent(norm_row_kernel<X, OUT, VEC, 256, 8, NORM>, dim3(g), dim3(256), st, p);
  if (p.N <= 4096) return launch_dependent(norm_row_kernel<X, OUT, VEC, 256, 16, NORM>, dim3(g), dim3(256), st, p);
  if (p.N <= 8192) return launch_dependent(norm_row_kernel<X, OUT, VEC, 512, 16, NORM>, dim3(g), dim3(512), st, p);
  if (p.N <= 16384) return launch_dependent(norm_row_kernel<X, OUT, VEC, 1024, 16, NORM>, dim3(g), dim3(1024), st, p);
  return launch_dependent(norm_long_kernel<X, OUT, NORM>, dim3(g), dim3(1024), st, p);
}

template <typename X, int OUT, bool NORM>
cudaError_t launch_norm_vec(const NormArgs &p, cudaStream_t st) {
  constexpr int e = sizeof(X);
  constexpr int eo = OUT == OUT_F32 ? 4 : (OUT == OUT_BF16 ? 2 : 1);
  const bool vec = p.N % 8 == 0 && at16(p.x) && at16(p.residual) && at16(p.sum_out) && at16(p.weight) && at16(p.out) &&
                   p.ldx * e % 16 == 0 && p.ldr * e % 16 == 0 && p.lds * e % 16 == 0 &&
                   p.ldo * eo % (eo == 1 ? 8 : 16) == 0;
  return vec ? launch_norm_rows<X, OUT, true, NORM>(p, st) : launch_norm_rows<X, OUT, false, NORM>(p, st);
}

template <typename X, bool VEC>
cudaError_t launch_bwd_rows(const NormBwdArgs &p, float *part, int grid, cudaStream_t st) {
  if (p.N <= 256) return launch_dependent(norm_bwd_kernel<X, VEC, 32, 8>, dim3(grid), dim3(256), st, p, part);
  if (p.N <= 1024) return launch_dependent(norm_bwd_kernel<X, VEC, 128, 8>, dim3(grid), dim3(128), st, p, part);
  if (p.N <= 2048) return launch_dependent(norm_bwd_kernel<X, VEC, 256, 8>, dim3(grid), dim3(256), st, p, part);
  if (p.N <= 4096) return launch_dependent(norm_bwd_kernel<X, VEC, 256, 16>, dim3(grid), dim3(256), st, p, part);
  if (p.N <= 8192) return launch_dependent(norm_bwd_kernel<X, VEC, 512, 16>, dim3(grid), dim3(512), st, p, part);
  if (p.N <= 16384) return launch_dependent(norm_bwd_kernel<X, VEC, 1024, 16>, dim3(grid), dim3(1024), st, p, part);
  return launch_dependent(norm_bwd_long_kernel<X>, dim3(grid), dim3(1024), st, p, part);
}

}  // namespace

cudaError_t launch_rms_norm(const NormArgs &p, bool norm, cudaStream_t st) {
  if (norm) {
    if (p.x_bf16)
      return p.out_kind == OUT_F32    ? launch_norm_vec<__nv_bfloat16, OUT_F32, true>(p, st)
             : p.out_kind == OUT_BF16 ? launch_norm_vec<__nv_bfloat16, OUT_BF16, true>(p, st)
                                      : launch_norm_vec<__nv_bfloat16, OUT_E4M3, true>(p, st);
    return p.out_kind == OUT_F32    ? launch_norm_vec<float, OUT_F32, true>(p, st)
           : p.out_kind == OUT_BF16 ? launch_norm_vec<float, OUT_BF16, true>(p, st)
                                    : launch_norm_vec<float, OUT_E4M3, true>(p, st);
  }
  return p.x_bf16 ? launch_norm_vec<__nv_bfloat16, OUT_E4M3, false>(p, st) : launch_norm_vec<float, OUT_E4M3, false>(p, st);
}

int rms_norm_bwd_parts(int64_t M, int64_t N) {
  // Blocks that fill the SMs (2048 threads each) once; no more than there are row groups.
  const int64_t threads = N <= 256 ? 256 : (N <= 1024 ? 128 : (N <= 4096 ? 256 : (N <= 8192 ? 512 : 1024)));
  const int64_t rows = N <= 256 ? 8 : 1;
  const int64_t groups = (M + rows - 1) / rows, most = 148 * (1024 / threads);
  return (int)(groups < most ? groups : most);
}

cudaError_t launch_rms_norm_bwd(const NormBwdArgs &p, float *part, int grid, cudaStream_t st) {
  const int e = p.x_bf16 ? 2 : 4;
  const bool vec = p.N % 8 == 0 && at16(p.dy) && at16(p.s) && at16(p.ds) && at16(p.dx) && p.lddy * e % 16 == 0 &&
                   p.lds * e % 16 == 0 && p.ldds * e % 16 == 0 && p.lddx * e % 16 == 0;
  if (p.x_bf16)
    return vec ? launch_bwd_rows<__nv_bfloat16, true>(p, part, grid, st) : launch_bwd_rows<__nv_bfloat16, false>(p, part, grid, st);
  return vec ? launch_bwd_rows<float, true>(p, part, grid, st) : launch_bwd_rows<float, false>(p, part, grid, st);
}

cudaError_t launch_column_sum(const float *part, int rows, int64_t N, float *out, cudaStream_t st) {
  return launch_dependent(column_sum_kernel, dim3((unsigned)((N + 31) / 32)), dim3(32, 32), st, part, rows, N, out);
}

}  // namespace tf
