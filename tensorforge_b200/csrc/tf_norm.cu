// tf_norm.cu -- root-mean-square norm with the residual's addition (f32, bf16 or 8-bit output with
// a scale a row), its gradient, and the row quantizer the 8-bit linear layer's operands come from.
//
// Forward, row by row, in f32:
//   s = x + residual;  rstd = (mean(s^2) + eps)^-1/2;  y = (s w) rstd
//   8-bit output: scale = max(max|y| / 448, 2^-126), q = e4m3(y (1 / scale))
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
// 16384 x 8192 bf16 with residual to 8 bits 143 us, 6.6 TB/s; the gradient of 16384 x 4096 bf16 with ds
// 88 us, 6.1 TB/s; 4097 x 1111 f32, single elements, 7 us, 5.3 TB/s; 16 x 4096, a launch, 2.4 us; the
// quantizer of 16384 x 16384 bf16 134 us, 6.0 TB/s, of 2048 x 28672 (two passes) 63, 2.8, of
// 16384 x 1111 31.5, 1.7.  (Replayed from graphs, or calls in a row where they last longer than the host
// takes to issue one.)
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>

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

// Sum of `a` and, with MAX, maximum of `b` over the T threads of one row (T a power of two: below
// 32 a part of a warp, above it the whole block).  `sm`: 64 words of shared memory for T > 32, not
// written again before the next reduction's barrier but one.  Every thread of the row gets the
// same bits.
template <int T, bool MAX>
__device__ __forceinline__ void row_reduce(float &a, uint32_t &b, uint32_t *sm) {
  constexpr int W = T < 32 ? T : 32, N = T / 32;
#pragma unroll
  for (int o = W / 2; o; o >>= 1) {
    a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
    if constexpr (MAX) b = max(b, __shfl_xor_sync(0xFFFFFFFFu, b, o));
  }
  if constexpr (T > 32) {
    const int w = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
      sm[w] = __float_as_uint(a);
      if constexpr (MAX) sm[32 + w] = b;
    }
    __syncthreads();
    // The same sum in every thread: four or eight warps' values by 16-byte reads that a warp shares,
    // else a read a lane and shuffles.
    if constexpr (N == 4 || N == 8) {
      float s[N];
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 v = *reinterpret_cast<const float4 *>(sm + i);
        s[i] = v.x; s[i + 1] = v.y; s[i + 2] = v.z; s[i + 3] = v.w;
      }
#pragma unroll
      for (int o = N / 2; o; o >>= 1)
#pragma unroll
        for (int i = 0; i < o; ++i) s[i] += s[i + o];
      a = s[0];
      if constexpr (MAX) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          const uint4 v = *reinterpret_cast<const uint4 *>(sm + 32 + i);
          b = max(max(max(v.x, v.y), max(v.z, v.w)), b);
        }
      }
    } else {
      const int i = threadIdx.x & (N - 1);
      a = __uint_as_float(sm[i]);
      if constexpr (MAX) b = sm[32 + i];
#pragma unroll
      for (int o = N / 2; o; o >>= 1) {
        a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
        if constexpr (MAX) b = max(b, __shfl_xor_sync(0xFFFFFFFFu, b, o));
      }
    }
  }
}

// The sum over a row that a cluster of CL blocks of T threads shares.  `sm`: CL T / 32 words of this
// block, written by all of them; not written again before the next reduction's barrier but one.
template <int T, int CL>
__device__ __forceinline__ float cluster_sum(float a, float *sm) {
  constexpr int W = T / 32, N = CL * W;
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane < CL) st_cluster_f32(map_to_cta(smem_u32(sm + cluster_ctarank() * W + w), lane), a);
  cluster_sync();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < (N + 31) / 32; ++i) s += N % 32 == 0 || lane + 32 * i < N ? sm[lane + 32 * i] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  return s;
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

// Writes the row's rstd and scale (one thread).  What out holds of t = s weight: t rstd, for 8 bits
// (t rstd) (1 / scale) -- in two steps, since rstd / scale overflows for a row of zeros, and by the
// rounded reciprocal: one value in ten thousand, which lies within 2^-23 of the middle between two
// e4m3 numbers, goes to the other one than its quotient would.  Dividing every value makes the norm of
// 16384 x 8192 bf16 165 us instead of 142, the quantizer of 16384 x 16384 191 instead of 134.
template <int OUT, bool NORM>
struct RowFactors {
  float rstd = 1.f, inv = 1.f;

  __device__ __forceinline__ RowFactors(const NormArgs &p, int64_t m, float sumsq, uint32_t amax_bits, bool writer) {
    if constexpr (NORM) {
      rstd = rsqrtf(fmaf(sumsq, p.inv_n, p.eps));
      if (writer && p.rstd) p.rstd[m] = rstd;
    }
    if constexpr (OUT == OUT_E4M3) {
      float scale = __fdiv_rn(__uint_as_float(amax_bits) * rstd, kE4m3Max);
      scale = scale < kTinyScale ? kTinyScale : scale;  // keeps a NaN
      // An infinite value: the whole row is NaN, where its other values would be zeros.
      if (isinf(scale)) scale = __int_as_float(0x7FFFFFFF);
      if (writer) p.scale[m] = scale;
      inv = __frcp_rn(scale);
    }
  }
  __device__ __forceinline__ float operator()(float t) const {
    if constexpr (NORM) t *= rstd;
    if constexpr (OUT == OUT_E4M3) t *= inv;
    return t;
  }
};

// One row on T threads, E elements a thread in registers; up to 32 threads a block of 256 holds
// several rows.  VEC: groups of eight consecutive elements (all rows on 16-byte boundaries, N a
// multiple of 8); else single elements, T apart.  NORM false: the quantizer (y = x).
template <typename X, int OUT, bool VEC, int T, int E, bool NORM>
__global__ void __launch_bounds__(T <= 32 ? 256 : T) norm_row_kernel(const NormArgs p) {
  grid_dependency_wait();
  grid_launch_dependents();
  constexpr int kRows = T <= 32 ? 256 / T : 1;
  __shared__ __align__(16) uint32_t sm[64];
  const int t = threadIdx.x & (T - 1);
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / T;
  const bool live = row < p.M;  // a part of a warp without a row goes along with no columns
  const int64_t m = live ? row : 0;
  const int N = live ? (int)p.N : 0;
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
  row_reduce<T, OUT == OUT_E4M3>(sumsq, amax, sm);
  const RowFactors<OUT, NORM> f(p, m, sumsq, amax, t == 0 && live);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
      const int c = (i * T + t) * 8;
      if (c < N) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = f(v[8 * i + j]);
        out8<OUT>(p, m, c, y);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = i * T + t;
      if (c < N) out1<OUT>(p, m, c, f(v[i]));
    }
  }
}

// Rows longer than the register kernels hold (16384): two passes over the row, the second mostly from L2.
// The first pass only reads (sum_out may be the residual's or x's own rows), the second writes.
template <typename X, int OUT, bool NORM>
__global__ void __launch_bounds__(1024) norm_long_kernel(const NormArgs p) {
  grid_dependency_wait();
  grid_launch_dependents();
  __shared__ __align__(16) uint32_t sm[64];
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
  row_reduce<1024, OUT == OUT_E4M3>(sumsq, amax, sm);
  const RowFactors<OUT, NORM> f(p, m, sumsq, amax, threadIdx.x == 0);
#pragma unroll 4
  for (int64_t c = threadIdx.x; c < p.N; c += 1024) {
    float s = to_f32(x[c]);
    if (r) s = __fadd_rn(s, to_f32(r[c]));
    if (so) store1(so + c, s);
    if constexpr (NORM) s *= weight_at(p, c);
    out1<OUT>(p, m, c, f(s));
  }
}

// ---- gradient ------------------------------------------------------------------------------------

// E elements of a row as they are loaded: 16-byte pieces (VEC), or single elements.
template <typename X, bool VEC, int E>
struct RawRow {
  using Piece = std::conditional_t<VEC, uint4, X>;
  static constexpr int kPer = VEC ? 16 / (int)sizeof(X) : 1, kPieces = E / kPer;
  Piece v[kPieces];

  // Columns of element e of thread t: groups of eight with VEC, else single ones T apart.
  template <int T>
  __device__ __forceinline__ static int col(int e, int t) { return VEC ? ((e / 8) * T + t) * 8 + e % 8 : e * T + t; }
  // Columns below n (a multiple of 8 with VEC); the others are zeros.
  template <int T>
  __device__ __forceinline__ void load(const X *row, int t, int n) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int c = col<T>(i * kPer, t);
      if (c < n) v[i] = *reinterpret_cast<const Piece *>(row + c);
      else v[i] = Piece{};
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (!VEC) {
      return to_f32(v[e]);
    } else {
      const uint4 &u = v[e / kPer];
      if constexpr (sizeof(X) == 4) {
        const uint32_t w = e % 4 == 0 ? u.x : e % 4 == 1 ? u.y : e % 4 == 2 ? u.z : u.w;
        return __uint_as_float(w);
      } else {
        const uint32_t w = e % 8 / 2 == 0 ? u.x : e % 8 / 2 == 1 ? u.y : e % 8 / 2 == 2 ? u.z : u.w;
        return __uint_as_float(e % 2 ? w & 0xFFFF0000u : w << 16);
      }
    }
  }
};

// Threads of a block and, up to 32 threads a row, its rows.
template <int T>
constexpr int kBwdBlock = T <= 32 ? 256 : T;

// Row groups b, b + gridDim.x / CL, ... of block (or of cluster of CL blocks, each with T E columns of
// the row) b.  AHEAD: the next rows' loads are under way while a row is reduced and written.  part:
// gridDim.x / CL rows of N f32, this block's column sums (null: no dweight).
template <typename X, bool VEC, int T, int E, int CL, bool AHEAD>
__global__ void __launch_bounds__(kBwdBlock<T>, T == 512 ? 2 : 1) norm_bwd_kernel(const NormBwdArgs p, float *part) {
  grid_dependency_wait();
  grid_launch_dependents();
  using Raw = RawRow<X, VEC, E>;
  constexpr int kRows = kBwdBlock<T> / T;
  static_assert(CL == 1 || (kRows == 1 && T >= 64), "a cluster has one row at a time");
  __shared__ __align__(16) uint32_t sm[2][CL * T / 32 > 64 ? CL * T / 32 : 64];
  __shared__ float comb[kRows > 1 ? kRows * T * E : 1];
  const int t = threadIdx.x & (T - 1), sub = threadIdx.x / T;
  if constexpr (CL > 1) cluster_sync();  // every block has started before another writes its memory
  // This block's columns: c0 .. c0 + width - 1.
  const int64_t c0 = CL > 1 ? (int64_t)cluster_ctarank() * (T * E) : 0;
  const int width = CL > 1 ? (int)(p.N - c0 < 0 ? 0 : p.N - c0 < T * E ? p.N - c0 : T * E) : (int)p.N;
  const int block = (int)blockIdx.x / CL, blocks = (int)gridDim.x / CL;
  NormArgs wa{};
  wa.weight = p.weight;
  wa.w_bf16 = p.w_bf16;
  float w[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = Raw::template col<T>(e, t);
    w[e] = c < width ? weight_at(wa, c0 + c) : 0.f;
    acc[e] = 0.f;
  }
  struct Rows {
    Raw y, s, d;
    float rstd;
  };
  Rows next;
  auto fetch = [&](int64_t m0) {
    const bool live = m0 + sub < p.M;  // a part of a warp without a row goes along with no columns
    const int64_t m = live ? m0 + sub : 0;
    const int n = live ? width : 0;
    next.y.template load<T>(static_cast<const X *>(p.dy) + m * p.lddy + c0, t, n);
    next.s.template load<T>(static_cast<const X *>(p.s) + m * p.lds + c0, t, n);
    if (p.ds) next.d.template load<T>(static_cast<const X *>(p.ds) + m * p.ldds + c0, t, n);
    next.rstd = p.rstd[m];
  };
  const int64_t step = (int64_t)blocks * kRows;
  int64_t m0 = (int64_t)block * kRows;
  if (AHEAD && m0 < p.M) fetch(m0);
  int par = 0;
  for (; m0 < p.M; m0 += step, par ^= 1) {
    // The row is kept as it was loaded, and unpacked before and after the reduction: fewer registers.
    if constexpr (!AHEAD) fetch(m0);
    const Rows row = next;
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float y = row.y.get(e), h = row.s.get(e) * row.rstd;
      acc[e] = fmaf(y, h, acc[e]);
      dot = fmaf(y * w[e], h, dot);
    }
    if (AHEAD && m0 + step < p.M) fetch(m0 + step);
    if constexpr (CL > 1) {
      dot = cluster_sum<T, CL>(dot, reinterpret_cast<float *>(sm[par]));
    } else {
      uint32_t none = 0u;
      row_reduce<T, false>(dot, none, sm[par]);
    }
    const float c1 = dot * p.inv_n;
    float g[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      g[e] = fmaf(row.rstd, fmaf(-row.s.get(e) * row.rstd, c1, row.y.get(e) * w[e]), p.ds ? row.d.get(e) : 0.f);
    const int n = m0 + sub < p.M ? width : 0;
    X *dx = static_cast<X *>(p.dx) + (m0 + sub) * p.lddx + c0;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < E / 8; ++i) {
        const int c = (i * T + t) * 8;
        if (c < n) store8(dx + c, *reinterpret_cast<const float (*)[8]>(&g[8 * i]));
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * T + t < n) store1(dx + e * T + t, g[e]);
    }
  }
  if (!part) return;
  float *row = part + (int64_t)block * p.N + c0;
  if constexpr (kRows > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) comb[(sub * E + e) * T + t] = acc[e];
    __syncthreads();
    // Element e of thread t, summed over the block's rows in order, by thread e T + t.
    for (int i = threadIdx.x; i < E * T; i += kBwdBlock<T>) {
      float v = 0.f;
#pragma unroll 4
      for (int q = 0; q < kRows; ++q) v += comb[q * E * T + i];
      const int c = Raw::template col<T>(i / T, i % T);
      if (c < width) row[c] = v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = Raw::template col<T>(e, t);
      if (c < width) row[c] = acc[e];
    }
  }
}

// Wider rows than eight blocks hold: two passes over a row, the second mostly from L2, the column sums
// in this block's row of `part`, each element read and written by one thread.  VEC: eight elements a
// thread and step; else one.
template <typename X, bool VEC>
__global__ void __launch_bounds__(512, 2) norm_bwd_wide_kernel(const NormBwdArgs p, float *part) {
  grid_dependency_wait();
  grid_launch_dependents();
  using Raw = RawRow<X, VEC, VEC ? 8 : 1>;
  constexpr int V = VEC ? 8 : 1;
  __shared__ __align__(16) uint32_t sm[2][64];
  NormArgs wa{};
  wa.weight = p.weight;
  wa.w_bf16 = p.w_bf16;
  float *acc = part ? part + (int64_t)blockIdx.x * p.N : nullptr;
  bool first = true;
  // Groups of V columns; a thread's own are 512 V apart.
  auto weights = [&](int64_t c, float (&w)[V]) {
    if constexpr (VEC) weight8(wa, c, w);
    else w[0] = weight_at(wa, c);
  };
  int par = 0;
  for (int64_t m = blockIdx.x; m < p.M; m += gridDim.x, par ^= 1, first = false) {
    const X *dy = static_cast<const X *>(p.dy) + m * p.lddy;
    const X *s = static_cast<const X *>(p.s) + m * p.lds;
    const X *ds = p.ds ? static_cast<const X *>(p.ds) + m * p.ldds : nullptr;
    X *dx = static_cast<X *>(p.dx) + m * p.lddx;
    const float rstd = p.rstd[m];
    float dot = 0.f;
    uint32_t none = 0u;
#pragma unroll 2
    for (int64_t c = (int64_t)threadIdx.x * V; c < p.N; c += 512 * V) {
      Raw y, h;
      float w[V];
      y.template load<1>(dy + c, 0, V);
      h.template load<1>(s + c, 0, V);
      weights(c, w);
#pragma unroll
      for (int j = 0; j < V; ++j) dot = fmaf(y.get(j) * w[j], h.get(j) * rstd, dot);
    }
    row_reduce<512, false>(dot, none, sm[par]);
    const float c1 = dot * p.inv_n;
#pragma unroll 2
    for (int64_t c = (int64_t)threadIdx.x * V; c < p.N; c += 512 * V) {
      Raw y, h, d;
      float w[V], g[V];
      y.template load<1>(dy + c, 0, V);
      h.template load<1>(s + c, 0, V);
      if (ds) d.template load<1>(ds + c, 0, V);
      weights(c, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float a = y.get(j), b = h.get(j) * rstd;
        if (acc) acc[c + j] = first ? a * b : fmaf(a, b, acc[c + j]);
        g[j] = fmaf(rstd, fmaf(-b, c1, a * w[j]), ds ? d.get(j) : 0.f);
      }
      if constexpr (VEC) store8(dx + c, g);
      else store1(dx + c, g[0]);
    }
  }
}

// out[c] = sum over r = 0 .. rows - 1, in a fixed order, of part[r * N + c]: 32 columns a block, 32
// threads share a column's rows.  256 x 16384 7 us, mostly from L2; 63 x 1000 under 4, a launch.
__global__ void __launch_bounds__(1024) column_sum_kernel(const float *part, int rows, int64_t N, float *out) {
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

// Rows that one an SM takes: then a row's own time counts, and more threads on it (16 x 4096 bf16 with
// residual to 8 bits 2.4 us on 256 x 16, 3.1 on 128 x 32).
constexpr int64_t kFewRows = 148;

bool at16(const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

// The first of the row kernels whose T threads x E elements hold N columns.  In 16-byte pieces many
// elements on few threads, two steps a power of two: threads without columns cost most, and blocks that
// end at a barrier soonest (50 331 648 elements bf16 to bf16 in rows of 640 5.3 TB/s on 32 x 24, 2.5 on
// 128 x 8; of 1024 5.7 on 32 x 32, 3.8 on 128 x 8; of 4160 5.1 on 256 x 24, 3.8 on 512 x 16).  f32
// rows of 1024 with residual 6.8 on 128 x 8, 6.4 on 32 x 32.  Single elements: 2 to 5 TB/s in bf16,
// the more threads the better above a warp (rows of 1660 4.1 on 256 x 8, 2.7 on 128 x 16; of 4095 3.8 on
// 512 x 8, 2.7 on 256 x 16; of 300 2.2 on 32 x 16, 1.2 on 64 x 8).  Aligned pairs of bf16 for such rows,
// singles at their ends, measured slower (rows of 1111 1.7 against 3.0).
template <typename X, int OUT, bool VEC, bool NORM, int T, int E, int... MORE>
cudaError_t launch_norm_rows(const NormArgs &p, cudaStream_t st) {
  constexpr int kRows = T <= 32 ? 256 / T : 1;
  if (p.N <= T * E)
    return launch_dependent(norm_row_kernel<X, OUT, VEC, T, E, NORM>, dim3((unsigned)((p.M + kRows - 1) / kRows)),
                            dim3(kRows * T), st, 0, p);
  if constexpr (sizeof...(MORE) > 0) return launch_norm_rows<X, OUT, VEC, NORM, MORE...>(p, st);
  else return launch_dependent(norm_long_kernel<X, OUT, NORM>, dim3((unsigned)p.M), dim3(1024), st, 0, p);
}

template <typename X, int OUT, bool NORM>
cudaError_t launch_norm_vec(const NormArgs &p, cudaStream_t st) {
  constexpr int e = sizeof(X);
  constexpr int eo = OUT == OUT_F32 ? 4 : (OUT == OUT_BF16 ? 2 : 1);
  const bool vec = p.N % 8 == 0 && at16(p.x) && at16(p.residual) && at16(p.sum_out) && at16(p.weight) && at16(p.out) &&
                   p.ldx * e % 16 == 0 && p.ldr * e % 16 == 0 && p.lds * e % 16 == 0 &&
                   p.ldo * eo % (eo == 1 ? 8 : 16) == 0;
  if (vec && p.M <= kFewRows)
    return launch_norm_rows<X, OUT, true, NORM, 8, 8, 16, 8, 32, 8, 128, 8, 256, 8, 256, 16, 512, 16, 512, 32>(p, st);
  if (!vec)
    return launch_norm_rows<X, OUT, false, NORM, 32, 4, 32, 8, 32, 16, 128, 8, 256, 8, 256, 12, 512, 8, 512, 12, 1024, 8, 1024, 16>(
        p, st);
  if constexpr (sizeof(X) == 4)
    return launch_norm_rows<X, OUT, true, NORM, 8, 8, 16, 8, 32, 8, 32, 16, 32, 24, 128, 8, 128, 16, 128, 24, 256, 16, 256, 24, 512, 16,
                            512, 32>(p, st);
  else
    return launch_norm_rows<X, OUT, true, NORM, 8, 8, 16, 8, 32, 8, 32, 16, 32, 24, 32, 32, 32, 48, 128, 16, 128, 24, 128, 32, 256, 24,
                            256, 32, 512, 24, 512, 32>(p, st);
}

// The gradient kernel of a call.  As forward, threads without columns cost most, and a row's next loads
// are worth more than more rows: 41 943 040 elements in rows of 1216 bf16 67 us on 64 x 24 (94 on
// 256 x 8), of 5120 f32 with ds 106 on 256 x 24 (142 on 1024 x 8), of 4096 bf16 52 on 512 x 8 (70 on
// 256 x 16).  Rows above 8192 columns are shared by clusters: 50 331 648 elements in rows of 12288 f32
// with ds 5.0 TB/s on two blocks of 256 x 24 (3.9 on four of 512 x 8), of 16384 4.7 on four of
// 512 x 8 (3.9 on four of 256 x 16).
struct BwdKernel {
  void (*kern)(const NormBwdArgs, float *);
  int threads, rows;  // of a block
  int cluster;
  int id;  // a number of its own, below 160
};
// Whether the next rows' loads start before a row is reduced: not where the registers for two rows would
// leave too few warps.
template <typename X, bool VEC, int T>
constexpr bool bwd_ahead() {
  return T < 512 || (T == 512 && VEC && sizeof(X) == 2) || (T == 1024 && VEC && sizeof(X) == 2);
}
// The first of the kernels whose T threads x E elements x CL blocks hold N columns.
template <typename X, bool VEC, int T, int E, int CL, int... MORE>
BwdKernel first_bwd(int64_t N, int id) {
  if (N <= (int64_t)T * E * CL)
    return {norm_bwd_kernel<X, VEC, T, E, CL, bwd_ahead<X, VEC, T>()>, kBwdBlock<T>, kBwdBlock<T> / T, CL, id};
  if constexpr (sizeof...(MORE) > 0) return first_bwd<X, VEC, MORE...>(N, id + 1);
  else return {norm_bwd_wide_kernel<X, VEC>, 512, 1, 1, id + 1};
}
template <typename X, bool VEC>
BwdKernel pick_bwd(int64_t M, int64_t N, int id) {
  if (M <= kFewRows)
    return first_bwd<X, VEC, 32, 8, 1, 64, 8, 1, 128, 8, 1, 256, 8, 1, 512, 8, 1, 1024, 8, 1, 512, 8, 4, 512, 8, 8>(N, id + 20);
  if constexpr (!VEC)
    return first_bwd<X, VEC, 32, 8, 1, 32, 16, 1, 32, 24, 1, 128, 8, 1, 256, 8, 1, 512, 8, 1, 1024, 8, 1, 512, 8, 4, 512, 8, 8>(N, id);
  else if constexpr (sizeof(X) == 2)
    return first_bwd<X, VEC, 8, 8, 1, 16, 8, 1, 32, 8, 1, 32, 16, 1, 32, 24, 1, 64, 16, 1, 64, 24, 1, 128, 16, 1, 512, 8, 1, 1024, 8,
                     1, 256, 24, 2, 512, 8, 4, 256, 24, 4, 512, 8, 8>(N, id);
  else
    return first_bwd<X, VEC, 8, 8, 1, 16, 8, 1, 32, 8, 1, 32, 16, 1, 32, 24, 1, 128, 8, 1, 64, 24, 1, 256, 8, 1, 128, 24, 1, 512, 8, 1,
                     256, 24, 1, 1024, 8, 1, 256, 24, 2, 512, 8, 4, 256, 24, 4, 512, 8, 8>(N, id);
}

bool bwd_vec(const NormBwdArgs &p) {
  const int e = p.x_bf16 ? 2 : 4;
  return p.N % 8 == 0 && at16(p.weight) && at16(p.dy) && at16(p.s) && at16(p.ds) && at16(p.dx) && p.lddy * e % 16 == 0 &&
         p.lds * e % 16 == 0 && p.ldds * e % 16 == 0 && p.lddx * e % 16 == 0;
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

static BwdKernel pick_bwd(const NormBwdArgs &p) {
  const bool vec = bwd_vec(p);
  if (p.x_bf16) return vec ? pick_bwd<__nv_bfloat16, true>(p.M, p.N, 0) : pick_bwd<__nv_bfloat16, false>(p.M, p.N, 40);
  return vec ? pick_bwd<float, true>(p.M, p.N, 80) : pick_bwd<float, false>(p.M, p.N, 120);
}

static void cluster_attr(cudaLaunchAttribute &a, int cluster) {
  a.id = cudaLaunchAttributeClusterDimension;
  a.val.clusterDim.x = (unsigned)cluster;
  a.val.clusterDim.y = a.val.clusterDim.z = 1;
}

// Blocks (or clusters of them) that the SMs hold at once, no more than there are row groups.
int rms_norm_bwd_blocks(const NormBwdArgs &p) {
  const BwdKernel k = pick_bwd(p);
  static std::atomic<int> resident[160];
  int n = resident[k.id].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaError_t e;
    if (k.cluster > 1) {
      cudaLaunchAttribute attr[1];
      cluster_attr(attr[0], k.cluster);
      cudaLaunchConfig_t cfg = {dim3(148 * 8), dim3((unsigned)k.threads), 0, nullptr, attr, 1};
      e = cudaOccupancyMaxActiveClusters(&n, k.kern, &cfg);
    } else {
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k.kern, k.threads, 0);
      n *= 148;
    }
    if (e != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = 148 / k.cluster;
    }
    resident[k.id].store(n, std::memory_order_relaxed);
  }
  const int64_t groups = (p.M + k.rows - 1) / k.rows;
  return (int)(groups < n ? groups : n);
}

cudaError_t launch_rms_norm_bwd(const NormBwdArgs &p, float *part, int blocks, cudaStream_t st) {
  const BwdKernel k = pick_bwd(p);
  cudaLaunchAttribute attr[2];
  pdl_attr(attr[0]);
  cluster_attr(attr[1], k.cluster);
  cudaLaunchConfig_t cfg = {dim3((unsigned)(blocks * k.cluster)), dim3((unsigned)k.threads), 0, st, attr, k.cluster > 1 ? 2u : 1u};
  return cudaLaunchKernelEx(&cfg, k.kern, p, part);
}

cudaError_t launch_column_sum(const float *part, int rows, int64_t N, float *out, cudaStream_t st) {
  return launch_dependent(column_sum_kernel, dim3((unsigned)((N + 31) / 32)), dim3(32, 32), st, 0, part, rows, N, out);
}

}  // namespace tf
