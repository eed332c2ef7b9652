// tf_linear_slim.cu -- the linear layer on one CTA per tile with the operands exchanged: the
// weights' columns are the tensor core's 128 rows and BT = 16 .. 256 tokens its columns, so that a
// few tokens (BT 16: a decoding batch) cost no padding to 128.
//
//   out[m, n] = act((sum_k A[m, k] B[k, n]) a_scale[m] b_scale[n] + bias[n]) + residual[m, n]
//
// Operands are bf16 or e4m3, 128 bytes of k a stage, each K-major or (bf16) MN-major as it lies in
// memory, brought by TMA into a ring of 128-B-swizzled tiles; one thread issues the MMAs; the
// accumulator is BT columns of tensor memory.  With few tiles a cluster of S CTAs shares a tile,
// CTA z taking the z-th part of k.
//
// Epilogue: the tile is transposed in tensor memory (lane = column n), so it is first left in the
// ring's shared memory as f32, token by token; after a barrier (of the cluster, if it shares the
// tile) each CTA takes 1/S of the tile's values in groups of eight neighbouring columns of a token,
// adds the S CTAs' sums in order of z (the same bits every time) and finishes them: 16-byte
// accesses where the caller's rows allow; elsewhere the eight columns lie 16 apart, so that
// neighbouring threads' single accesses are neighbouring elements.
//
// Bound by HBM, where few tokens read the weights once, and by latency: 1 x 4096 -> 4096 bf16 8.8 us
// (33.5 MB of weights: 5.1 at the copy rate), 16 x 4096 -> 16384 e4m3 with silu 15.9 us (67 MB: 10.4),
// replayed from graphs; the host issues a call through Python in 13.5 us.
// Tokens as the tensor core's rows would pay for 128 of them.
//
// 256 threads: warp 0 TMA producer, warp 1 MMA issuer, then all eight warps the epilogue.  Every
// wait is bounded (tf_ptx.cuh), and none begins before the kernel that this launch follows is done.
#include <cuda.h>
#include <cuda_runtime.h>

#include "tf_epilogue.cuh"
#include "tf_internal.h"
#include "tf_ptx.cuh"

namespace tf {

namespace {

template <int BT, int STAGES>
struct SlimLayout {
  static constexpr int kThreads = 256;
  static constexpr int kWBytes = 128 * 128;  // 128 columns n x 128 B of k
  static constexpr int kTBytes = BT * 128;   // BT tokens x 128 B of k
  static constexpr int kStageBytes = kWBytes + kTBytes;
  static constexpr int kRing = STAGES * kStageBytes;
  static constexpr int kBarOff = kRing;
  // full[STAGES], empty[STAGES], accf; then the TMEM slot and the abort flag.
  static constexpr int kSmemBytes = 1024 + kBarOff + 8 * (2 * STAGES + 1) + 16;
  // Columns of one accumulator and, for sums in pieces, of as many as two CTAs an SM can have.
  static constexpr int kTmemCols = BT < 32 ? 32 : BT, kSumCols = 256, kAccs = kSumCols / BT;
  static_assert(BT * 512 <= kRing, "the partial sums reuse the ring");
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

__device__ __forceinline__ float residual_at(const LinearParams &p, int64_t i) {
  return p.res_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p.residual)[i])
                    : static_cast<const float *>(p.residual)[i];
}
// Eight f32 at a 16-byte boundary.
__device__ __forceinline__ void read8(const float *src, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(src)[0], b = reinterpret_cast<const float4 *>(src)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
// Column j of a thread's eight: n + j with VEC, else n + 16 j; below N by `live` = N - n.
template <bool VEC>
__device__ __forceinline__ void put8(void *base, bool bf16, int64_t i, int live, const float (&v)[8]) {
  if (bf16) {
    __nv_bfloat16 *o = static_cast<__nv_bfloat16 *>(base) + i;
    if constexpr (VEC) {
      *reinterpret_cast<uint4 *>(o) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                 pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (16 * j < live) o[16 * j] = __float2bfloat16_rn(v[j]);
    }
  } else {
    float *o = static_cast<float *>(base) + i;
    if constexpr (VEC) {
      reinterpret_cast<float4 *>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4 *>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (16 * j < live) o[16 * j] = v[j];
    }
  }
}
template <bool VEC>
__device__ __forceinline__ void get8(const float *src, int live, float (&v)[8]) {
  if constexpr (VEC) {
    read8(src, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 16 * j < live ? src[16 * j] : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void get_residual(const LinearParams &p, int64_t i, int live, float (&v)[8]) {
  if constexpr (VEC) {
    if (p.res_bf16) {
      const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(p.residual) + i);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    } else {
      read8(static_cast<const float *>(p.residual) + i, v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 16 * j < live ? residual_at(p, i + 16 * j) : 0.f;
  }
}

// Group g of the tile: token g / 16, eight columns; `part` holds its sums (token by token), in
// `splits` CTAs' shared memory at `sbase`.
template <bool VEC>
__device__ __forceinline__ void finish8(const LinearParams &p, int g, int m0, int n0, const float *part, uint32_t sbase,
                                        int splits) {
  const int at = VEC ? 8 * (g & 15) : g & 15, n = n0 + at, live = p.N - n;
  const int64_t m = m0 + (g >> 4);
  if (live <= 0) return;
  float res[8], v[8], c[8];
  if (p.residual) get_residual<VEC>(p, m * p.ldr + n, live, res);
  const int first = (g >> 4) * 128 + at;  // of the token-by-token sums
  if (splits == 1) {
    get8<VEC>(part + first, 1 << 30, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if (s < splits) {
        const uint32_t src = map_to_cta(sbase + 4 * first, s);
        if constexpr (VEC) {
          const float4 a = ld_cluster_f32x4(src), b = ld_cluster_f32x4(src + 16);
          v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
          v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] += ld_cluster_f32(src + 64 * j);
        }
      }
    }
  }
  if (p.a_scale) {
    const float sa = p.a_scale[m];
    get8<VEC>(p.b_scale + n, live, c);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * sa * c[j];
  }
  if (p.bias) {
    get8<VEC>(p.bias + n, live, c);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += c[j];
  }
  if (p.pre) put8<VEC>(p.pre, p.out_bf16, m * p.ldp + n, live, v);
  with_activation(p.act, [&](auto act) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = activate<decltype(act)::value>(v[j]);
  });
  if (p.residual) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += res[j];
  }
  put8<VEC>(p.out, p.out_bf16, m * p.ldo + n, live, v);
}

// F8: e4m3 operands (both K-major).  WMN / TMN: the weights' / tokens' tile is MN-major (bf16).
template <bool F8, bool WMN, bool TMN, int BT, int STAGES>
__global__ void __launch_bounds__(256)
    linear_slim_kernel(const __grid_constant__ CUtensorMap tmT, const __grid_constant__ CUtensorMap tmW,
                       const LinearParams p) {
  using L = SlimLayout<BT, STAGES>;
  static_assert(!F8 || (!WMN && !TMN), "8-bit operands are K-major");
  static_assert(!TMN || BT % 64 == 0, "MN-major tokens come in blocks of 64");
  constexpr int kElem = F8 ? 1 : 2, kBK = 128 / kElem;
  constexpr uint32_t kIdesc = instr_desc_majors(F8 ? 0u : 1u, 128, BT, WMN, TMN);
  using MN = BTileMN<2>;

  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBarOff);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * STAGES, accf = empty0 + 8 * STAGES;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * STAGES + 1);
  volatile uint32_t *abort_flag = tmem_slot + 1;
  const WaitCtl wc{abort_flag, p.status, p.limit_ns};

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_m = (p.M + BT - 1) / BT, tiles_n = (p.N + 127) / 128;
  int tm, tn;
  raster_tile((int)blockIdx.x, tiles_m, tiles_n, kRasterGroup, tm, tn);
  const int m0 = tm * BT, n0 = tn * 128;
  const int z = (int)blockIdx.z, splits = (int)gridDim.z;
  const int nkb_all = (p.K + kBK - 1) / kBK;
  const int kb0 = (int)((int64_t)nkb_all * z / splits), nkb = (int)((int64_t)nkb_all * (z + 1) / splits) - kb0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    mbar_init(accf, 1);
    *abort_flag = 0u;
    fence_mbar_init();
    if (p.K > 0) {  // K = 0: no maps
      tma_prefetch_desc(&tmT);
      tma_prefetch_desc(&tmW);
    }
  }
  // Accumulators of `per` stages each, BT columns apart (one of all stages unless p.sum_stages).
  const int per = p.sum_stages ? max(1, (nkb + L::kAccs - 1) / L::kAccs) : max(1, nkb), accs = (nkb + per - 1) / per;
  const uint32_t tmem_cols = p.sum_stages ? L::kSumCols : L::kTmemCols;
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Nothing of global memory is read or written, and no bounded wait begins, before this.
  grid_dependency_wait();
  if (warp == 0 && lane == 0) {
    grid_launch_dependents();
    int kb = 0;
    for (; kb < nkb; ++kb) {
      const int s = kb % STAGES, round = kb / STAGES;
      if (round > 0 && !mbar_wait(empty0 + 8 * s, (round - 1) & 1, wc)) break;
      if (p.debug_skip && kb == 0) continue;  // test hook: this stage never fills
      const uint32_t slot = sbase + s * L::kStageBytes, bar = full0 + 8 * s;
      const int kc = (kb0 + kb) * kBK;
      mbar_arrive_expect_tx(bar, L::kStageBytes);
      // MN-major: blocks of 64 columns, in one load where the map has blocks.
      if constexpr (WMN) {
        if (p.cols_blocks) {
          tma_load_3d(slot, &tmW, 0, kc, n0 / 64, bar);
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) tma_load_2d(slot + j * 8192, &tmW, n0 + 64 * j, kc, bar);
        }
      } else {
        tma_load_2d(slot, &tmW, kc, n0, bar);
      }
      if constexpr (TMN) {
        if (p.rows_blocks) {
          tma_load_3d(slot + L::kWBytes, &tmT, 0, kc, m0 / 64, bar);
        } else {
#pragma unroll
          for (int j = 0; j < BT / 64; ++j) tma_load_2d(slot + L::kWBytes + j * 8192, &tmT, m0 + 64 * j, kc, bar);
        }
      } else {
        tma_load_2d(slot + L::kWBytes, &tmT, kc, m0, bar);
      }
    }
    if (*abort_flag) {  // no load may be in flight when this CTA leaves
#pragma unroll 1
      for (int s = 0; s < STAGES; ++s) {
        if (kb - 1 < s) continue;
        const int last = kb - 1 - ((kb - 1 - s) % STAGES);
        if (p.debug_skip && last == 0) continue;
        mbar_wait_drain(full0 + 8 * s, (last / STAGES) & 1, p.limit_ns);
      }
    }
  } else if (warp == 1 && lane == 0 && nkb > 0) {
    const uint64_t w_d0 = WMN ? MN::desc(sbase, 0, false) : smem_desc(sbase, 16, 1024, 2);
    const uint64_t t_d0 = TMN ? MN::desc(sbase + L::kWBytes, 0, false) : smem_desc(sbase + L::kWBytes, 16, 1024, 2);
    constexpr uint32_t kWStep = WMN ? MN::step(false) >> 4 : 2u, kTStep = TMN ? MN::step(false) >> 4 : 2u;
    int s = 0, piece = 0;  // stages in the current accumulator
    uint32_t phase = 0, acc = tmem;
    uint64_t so = 0;
    for (int kb = 0; kb < nkb; ++kb) {
      if (!mbar_wait(full0 + 8 * s, phase, wc)) break;
      tc_fence_after();
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        if constexpr (F8) mma_ss_f8(acc, w_d0 + so + ks * kWStep, t_d0 + so + ks * kTStep, kIdesc, (piece | ks) ? 1u : 0u);
        else mma_ss<false>(acc, w_d0 + so + ks * kWStep, t_d0 + so + ks * kTStep, kIdesc, (piece | ks) ? 1u : 0u);
      }
      if (++piece == per) {
        piece = 0;
        acc += BT;
      }
      mma_commit(empty0 + 8 * s);
      so += L::kStageBytes >> 4;
      if (++s == STAGES) {
        s = 0;
        phase ^= 1u;
        so = 0;
      }
    }
    mma_commit(accf);
    if (*abort_flag) mbar_wait_drain(accf, 0, p.limit_ns);
  }
  __syncwarp();

  // ---------------- epilogue ----------------
  // Warp w reads TMEM lanes 32 (w % 4) .. + 31, tokens in chunks of 16 by its half.  Value (token j,
  // column r) goes to float j * 128 + r of the ring (every load has been consumed).
  const int q = warp & 3, half = warp >> 2, r = q * 32 + lane;
  const bool ok = nkb == 0 || (mbar_wait(accf, 0, WaitCtl{abort_flag, p.status, p.sum_limit_ns}) && !*abort_flag);
  tc_fence_after();
  const int tokens = p.M - m0 < BT ? p.M - m0 : BT;
  float *part = reinterpret_cast<float *>(smem);
  const uint32_t tacc = tmem + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
  for (int c = half; 16 * c < tokens; c += 2) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = 0.f;
    if (__all_sync(0xFFFFFFFFu, ok)) {
      for (int a = 0; a < accs; ++a) {
        uint32_t rr[16];
        tmem_ld_32x32b_x16(tacc + BT * a + 16 * c, rr);
        tmem_ld_wait(rr);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] += __uint_as_float(rr[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) part[(16 * c + j) * 128 + r] = v[j];
  }
  const bool all_ok = __syncthreads_and(ok);
  if (splits > 1) cluster_sync();
  // This CTA's share of the tile's groups of eight columns, 16 a token.  A tile that reaches beyond N
  // in the middle of a group goes element by element.
  const int groups = tokens * 16, share = (groups + splits - 1) / splits;
  const int g1 = (z + 1) * share < groups ? (z + 1) * share : groups;
  const bool vec = p.vec && (p.N % 8 == 0 || n0 + 128 <= p.N);
  if (all_ok) {
#pragma unroll 1
    for (int g = z * share + (int)threadIdx.x; g < g1; g += L::kThreads) {
      if (vec) finish8<true>(p, g, m0, n0, part, sbase, splits);
      else finish8<false>(p, g, m0, n0, part, sbase, splits);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (splits > 1) cluster_sync();  // no CTA leaves while another may read its sums
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

template <bool F8, bool WMN, bool TMN, int BT, int STAGES>
cudaError_t launch_slim_kern(const CUtensorMap &tmT, const CUtensorMap &tmW, const LinearParams &p, cudaStream_t st) {
  using L = SlimLayout<BT, STAGES>;
  auto kern = linear_slim_kernel<F8, WMN, TMN, BT, STAGES>;
  static unsigned long long configured = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(__atomic_load_n(&configured, __ATOMIC_ACQUIRE) & bit)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemBytes);
    if (e != cudaSuccess) return e;
    __atomic_fetch_or(&configured, bit, __ATOMIC_RELEASE);
  }
  const int64_t tiles = (int64_t)((p.M + BT - 1) / BT) * ((p.N + 127) / 128);
  if (tiles > INT32_MAX) return cudaErrorInvalidConfiguration;
  cudaLaunchAttribute attr[2];
  pdl_attr(attr[0]);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = (unsigned)p.splits;
  cudaLaunchConfig_t cfg = {dim3((unsigned)tiles, 1, (unsigned)p.splits), dim3(L::kThreads), (size_t)L::kSmemBytes, st, attr, 2};
  return cudaLaunchKernelEx(&cfg, kern, tmT, tmW, p);
}

// Ring depths: about 100 KB a CTA, so that two share an SM; one with 256 tokens.  (Twice the depth
// for launches of no more CTAs than SMs measured no faster, and a cluster of eight such CTAs finds
// fewer places: 64 x 512 x 8192 19.1 us instead of 10.9.)
template <bool F8, bool WMN, bool TMN>
cudaError_t launch_slim_bt(int bt, const CUtensorMap &tmT, const CUtensorMap &tmW, const LinearParams &p, cudaStream_t st) {
  if constexpr (!TMN) {
    if (bt == 16) return launch_slim_kern<F8, WMN, TMN, 16, 6>(tmT, tmW, p, st);
    if (bt == 32) return launch_slim_kern<F8, WMN, TMN, 32, 5>(tmT, tmW, p, st);
  }
  if (bt == 64) return launch_slim_kern<F8, WMN, TMN, 64, 4>(tmT, tmW, p, st);
  if (bt == 128) return launch_slim_kern<F8, WMN, TMN, 128, 3>(tmT, tmW, p, st);
  if (bt == 256) return launch_slim_kern<F8, WMN, TMN, 256, 4>(tmT, tmW, p, st);
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_linear_slim(bool f8, bool w_mn, bool t_mn, int bt, const CUtensorMap &tmT, const CUtensorMap &tmW,
                               const LinearParams &p, cudaStream_t st) {
  if (f8) return w_mn || t_mn ? cudaErrorInvalidValue : launch_slim_bt<true, false, false>(bt, tmT, tmW, p, st);
  if (t_mn) return w_mn ? launch_slim_bt<false, true, true>(bt, tmT, tmW, p, st) : cudaErrorInvalidValue;
  return w_mn ? launch_slim_bt<false, true, false>(bt, tmT, tmW, p, st)
              : launch_slim_bt<false, false, false>(bt, tmT, tmW, p, st);
}

}  // namespace tf
