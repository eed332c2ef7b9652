// tf_linear_pair.cu -- the linear layer's large products: persistent CTA pairs on 256 x 256 tiles.
//
//   out[m, n] = act((sum_k A[m, k] B[k, n]) a_scale[m] b_scale[n] + bias[n]) + residual[m, n]
//
// Each cluster of two CTAs walks over output tiles (grouped raster order) with one ring of TMA
// stages running across them -- 128 bytes of k of this CTA's 128 rows of A and of its 128 columns
// of B, each operand K-major or (bf16) MN-major as it lies in memory -- and two accumulators of 256
// TMEM columns: the pair's MMAs (cta_group::2, 256 x 256, bf16 or e4m3) fill one while the epilogue
// empties the other.
//
// Epilogue: sixteen warps a CTA, each by itself (no barrier between them): 32 rows (its TMEM lanes)
// and every fourth chunk of 32 columns.  A thread holds 32 columns of one row; the row's scale is its
// own, the columns' bias and scale are a lane's and go round by shuffles.  Outputs whose rows start on
// 16-byte boundaries leave through the warp's 4 KB of swizzled staging and TMA stores, others through
// the same memory turned round, 32 neighbouring columns of one row at a time.  The residual's chunk
// is brought into the staging by TMA one chunk ahead, so a tile's first while its MMAs run.
//
// Bound by the tensor pipe: 4096 x 4096 -> 16384 bf16 with tanh gelu and pre 377 us (1458 TFLOP/s; ncu
// 85 % busy), 8192 x 16384 -> 4096 e4m3 with residual 392 us (2805; 79 %), replayed from graphs in short
// bursts; 440 to 460 and 460 to 490 in a long run of calls, at the clock that the power cap leaves.
// With few stages of k a tile is bound by this epilogue: 4096 x 256 -> 8192 bf16 with silu takes 56 us
// with eight warps in two groups that meet at barriers and read the residual themselves, 48 as it is
// here; with the bf16 residual 95 and 59.
//
// 640 threads: warp 0 TMA producer (both CTAs), warp 1 MMA issuer (leader), warps 4..19 epilogue.
// Every wait is bounded (tf_ptx.cuh); after an expiry each role stops, the producer, the issuer and
// the epilogue wait (bounded) for what they have in flight, and both CTAs meet before TMEM is freed.
#include <cuda.h>
#include <cuda_runtime.h>

#include "tf_epilogue.cuh"
#include "tf_internal.h"
#include "tf_ptx.cuh"

namespace tf {

namespace {

constexpr int kEpiWarps = 16;

// Forms of the kernel: any call; many stages of k (DEEP); f32 outputs over a long k, whose sums are
// taken in pieces of p.sum_stages stages (SUMS).
enum Form : int { FORM_ANY = 0, FORM_DEEP = 1, FORM_SUMS = 2 };

// Two divisions of the shared memory: five stages and 4 KB of staging an epilogue warp, for every
// call; six stages and 2 KB (deep), for many stages of k and bf16 rows on 16-byte boundaries whose
// chunk needs one box at a time (pair_deep).
template <bool DEEP>
struct PairL {
  static constexpr int kStages = DEEP ? 6 : 5;
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  static constexpr int kABytes = 128 * 128, kBBytes = 128 * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kBoxOff = kStages * kStageBytes;
  static constexpr int kBoxBytes = DEEP ? 2048 : 4096;  // 32 rows x 32 bf16; or f32, or two of bf16
  static constexpr int kBarOff = kBoxOff + kEpiWarps * kBoxBytes;
  // full[], empty[], accf[2], acce[2], drain, resf[warps]; then the TMEM slot and the abort flag.
  static constexpr int kNumBars = 2 * kStages + 5 + kEpiWarps;
  static constexpr int kSmemBytes = 1024 + kBarOff + 8 * kNumBars + 16;
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

__device__ __forceinline__ void add_bf16x8(float *v, const uint4 &u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] += __uint_as_float(w[i] << 16);
    v[2 * i + 1] += __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void add_f32x4(float *v, const float4 &f) {
  v[0] += f.x;
  v[1] += f.y;
  v[2] += f.z;
  v[3] += f.w;
}

// Adds row r of a residual box to v (stage_row's layout).
__device__ __forceinline__ void add_staged(const uint8_t *box, int r, bool bf16, float (&v)[32]) {
  if (bf16) {
#pragma unroll
    for (int u = 0; u < 4; ++u) add_bf16x8(v + 8 * u, *reinterpret_cast<const uint4 *>(box + r * 64 + ((u ^ ((r >> 1) & 3)) << 4)));
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) add_f32x4(v + 4 * u, *reinterpret_cast<const float4 *>(box + r * 128 + ((u ^ (r & 7)) << 4)));
  }
}

// Adds columns col .. col + 31 of a residual row (16-byte aligned groups), those below N.
__device__ __forceinline__ void add_row(const LinearParams &p, int64_t row, int col, float (&v)[32]) {
  if (p.res_bf16) {
    const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(p.residual) + row * p.ldr + col;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (col + 8 * u + 8 <= p.N) {
        add_bf16x8(v + 8 * u, *reinterpret_cast<const uint4 *>(src + 8 * u));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + 8 * u + i < p.N) v[8 * u + i] += __bfloat162float(src[8 * u + i]);
      }
    }
  } else {
    const float *src = static_cast<const float *>(p.residual) + row * p.ldr + col;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (col + 4 * u + 4 <= p.N) {
        add_f32x4(v + 4 * u, *reinterpret_cast<const float4 *>(src + 4 * u));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + 4 * u + i < p.N) v[4 * u + i] += src[4 * u + i];
      }
    }
  }
}

// f(j, x[col0 + j]) for a chunk's columns, those from N on with 0: four at a time by loads that the
// whole warp shares where they are on 16-byte boundaries, else a column a lane by shuffles.
template <typename F>
__device__ __forceinline__ void with_columns(const float *x, int col0, int n, bool vec, int lane, F &&f) {
  if (vec && col0 + 32 <= n) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float4 q = reinterpret_cast<const float4 *>(x + col0)[u];
      f(4 * u, q.x);
      f(4 * u + 1, q.y);
      f(4 * u + 2, q.z);
      f(4 * u + 3, q.w);
    }
  } else {
    const float own = col0 + lane < n ? x[col0 + lane] : 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) f(j, __shfl_sync(0xFFFFFFFFu, own, j));
  }
}

// Row r (of 32) of a staging box: 32 f32 (128-B swizzle) or 32 bf16 (64-B swizzle), as the maps say.
__device__ __forceinline__ void stage_row(uint8_t *box, int r, bool bf16, const float (&v)[32]) {
  if (bf16) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      *reinterpret_cast<uint4 *>(box + r * 64 + ((u ^ ((r >> 1) & 3)) << 4)) =
          make_uint4(pack_bf16x2(v[8 * u], v[8 * u + 1]), pack_bf16x2(v[8 * u + 2], v[8 * u + 3]),
                     pack_bf16x2(v[8 * u + 4], v[8 * u + 5]), pack_bf16x2(v[8 * u + 6], v[8 * u + 7]));
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      *reinterpret_cast<float4 *>(box + r * 128 + ((u ^ (r & 7)) << 4)) =
          make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
  }
}

// A warp's 32 rows x 32 columns turned round through its own 4 KB (column j of row l at j ^ l) and
// stored row by row, a lane a column: any alignment.  R: the residual's type (NoResidual: none),
// added on the way, sixteen rows' loads in flight.  Whole tiles step pointers without conditions.
struct NoResidual {};
template <typename T>
__device__ __forceinline__ void store_as(T *dst, float y) {
  if constexpr (sizeof(T) == 2) *dst = __float2bfloat16_rn(y);
  else *dst = y;
}
template <typename T, typename R>
__device__ __forceinline__ void store_turned(const float *buf, int lane, int rows, T *dst, int64_t ld, const R *res, int64_t ldr) {
  constexpr bool kRes = !std::is_same<R, NoResidual>::value;
  if (__all_sync(0xFFFFFFFFu, rows == 32)) {
#pragma unroll 1
    for (int l0 = 0; l0 < 32; l0 += 16) {
      float x[16];
      if constexpr (kRes) {
#pragma unroll
        for (int i = 0; i < 16; ++i, res += ldr) x[i] = (float)*res;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i, dst += ld) {
        float y = buf[(l0 + i) * 32 + (lane ^ (l0 + i))];
        if constexpr (kRes) y += x[i];
        store_as(dst, y);
      }
    }
  } else {
#pragma unroll 1
    for (int l = 0; l < rows; ++l) {
      float y = buf[l * 32 + (lane ^ l)];
      if constexpr (kRes) y += (float)res[l * ldr];
      store_as(dst + l * ld, y);
    }
  }
}
template <typename T>
__device__ __forceinline__ void store_turned(const LinearParams &p, float *buf, int lane, int64_t row0, int col0, T *base,
                                             int64_t ld, bool res, const float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j) buf[lane * 32 + (j ^ lane)] = v[j];
  __syncwarp();
  const int rows = col0 + lane < p.N ? (int)(p.M - row0 < 32 ? p.M - row0 : 32) : 0;
  T *dst = base + row0 * ld + col0 + lane;
  const int64_t r = row0 * p.ldr + col0 + lane;
  if (!res) store_turned(buf, lane, rows, dst, ld, static_cast<const NoResidual *>(nullptr), 0);
  else if (p.res_bf16) store_turned(buf, lane, rows, dst, ld, static_cast<const __nv_bfloat16 *>(p.residual) + r, p.ldr);
  else store_turned(buf, lane, rows, dst, ld, static_cast<const float *>(p.residual) + r, p.ldr);
  __syncwarp();
}

// This CTA's 128 columns from c0 of an MN-major operand, 64 rows of k: two blocks of 64 columns, in one
// load where the map has blocks.  One load instead of two: 8192 x 4096 x 16384's weight gradient,
// both operands MN-major, 870 -> 830 us (calls in a row under the power cap).
__device__ __forceinline__ void load_mn(uint32_t dst, const void *tmap, int32_t blocks, int c0, int kc, uint32_t bar) {
  if (blocks) {
    tma_load_3d_pair(dst, tmap, 0, kc, c0 / 64, bar);
  } else {
    tma_load_2d_pair(dst, tmap, c0, kc, bar);
    tma_load_2d_pair(dst + 8192, tmap, c0 + 64, kc, bar);
  }
}

// F8: e4m3 operands (both K-major).  AMN / BMN: A / B is MN-major (bf16).
template <bool F8, bool AMN, bool BMN, int FORM>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairL<FORM == FORM_DEEP>::kThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmP,
                       const __grid_constant__ CUtensorMap tmR, const LinearParams p) {
  constexpr bool DEEP = FORM == FORM_DEEP, SUMS = FORM == FORM_SUMS;
  using L = PairL<DEEP>;
  constexpr int STAGES = L::kStages;
  static_assert(!F8 || (!AMN && !BMN), "8-bit operands are K-major");
  constexpr int kBK = F8 ? 128 : 64;
  constexpr uint32_t kIdesc = instr_desc_majors(F8 ? 0u : 1u, 256, 256, AMN, BMN);
  using MN = BTileMN<2>;

  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBarOff);
  // full[s] (leader's): both CTAs' bytes of slot s landed; empty[s]: the MMAs reading slot s are done
  // (both CTAs); accf[b]: accumulator b holds a tile (both CTAs); acce[b] (leader's): both CTAs'
  // epilogues have read accumulator b; drain: MMAs in flight after an abort; resf[w]: epilogue warp
  // w's residual box landed.
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * STAGES, accf0 = empty0 + 8 * STAGES, acce0 = accf0 + 16,
                 drainf = acce0 + 16, resf0 = drainf + 8;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + L::kNumBars);
  volatile uint32_t *abort_flag = tmem_slot + 1;
  const WaitCtl wc{abort_flag, p.status, p.limit_ns}, wsum{abort_flag, p.status, p.sum_limit_ns};

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int tiles_m = (p.M + 255) / 256, tiles_n = (p.N + 255) / 256, tiles = tiles_m * tiles_n;
  const int pair = (int)(blockIdx.x >> 1), npairs = (int)(gridDim.x >> 1);
  const int my_tiles = pair < tiles ? (tiles - 1 - pair) / npairs + 1 : 0;
  const int nkb = (p.K + kBK - 1) / kBK;
  // Pieces of a tile's k, an accumulator each in turn.
  const int per = SUMS ? p.sum_stages : nkb, pieces = SUMS ? (nkb + per - 1) / per : 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf0 + 8 * b, 1);
      mbar_init(acce0 + 8 * b, 2 * kEpiWarps);  // lane 0 of the epilogue warps of both CTAs
    }
    mbar_init(drainf, 1);
    for (int w = 0; w < kEpiWarps; ++w) mbar_init(resf0 + 8 * w, 1);
    *abort_flag = 0u;
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (p.vec) tma_prefetch_desc(&tmO);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers are initialised before any remote arrive or TMA
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Nothing of global memory is read or written, and no bounded wait begins, before this.
  grid_dependency_wait();
  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    grid_launch_dependents();
    const uint32_t lead_full0 = map_to_cta(full0, 0);
    int g = 0;  // k-blocks issued so far
    bool ok = true;
    for (int i = 0; i < my_tiles && ok; ++i) {
      int tm, tn;
      raster_tile(pair + i * npairs, tiles_m, tiles_n, kRasterGroup, tm, tn);
      const int m0 = tm * 256 + (int)rank * 128, n0 = tn * 256 + (int)rank * 128;
      for (int kb = 0; kb < nkb; ++kb, ++g) {
        const int s = g % STAGES, round = g / STAGES;
        if (round > 0 && !mbar_wait_cluster(empty0 + 8 * s, (round - 1) & 1, wc)) {
          ok = false;
          break;
        }
        if (p.debug_skip && g == 0) continue;  // test hook: this stage never fills
        const int kc = kb * kBK;
        const uint32_t slot = sbase + s * L::kStageBytes, bar = lead_full0 + 8 * s;
        if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, 2 * L::kStageBytes);
        if constexpr (AMN) {
          load_mn(slot, &tmA, p.rows_blocks, m0, kc, bar);
        } else {
          tma_load_2d_pair(slot, &tmA, kc, m0, bar);
        }
        if constexpr (BMN) {
          load_mn(slot + L::kABytes, &tmB, p.cols_blocks, n0, kc, bar);
        } else {
          tma_load_2d_pair(slot + L::kABytes, &tmB, kc, n0, bar);
        }
      }
    }
    if (*abort_flag) {
      if (rank == 0) {
#pragma unroll 1
        for (int s = 0; s < STAGES; ++s) {
          if (g - 1 < s) continue;
          const int last = g - 1 - ((g - 1 - s) % STAGES);
          if (p.debug_skip && last == 0) continue;
          mbar_wait_drain_cluster(full0 + 8 * s, (last / STAGES) & 1, p.limit_ns);
        }
      } else {  // this CTA's loads complete on the leader's barriers
        const uint64_t t0 = globaltimer();
        while (globaltimer() - t0 < 200000) __nanosleep(1000);
      }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---------------- pair MMA issuer (leader CTA) ----------------
    bool ok = true;
    const uint64_t a_d0 = AMN ? MN::desc(sbase, 0, false) : smem_desc(sbase, 16, 1024, 2);
    const uint64_t b_d0 = BMN ? MN::desc(sbase + L::kABytes, 0, false) : smem_desc(sbase + L::kABytes, 16, 1024, 2);
    constexpr uint32_t kAStep = AMN ? MN::step(false) >> 4 : 2u, kBStep = BMN ? MN::step(false) >> 4 : 2u;
    int s = 0;
    uint32_t phase = 0, bar = full0;
    uint64_t so = 0;
    for (int u = 0; u < my_tiles * pieces && ok; ++u) {
      const int b = u & 1;
      const uint32_t acc = tmem + 256u * b;
      if (u >= 2 && !mbar_wait_cluster(acce0 + 8 * b, ((u >> 1) - 1) & 1, wc)) break;
      tc_fence_after();
      const int kb0 = SUMS ? u % pieces * per : 0, kb1 = SUMS && kb0 + per < nkb ? kb0 + per : nkb;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_cluster(bar, phase, wc)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t ad = a_d0 + so, bd = b_d0 + so;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const uint32_t add = kb != kb0 || ks ? 1u : 0u;
          if constexpr (F8) mma_ss_pair_f8(acc, ad + ks * kAStep, bd + ks * kBStep, kIdesc, add);
          else mma_ss_pair<false>(acc, ad + ks * kAStep, bd + ks * kBStep, kIdesc, add);
        }
        mma_commit_pair(bar + 8 * STAGES, 0x3);
        if (++s == STAGES) {
          s = 0;
          phase ^= 1u;
          bar = full0;
          so = 0;
        } else {
          bar += 8;
          so += L::kStageBytes >> 4;
        }
      }
      if (!ok) break;
      mma_commit_pair(accf0 + 8 * b, 0x3);
    }
    if (*abort_flag) {
      mma_commit_pair(drainf, 0x1);
      mbar_wait_drain_cluster(drainf, 0, p.limit_ns);
    }
  } else if (warp >= 4) {
    // ---------------- epilogue (both CTAs): warps 4..19 ----------------
    // TMEM lanes 32 q .. + 31, chunks part and part + 4 of a tile's eight.
    const int part = (warp - 4) >> 2, q = warp & 3;
    const uint32_t lead_acce0 = map_to_cta(acce0, 0), resf = resf0 + 8 * (warp - 4);
    uint8_t *box = smem + L::kBoxOff + (warp - 4) * L::kBoxBytes;
    const bool bf16 = !SUMS && (DEEP || p.out_bf16), pre = p.pre != nullptr, vec = DEEP || p.vec, res_bf16 = DEEP || p.res_bf16;
    const bool pingpong = !DEEP && bf16 && !pre && !p.residual;
    // The residual comes by TMA into the box, in whose place the chunk's output is then staged, but
    // where pre needs the box first (f32 out or residual with pre): then by the row's own loads.
    const bool res_tma = p.residual && vec && !(pre && (!bf16 || !res_bf16));
    const uint32_t res_bytes = res_bf16 ? 2048u : 4096u;
    uint32_t turn = 0, res_phase = 0;
    bool res_flight = false;
    auto tile_at = [&](int i, int &m0, int &n0) {
      int tm, tn;
      raster_tile(pair + i * npairs, tiles_m, tiles_n, kRasterGroup, tm, tn);
      m0 = tm * 256 + (int)rank * 128 + q * 32;  // this warp's first row
      n0 = tn * 256;
    };
    auto inside = [&](int m0, int col0) { return m0 < p.M && col0 < p.N; };  // the same for the whole warp
    // Starts the residual's way into the box, once the stores from it have read it.
    auto fetch_residual = [&](int m0, int col0) {
      if (!res_tma || !inside(m0, col0)) return;
      if (lane == 0) {
        bulk_wait_group_read0();
        mbar_arrive_expect_tx(resf, res_bytes);
        tma_load_2d(smem_u32(box), &tmR, col0, m0, resf);
      }
      res_flight = true;
    };
    int m0 = 0, n0 = 0;
    if (my_tiles > 0) {
      tile_at(0, m0, n0);
      if (!SUMS) fetch_residual(m0, n0 + 32 * part);
    }
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i < my_tiles && ok; ++i) {
      const int u = i * pieces + pieces - 1, b = u & 1;  // the tile's last piece
      const uint32_t lanes = (uint32_t)(q * 32) << 16;
      if constexpr (SUMS) {
        // The pieces' sums, in order: half of them in registers, half in the warp's box; the last piece's
        // go back into its accumulator, from where they go on as a whole sum would.  (What does not fit
        // the registers is spilled past the small L1 to L2: with all of them in registers 4096 x 1024 ->
        // 4096 takes 55 us instead of 45.)
        constexpr int kBoxed = 4;  // groups of eight columns whose sums are in the box
        if (lane == 0) bulk_wait_group_read0();
        __syncwarp();
        float *boxed = reinterpret_cast<float *>(box) + lane;
        float sum[64 - 8 * kBoxed];
#pragma unroll
        for (int j = 0; j < 64 - 8 * kBoxed; ++j) sum[j] = 0.f;
#pragma unroll
        for (int j = 0; j < 8 * kBoxed; ++j) boxed[32 * j] = 0.f;
#pragma unroll 1
        for (int w = i * pieces; w <= u; ++w) {
          ok = __all_sync(0xFFFFFFFFu, mbar_wait_cluster(accf0 + 8 * (w & 1), (w >> 1) & 1, wc, 64));
          if (!ok) break;
          tc_fence_after();
          const uint32_t tacc = tmem + 256u * (w & 1) + lanes + part * 32;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            uint32_t rr[8];
            tmem_ld_32x32b_x8(tacc + g / 4 * 128 + g % 4 * 8, rr);
            tmem_ld_wait(rr);
            if (g < kBoxed) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float x = boxed[32 * (8 * g + j)] + __uint_as_float(rr[j]);
                boxed[32 * (8 * g + j)] = x;
                rr[j] = __float_as_uint(x);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) sum[8 * (g - kBoxed) + j] += __uint_as_float(rr[j]);
              if (w == u) {
#pragma unroll
                for (int j = 0; j < 8; ++j) rr[j] = __float_as_uint(sum[8 * (g - kBoxed) + j]);
              }
            }
            if (w == u) tmem_st_32x32b_x8(tacc + g / 4 * 128 + g % 4 * 8, rr);
          }
          if (w < u) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(lead_acce0 + 8 * (w & 1));
          }
        }
        if (!ok) break;
        tmem_st_wait();
        fence_proxy_async_smem();  // the sums' accesses of the box, before TMA writes there
        __syncwarp();
        fetch_residual(m0, n0 + 32 * part);
      }
      const float sa = p.a_scale && m0 + lane < p.M ? p.a_scale[m0 + lane] : 1.f;
      // Not unrolled: the body, with an activation's 32 copies, should stay in the instruction cache.
#pragma unroll 1
      for (int k = 0; k < 2; ++k) {
        const int c = part + 4 * k, col0 = n0 + 32 * c;
        const bool live = inside(m0, col0);
        if (!SUMS && k == 0) {
          ok = __all_sync(0xFFFFFFFFu, mbar_wait_cluster(accf0 + 8 * b, (u >> 1) & 1, wsum, 64));
          if (!ok) break;
          tc_fence_after();
        }
        uint32_t rr[32];
        if (live) {
          tmem_ld_32x32b_x32(tmem + 256u * b + lanes + c * 32, rr);
          tmem_ld_wait(rr);
        }
        if (k == 1) {  // this warp's last read of accumulator b is done: release it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(lead_acce0 + 8 * b);
        }
        if (!live) continue;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(rr[j]);
        if constexpr (F8) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= sa;
          with_columns(p.b_scale, col0, p.N, vec, lane, [&](int j, float x) { v[j] *= x; });
        }
        if (p.bias) with_columns(p.bias, col0, p.N, vec, lane, [&](int j, float x) { v[j] += x; });
        if (vec && !res_tma) {
          // The box is free once the stores issued from it have read it: all but the last one when it
          // has two bf16 halves to alternate between.
          if (lane == 0) {
            if (pingpong) bulk_wait_group_read1();
            else bulk_wait_group_read0();
          }
          __syncwarp();
        }
        if (pre) {
          if (!vec) {
            float *buf = reinterpret_cast<float *>(box);
            if (bf16) store_turned(p, buf, lane, m0, col0, static_cast<__nv_bfloat16 *>(p.pre), p.ldp, false, v);
            else store_turned(p, buf, lane, m0, col0, static_cast<float *>(p.pre), p.ldp, false, v);
          } else {
            const bool beside = !DEEP && bf16;  // the output has a place of its own
            uint8_t *pbox = beside ? box + 2048 : box;
            stage_row(pbox, lane, bf16, v);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmP, smem_u32(pbox), col0, m0);
              bulk_commit_group();
              if (!beside) bulk_wait_group_read0();
            }
            __syncwarp();
          }
        }
        with_activation(p.act, [&](auto act) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = activate<decltype(act)::value>(v[j]);
        });
        if (!vec) {
          float *buf = reinterpret_cast<float *>(box);
          if (bf16) store_turned(p, buf, lane, m0, col0, static_cast<__nv_bfloat16 *>(p.out), p.ldo, p.residual != nullptr, v);
          else store_turned(p, buf, lane, m0, col0, static_cast<float *>(p.out), p.ldo, p.residual != nullptr, v);
          continue;
        }
        if (res_tma) {
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(resf, res_phase, wc));
          if (!ok) break;
          res_phase ^= 1u;
          res_flight = false;
          add_staged(box, lane, res_bf16, v);
          __syncwarp();  // every row has been read before the output takes its place
        } else if (p.residual && m0 + lane < p.M) {
          add_row(p, m0 + lane, col0, v);
        }
        uint8_t *obox = pingpong && (turn & 1) ? box + 2048 : box;
        ++turn;
        stage_row(obox, lane, bf16, v);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&tmO, smem_u32(obox), col0, m0);
          bulk_commit_group();
        }
        if (k == 0) fetch_residual(m0, col0 + 128);
      }
      if (ok && i + 1 < my_tiles) {
        tile_at(i + 1, m0, n0);
        if (!SUMS) fetch_residual(m0, n0 + 32 * part);
      }
    }
    if (lane == 0) {
      if (res_flight) mbar_wait_drain(resf, res_phase, p.limit_ns);  // after an abort
      bulk_wait_group_read0();  // staging stays valid until read
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while the pair MMA may still read its memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Co-resident clusters of one instantiation on the current device (0 on failure).
template <bool F8, bool AMN, bool BMN, int FORM>
int pair_clusters() {
  using L = PairL<FORM == FORM_DEEP>;
  auto kern = linear_pair_kernel<F8, AMN, BMN, FORM>;
  static int cached[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  int *slot = &cached[dev & 63];
  int v = __atomic_load_n(slot, __ATOMIC_ACQUIRE);
  if (v > 0) return v;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemBytes) != cudaSuccess) return 0;
  int sms = 0;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (sms / 2 > 0 ? sms / 2 : 1), 1, 1);
  cfg.blockDim = dim3(L::kThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kSmemBytes;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 0;
  }
  __atomic_store_n(slot, n, __ATOMIC_RELEASE);
  return n;
}

template <bool F8, bool AMN, bool BMN, int FORM>
cudaError_t launch_pair_form(const CUtensorMap &tmA, const CUtensorMap &tmB, const CUtensorMap &tmO, const CUtensorMap &tmP,
                        const CUtensorMap &tmR, const LinearParams &p, cudaStream_t st) {
  using L = PairL<FORM == FORM_DEEP>;
  const int clusters = pair_clusters<F8, AMN, BMN, FORM>();
  if (clusters <= 0) return cudaErrorInvalidConfiguration;
  const int64_t tiles = (int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256);
  if (tiles > INT32_MAX) return cudaErrorInvalidConfiguration;
  const int pairs = tiles < clusters ? (int)tiles : clusters;
  cudaLaunchAttribute attr[1];
  pdl_attr(attr[0]);
  cudaLaunchConfig_t cfg = {dim3(2 * pairs), dim3(L::kThreads), (size_t)L::kSmemBytes, st, attr, 1};
  return cudaLaunchKernelEx(&cfg, linear_pair_kernel<F8, AMN, BMN, FORM>, tmA, tmB, tmO, tmP, tmR, p);
}

// The deep form from 32 stages of k: 4096 x 16384 x 4096 bf16 424 us and, with tanh gelu and pre, 447
// (five stages 434 and 459; calls in a row under the power cap).  With few stages the epilogue's
// second box counts for more.  It takes bf16 outputs whose rows start on 16-byte boundaries, with pre
// or a bf16 residual but not both.
bool pair_deep(const LinearParams &p, int esz) {
  return (int64_t)p.K * esz >= 32 * 128 && p.out_bf16 && p.vec && !(p.pre && p.residual) && (!p.residual || p.res_bf16);
}

template <bool F8, bool AMN, bool BMN>
cudaError_t launch_pair(const CUtensorMap &tmA, const CUtensorMap &tmB, const CUtensorMap &tmO, const CUtensorMap &tmP,
                        const CUtensorMap &tmR, const LinearParams &p, cudaStream_t st) {
  if (p.sum_stages) return launch_pair_form<F8, AMN, BMN, FORM_SUMS>(tmA, tmB, tmO, tmP, tmR, p, st);
  return pair_deep(p, F8 ? 1 : 2) ? launch_pair_form<F8, AMN, BMN, FORM_DEEP>(tmA, tmB, tmO, tmP, tmR, p, st)
                                  : launch_pair_form<F8, AMN, BMN, FORM_ANY>(tmA, tmB, tmO, tmP, tmR, p, st);
}

}  // namespace

cudaError_t launch_linear_pair(bool f8, bool a_mn, bool b_mn, const CUtensorMap &tmA, const CUtensorMap &tmB,
                               const CUtensorMap &tmO, const CUtensorMap &tmP, const CUtensorMap &tmR, const LinearParams &p,
                               cudaStream_t st) {
  if (p.K <= 0 || (f8 && (a_mn || b_mn)) || (a_mn && !b_mn)) return cudaErrorInvalidValue;
  if (f8) return launch_pair<true, false, false>(tmA, tmB, tmO, tmP, tmR, p, st);
  if (a_mn) return launch_pair<false, true, true>(tmA, tmB, tmO, tmP, tmR, p, st);
  return b_mn ? launch_pair<false, false, true>(tmA, tmB, tmO, tmP, tmR, p, st)
              : launch_pair<false, false, false>(tmA, tmB, tmO, tmP, tmR, p, st);
}

}  // namespace tf
