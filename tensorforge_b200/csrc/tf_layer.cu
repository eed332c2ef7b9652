// tf_layer.cu -- C-ABI of the transformer-layer operators (include/tforge.h): argument checks,
// operand copies where TMA cannot read the caller's rows, the choice of the product's kernel, and
// the gradient's elementwise pass.  The kernels are in tf_linear_slim.cu, tf_linear_pair.cu and
// tf_norm.cu.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "tf_epilogue.cuh"
#include "tf_internal.h"

using namespace tf;

namespace {

// tforge_debug_linear_kernel: kernel | tile << 8 | splits << 24.
std::atomic<uint32_t> g_force{0};

bool at(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int elem_size(int dtype) { return dtype == TFORGE_F32 ? 4 : (dtype == TFORGE_BF16 ? 2 : 1); }
bool is_float(int dtype) { return dtype == TFORGE_F32 || dtype == TFORGE_BF16; }

// A row-pitched array of the call, for the checks that every entry makes.
struct Array {
  const void *p;
  int64_t rows, cols, ld;
  int esz;
  uint64_t bytes() const { return rows > 0 && cols > 0 ? ((uint64_t)(rows - 1) * ld + cols) * esz : 0; }
};

// Column slices of one buffer (equal pitches, different columns) do not overlap.
bool overlap(const Array &a, const Array &b) {
  if (!a.p || !b.p || !a.bytes() || !b.bytes()) return false;
  const uintptr_t a0 = reinterpret_cast<uintptr_t>(a.p), b0 = reinterpret_cast<uintptr_t>(b.p);
  if (!(a0 < b0 + b.bytes() && b0 < a0 + a.bytes())) return false;
  const uint64_t pitch = (uint64_t)a.ld * a.esz;
  if (pitch != (uint64_t)b.ld * b.esz) return true;
  const uint64_t behind = a0 <= b0 ? (b0 - a0) % pitch : (pitch - (a0 - b0) % pitch) % pitch;  // b's columns behind a's
  return behind < (uint64_t)a.cols * a.esz || behind + (uint64_t)b.cols * b.esz > pitch;
}
bool same(const Array &a, const Array &b) { return a.p == b.p && a.ld == b.ld && a.esz == b.esz; }

// Every array element-aligned; no output overlapping another output or an input, but that
// outs[share] may be the same array as ins[with0] or ins[with1].
template <int NI, int NO>
int check_arrays(const Array (&ins)[NI], const Array (&outs)[NO], int share = -1, int with0 = -1, int with1 = -1) {
  for (const Array &a : ins)
    if (!at(a.p, a.esz)) return TFORGE_ERR_ALIGN;
  for (const Array &a : outs)
    if (!at(a.p, a.esz)) return TFORGE_ERR_ALIGN;
  for (int o = 0; o < NO; ++o) {
    for (int i = 0; i < NI; ++i)
      if (overlap(outs[o], ins[i]) && !(o == share && (i == with0 || i == with1) && same(outs[o], ins[i])))
        return TFORGE_ERR_ALIAS;
    for (int q = 0; q < o; ++q)
      if (overlap(outs[o], outs[q])) return TFORGE_ERR_ALIAS;
  }
  return TFORGE_OK;
}

// Up to 2^30: rounded up to a tile a coordinate stays in 32 bits.
bool dims_ok(int64_t a, int64_t b, int64_t c = 0) {
  constexpr int64_t most = (int64_t)1 << 30;
  return a >= 0 && b >= 0 && c >= 0 && a <= most && b <= most && c <= most;
}
// Fills a zero pitch in; false when a pitch is shorter than its row (or unreasonably long: byte
// offsets stay within 63 bits).  The pitch of an array that is not there says nothing, and is made the
// packed one, which keeps no kernel from wide accesses.
bool pitch(int64_t &ld, int64_t cols, bool there = true) {
  if (ld == 0 || !there) ld = cols;
  return ld >= cols && ld <= (int64_t)1 << 31;
}

// Stream-ordered scratch of one call: parts are asked for, then taken in one allocation, released (in
// stream order) when the call returns.
class Scratch {
 public:
  explicit Scratch(cudaStream_t st) : st_(st) {}
  Scratch(const Scratch &) = delete;
  ~Scratch() {
    if (base_) cudaFreeAsync(base_, st_);
  }
  // Offset of `bytes` more, on a 256-byte boundary.
  uint64_t want(uint64_t bytes) {
    const uint64_t at = size_;
    size_ += (bytes + 255) & ~uint64_t(255);
    return at;
  }
  int take() {
    if (!size_) return TFORGE_OK;
    cudaMemPool_t pool = nullptr;
    int rc = device_pool(&pool);
    if (rc) return rc;
    void *p = nullptr;
    cudaError_t e = cudaMallocFromPoolAsync(&p, size_, pool, st_);
    if (e != cudaSuccess) return cuda_failure(e, "cudaMallocFromPoolAsync(layer scratch)");
    base_ = static_cast<char *>(p);
    return TFORGE_OK;
  }
  char *at(uint64_t offset) const { return base_ + offset; }

 private:
  cudaStream_t st_;
  char *base_ = nullptr;
  uint64_t size_ = 0;
};

// ---- operand copies -------------------------------------------------------------------------------

// dst[r * ldd + c] = src[r * lds + c]; dtype is src's: f32 is rounded to bf16.
struct RowCopy {
  const void *src;
  void *dst;
  int64_t rows, cols, lds, ldd;
  int32_t dtype;
};

// Sixteen bytes of the copy a thread.  The source row may start anywhere: 8- and 16-bit elements are
// read as the aligned words around them and shifted into place, element by element only where a word
// would reach outside the array.  What a row's last group holds beyond its end is not read by anyone.
template <int ESZ>
__device__ __forceinline__ void copy_groups(const RowCopy &j, int64_t first, int64_t step) {
  constexpr int kPer = 16 / ESZ;
  const int64_t groups = (j.cols + kPer - 1) / kPer, total = j.rows * groups;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(j.src), end = begin + ((j.rows - 1) * j.lds + j.cols) * ESZ;
  for (int64_t i = first; i < total; i += step) {
    const int64_t r = i / groups, c = (i - r * groups) * kPer;
    const uintptr_t at = begin + (uintptr_t)((r * j.lds + c) * ESZ), word = at & ~uintptr_t(3);
    const uint32_t shift = 8u * (uint32_t)(at & 3);
    uint32_t w[5] = {0, 0, 0, 0, 0};
    if (word >= begin && word + (shift ? 20 : 16) <= end) {
      const uint32_t *src = reinterpret_cast<const uint32_t *>(word);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = src[k];
      if (shift) {
        w[4] = src[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], shift);
      }
    } else {
      const int live = j.cols - c < kPer ? (int)(j.cols - c) : kPer;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        if (k < live) {
          const uint32_t v = ESZ == 1 ? reinterpret_cast<const uint8_t *>(at)[k] : reinterpret_cast<const uint16_t *>(at)[k];
          w[k * ESZ / 4] |= v << (8 * (k * ESZ % 4));
        }
      }
    }
    *reinterpret_cast<uint4 *>(static_cast<uint8_t *>(j.dst) + (r * j.ldd + c) * ESZ) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// f32 to bf16, eight elements a thread.
__device__ __forceinline__ void convert_groups(const RowCopy &j, int64_t first, int64_t step) {
  const int64_t groups = (j.cols + 7) / 8, total = j.rows * groups;
  const bool vec = (reinterpret_cast<uintptr_t>(j.src) & 15) == 0 && j.lds % 4 == 0;
  for (int64_t i = first; i < total; i += step) {
    const int64_t r = i / groups, c = (i - r * groups) * 8;
    const float *s = static_cast<const float *>(j.src) + r * j.lds + c;
    float v[8];
    if (vec && c + 8 <= j.cols) {
      const float4 a = reinterpret_cast<const float4 *>(s)[0], b = reinterpret_cast<const float4 *>(s)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = c + k < j.cols ? s[k] : 0.f;
    }
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(j.dst) + r * j.ldd + c) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
}

// Bound by HBM: 13824 x 9754 bf16 (270 MB) 92 us, 5.9 TB/s.
// One or two operands' copies in one launch: blocks below `split` the first's, the others the second's.
__global__ void __launch_bounds__(256) copy_rows_kernel(const RowCopy a, const RowCopy b, int split) {
  grid_dependency_wait();
  grid_launch_dependents();
  const bool second = (int)blockIdx.x >= split;
  const RowCopy &j = second ? b : a;
  const int64_t block = second ? blockIdx.x - split : blockIdx.x, blocks = second ? gridDim.x - split : split;
  const int64_t first = block * 256 + threadIdx.x, step = blocks * 256;
  if (j.dtype == TFORGE_F32) convert_groups(j, first, step);
  else if (j.dtype == TFORGE_BF16) copy_groups<2>(j, first, step);
  else copy_groups<1>(j, first, step);
}

int64_t padded(int64_t cols, int esz) { return (cols * esz + 15) / 16 * 16 / esz; }

// An operand as the tensor core takes it: bf16 or e4m3 rows on 16-byte boundaries.
struct Operand {
  const void *p;
  int64_t rows, cols, ld;  // as stored
};

// The operand copies of one call (at most two).
class Copies {
 public:
  // Notes the copy that `o` needs, if any, and asks for its place.
  void add(Operand &o, int dtype, Scratch &scratch) {
    const int esz = dtype == TFORGE_E4M3 ? 1 : 2;
    if (o.rows == 0 || o.cols == 0) return;
    if (dtype != TFORGE_F32 && at(o.p, 16) && o.ld * esz % 16 == 0) return;
    const int64_t ldd = padded(o.cols, esz);
    offset_[n_] = scratch.want((uint64_t)o.rows * ldd * esz);
    job_[n_] = {o.p, nullptr, o.rows, o.cols, o.ld, ldd, dtype};
    operand_[n_++] = &o;
  }
  // After scratch.take(): launches the copies and points the operands at them.
  int run(const Scratch &scratch, cudaStream_t st) {
    if (!n_) return TFORGE_OK;
    int64_t blocks[2] = {0, 0};
    for (int i = 0; i < n_; ++i) {
      job_[i].dst = scratch.at(offset_[i]);
      operand_[i]->p = job_[i].dst;
      operand_[i]->ld = job_[i].ldd;
      const int64_t per = job_[i].dtype == TFORGE_E4M3 ? 16 : 8;
      blocks[i] = (job_[i].rows * ((job_[i].cols + per - 1) / per) + 255) / 256;
    }
    // Up to 16 blocks an SM, shared by the groups that each operand has.
    const int64_t most = 148 * 16, total = blocks[0] + blocks[1];
    if (total > most) {
      blocks[0] = std::max<int64_t>(1, most * blocks[0] / total);
      if (blocks[1]) blocks[1] = std::max<int64_t>(1, most - blocks[0]);
    }
    cudaError_t e = launch_dependent(copy_rows_kernel, dim3((unsigned)(blocks[0] + blocks[1])), dim3(256), st, 0, job_[0],
                                     job_[n_ - 1], (int)blocks[0]);
    return e == cudaSuccess ? TFORGE_OK : cuda_failure(e, "operand copy");
  }

 private:
  int n_ = 0;
  uint64_t offset_[2];
  RowCopy job_[2];
  Operand *operand_[2];
};

// ---- the products ---------------------------------------------------------------------------------

// The kernel of a product: tile 0 = CTA pairs on 256 x 256 tiles, else the slim kernel's tile rows
// and the CTAs that share a tile.
struct Choice {
  int tile;
  int splits;
};

// The pair kernel where its tiles fill the 74 pairs once; else the least estimated time in us over it
// and the slim kernel's tiles and splits.  Such products need no estimate, few stages of k among them:
// bf16 8192 x 8192 with k = 32 .. 512 takes pairs 59 to 71 us and the slim kernel's best tile 104 to
// 138, 2560 x 2048 (80 tiles) 11 to 14 and 14 to 18, 32768 x 640 27 to 33 and 36 to 51, with f32 out,
// gelu or a residual the same way; of 90 forms only some of 9472 x 512 went to the slim kernel, by 2 to
// 8 % (k = 64 with gelu 11.2 and 10.3).  The estimates are fits to a sweep of 162 problems (M 1 ..
// 4096, nine N x K from 128 x 2048 to 16384 x 4096, bf16 and e4m3) by every kernel: the choice is
// 2.8 % slower than the fastest on average, and at worst 25 % (2048 x 1024 x 1024: 13.8 us, 11.0).
//   memory: operands and output once at the measured copy rate.
//   pair:   waves of 74 pairs, each 0.356 us a stage of k (at least 5.1: an epilogue), or 1.58 x memory.
//   slim:   a stage of k costs a CTA 0.265 us and 0.0005 per row of its tile, two CTAs an SM each
//           0.55 of that (one with 256 rows); smoothly no less than 1.17 x memory; per round of
//           resident CTAs 2.6 us and what a cluster of S costs to meet; per CTA on an SM the
//           epilogue's rows.
// f32 outputs take only kernels that sum in pieces short enough: the pair kernel always can, the slim
// kernel's accumulators share a CTA's k.
Choice choose(int64_t M, int64_t N, int64_t K, bool t_mn, int esz, bool f32_out) {
  const double nkb = (double)((K * esz + 127) / 128);
  const double most = f32_out ? (esz == 1 ? 64.0 : 12.0) : 1e300;  // stages of k in one sum
  const double memory = ((double)esz * K * (M + N) + 2.0 * M * N) / 6.55e6;
  const double tiles256 = std::ceil(M / 256.0) * std::ceil(N / 256.0);
  Choice best{0, 1};
  if (K > 0 && tiles256 >= 74) return best;
  double least = 5.65 + std::fmax(std::fmax(0.356 * nkb, 5.1), 1.58 * memory);
  if (K == 0) least = 1e300;  // the pair kernel needs a k
  for (int tile = t_mn ? 64 : 16; tile <= 256; tile *= 2) {
    const double tiles = std::ceil((double)M / tile) * std::ceil(N / 128.0), live = M < tile ? (double)M : tile;
    for (int s = 1; s <= 8; s *= 2) {
      if (std::ceil(nkb / s) > most * (256 / tile)) continue;
      // CTAs that the SMs hold at once: clusters of 4 and 8 do not find a place on every SM.
      const double slots = tile == 256 ? (s <= 2 ? 148 : s == 4 ? 132 : 120) : (s <= 2 ? 296 : s == 4 ? 284 : 264);
      const double ctas = tiles * s, deep = std::ceil(ctas / 148.0), rounds = std::ceil(ctas / slots);
      const double load = (deep == 1 || tile == 256 ? deep : 0.55 * deep) * std::ceil(nkb / s) * (0.265 + 0.000511 * tile);
      const double l2 = load * load, m2 = 1.17 * 1.17 * memory * memory;
      const double t = std::sqrt(std::sqrt(l2 * l2 + m2 * m2)) + rounds * (2.57 + (s > 1 ? 0.21 + 0.29 * s : 0.0)) +
                       deep * live * (s > 1 ? 0.0351 : 0.0319);
      if (t < least) {
        least = t;
        best = Choice{tile, s};
      }
    }
    if (tile >= M) break;  // a wider tile would only add empty rows
  }
  return best;
}

// out (M x N) = epilogue(rows . cols).  rows: M x K, or K x M with t_mn; cols: N x K, or K x N
// with w_mn.  p carries the epilogue.
int product(const Operand &rows, bool t_mn, const Operand &cols, bool w_mn, bool f8, int64_t M, int64_t N, int64_t K,
            LinearParams p, cudaStream_t st) {
  if (M == 0 || N == 0) return TFORGE_OK;
  const int esz = f8 ? 1 : 2;
  p.M = (int32_t)M;
  p.N = (int32_t)N;
  p.K = (int32_t)K;
  int rc = device_status_word(&p.status);
  if (rc) return rc;
  p.limit_ns = wait_limit_ns();
  p.debug_skip = debug_skip_load();
  auto rows16 = [](const void *q, int64_t ld, int e) { return !q || (at(q, 16) && ld * e % 16 == 0); };
  const int eo = p.out_bf16 ? 2 : 4;
  p.vec = rows16(p.out, p.ldo, eo) && rows16(p.pre, p.ldp, eo) && rows16(p.residual, p.ldr, p.res_bf16 ? 2 : 4) &&
          at(p.bias, 16) && at(p.b_scale, 16);
  Choice c = choose(M, N, K, t_mn, esz, !p.out_bf16);
  const uint32_t force = g_force.load();
  if ((force & 255) == 1) c = Choice{(int)((force >> 8) & 0xFFFF), (int)(force >> 24)};
  else if ((force & 255) == 2) c = Choice{0, 1};
  if ((c.tile == 0 && K == 0) || (c.tile != 0 && t_mn && c.tile < 64)) return TFORGE_ERR_UNSUPPORTED;
  // f32 outputs: sums in pieces (of the pair kernel; the slim kernel divides its k by its accumulators).
  const int64_t stages = (K * esz + 127) / 128, piece = f8 ? 64 : 12;
  // The epilogue waits for a CTA's whole sum at once, which may well take longer than a stage may: 2^21
  // stages (K 2^30 on eight CTAs) 0.6 s, of a default limit of 1 s.  It gets the limit for each 2^14.
  const uint64_t times = 1 + (uint64_t)(stages / c.splits >> 14);
  p.sum_limit_ns = p.limit_ns > UINT64_MAX / times ? UINT64_MAX : p.limit_ns * times;
  p.sum_stages = !p.out_bf16 && stages > piece ? (int32_t)piece : 0;
  if (c.tile == 0) {
    CUtensorMap tmA{}, tmB{}, tmO{}, tmP{}, tmR{};
    const uint32_t bk = 128 / esz;
    rc = t_mn ? encode_mn_map(&tmA, rows.p, K, M, rows.ld, 2, &p.rows_blocks) : encode_rows_map(&tmA, rows.p, esz, M, K, rows.ld, bk, 128);
    if (!rc) rc = w_mn ? encode_mn_map(&tmB, cols.p, K, N, cols.ld, 2, &p.cols_blocks) : encode_rows_map(&tmB, cols.p, esz, N, K, cols.ld, bk, 128);
    if (!rc && p.vec) rc = encode_out_map(&tmO, p.out, p.out_bf16 != 0, M, N, p.ldo);
    if (!rc && p.vec && p.pre) rc = encode_out_map(&tmP, p.pre, p.out_bf16 != 0, M, N, p.ldp);
    if (!rc && p.vec && p.residual) rc = encode_out_map(&tmR, p.residual, p.res_bf16 != 0, M, N, p.ldr);
    if (rc) return rc;
    cudaError_t e = launch_linear_pair(f8, t_mn, w_mn, tmA, tmB, tmO, tmP, tmR, p, st);
    return e == cudaSuccess ? TFORGE_OK : cuda_failure(e, "linear launch");
  }
  p.splits = c.splits;
  CUtensorMap tmT{}, tmW{};
  if (K > 0) {
    const uint32_t bk = 128 / esz;
    rc = t_mn ? encode_mn_map(&tmT, rows.p, K, M, rows.ld, (uint32_t)c.tile / 64, &p.rows_blocks)
              : encode_rows_map(&tmT, rows.p, esz, M, K, rows.ld, bk, (uint32_t)c.tile);
    if (rc) return rc;
    rc = w_mn ? encode_mn_map(&tmW, cols.p, K, N, cols.ld, 2, &p.cols_blocks)
              : encode_rows_map(&tmW, cols.p, esz, N, K, cols.ld, bk, 128);
    if (rc) return rc;
  }
  cudaError_t e = launch_linear_slim(f8, w_mn, t_mn, c.tile, tmT, tmW, p, st);
  return e == cudaSuccess ? TFORGE_OK : cuda_failure(e, "linear launch");
}

// ---- the gradient's elementwise pass ---------------------------------------------------------------

// dz = dout * act'(pre) rounded to bf16 (dz null: not written), and part[b, n] = the f32 sum of the
// unrounded dz over row block b (part null: not wanted).  A block takes 256 columns (a lane eight:
// neighbouring ones with VEC, else 32 apart) of row block blockIdx.y, a warp every eighth row.  (Warps
// side by side on wider rows instead leave threads without columns: 6661 x 4264 bf16 with tanh gelu
// 15 us more, 4096 x 11008 too; 8192 x 16384 the same.)  Bound by HBM (reads two values and writes
// one an element) and the slope's arithmetic: 8192 x 16384 bf16 with tanh gelu 130 us, 6.2 TB/s.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    activation_grad_kernel(int act, const T *dout, int64_t lddo, const T *pre, int64_t ldp, __nv_bfloat16 *dz,
                           int64_t ldz, float *part, int64_t M, int64_t N) {
  grid_dependency_wait();
  grid_launch_dependents();
  constexpr int kWarps = 8;
  __shared__ float sm[kWarps][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c0 = (int64_t)blockIdx.x * 256;
  const int64_t per = (M + gridDim.y - 1) / gridDim.y, r0 = per * blockIdx.y, r1 = r0 + per < M ? r0 + per : M;
  auto off = [&](int j) { return VEC ? lane * 8 + j : j * 32 + lane; };
  float sum[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) sum[j] = 0.f;
  struct Raw {
    std::conditional_t<VEC, uint4, T> v[VEC ? (int)sizeof(T) / 2 : 8];
  };
  auto read = [&](const T *row, Raw &q) {
    if constexpr (VEC) {
#pragma unroll
      for (int h = 0; h < (int)sizeof(T) / 2; ++h)
        q.v[h] = c0 + lane * 8 < N ? reinterpret_cast<const uint4 *>(row + c0 + lane * 8)[h] : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) q.v[j] = c0 + off(j) < N ? row[c0 + off(j)] : T(0.f);
    }
  };
  auto value = [&](const Raw &q, int j) -> float {
    if constexpr (!VEC) {
      return (float)q.v[j];
    } else {
      constexpr int per16 = 16 / (int)sizeof(T);
      const uint4 &u = q.v[j / per16];
      const int k = j % per16 * (int)sizeof(T) / 4;
      const uint32_t w = k == 0 ? u.x : k == 1 ? u.y : k == 2 ? u.z : u.w;
      if constexpr (sizeof(T) == 4) return __uint_as_float(w);
      else return __uint_as_float(j % 2 ? w & 0xFFFF0000u : w << 16);
    }
  };
  with_activation(act, [&](auto a) {
    constexpr int ACT = decltype(a)::value;
    auto finish = [&](int64_t m, const Raw &d, const Raw &z) {
      float g[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g[j] = value(d, j);
        if constexpr (ACT != TFORGE_ACT_NONE) g[j] *= activate_slope<ACT>(value(z, j));
        sum[j] += g[j];
      }
      if (dz) {
        if constexpr (VEC) {
          if (c0 + lane * 8 < N)
            *reinterpret_cast<uint4 *>(dz + m * ldz + c0 + lane * 8) =
                make_uint4(pack_bf16x2(g[0], g[1]), pack_bf16x2(g[2], g[3]), pack_bf16x2(g[4], g[5]), pack_bf16x2(g[6], g[7]));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (c0 + off(j) < N) dz[m * ldz + c0 + off(j)] = __float2bfloat16_rn(g[j]);
        }
      }
    };
    // Two rows' loads in flight.
    int64_t m = r0 + warp;
    for (; m + kWarps < r1; m += 2 * kWarps) {
      Raw d[2], z[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        read(dout + (m + i * kWarps) * lddo, d[i]);
        if constexpr (ACT != TFORGE_ACT_NONE) read(pre + (m + i * kWarps) * ldp, z[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) finish(m + i * kWarps, d[i], z[i]);
    }
    if (m < r1) {
      Raw d, z;
      read(dout + m * lddo, d);
      if constexpr (ACT != TFORGE_ACT_NONE) read(pre + m * ldp, z);
      finish(m, d, z);
    }
  });
  if (!part) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) sm[warp][off(j)] = sum[j];
  __syncthreads();
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) v += sm[w][threadIdx.x];
  if (c0 + threadIdx.x < N) part[(int64_t)blockIdx.y * N + c0 + threadIdx.x] = v;
}

// Row blocks: eight blocks an SM in all (two rounds of resident ones), each of at least eight rows, a
// warp one.  At most 256: narrow matrices' block sums would take longer to add than to make.
int grad_row_blocks(int64_t M, int64_t N) {
  const int64_t cols = (N + 255) / 256, r = std::min<int64_t>(std::min<int64_t>(148 * 8 / cols, 256), (M + 7) / 8);
  return r < 1 ? 1 : (int)r;
}

template <typename T>
cudaError_t launch_activation_grad(int act, const void *dout, int64_t lddo, const void *pre, int64_t ldp, void *dz,
                                   int64_t ldz, float *part, int row_blocks, int64_t M, int64_t N, cudaStream_t st) {
  const int e = sizeof(T);
  const bool vec = N % 8 == 0 && at(dout, 16) && lddo * e % 16 == 0 &&
                   (act == TFORGE_ACT_NONE || (at(pre, 16) && ldp * e % 16 == 0));
  const dim3 g((unsigned)((N + 255) / 256), (unsigned)row_blocks);
  auto kern = vec ? activation_grad_kernel<T, true> : activation_grad_kernel<T, false>;
  return launch_dependent(kern, g, dim3(256), st, 0, act, static_cast<const T *>(dout), lddo, static_cast<const T *>(pre),
                          ldp, static_cast<__nv_bfloat16 *>(dz), ldz, part, M, N);
}

int check_linear_types(int act, int trans_b, int a_dtype, int b_dtype) {
  if (act < TFORGE_ACT_NONE || act > TFORGE_ACT_SILU || trans_b < 0 || trans_b > 1) return TFORGE_ERR_MODE;
  return is_float(a_dtype) && is_float(b_dtype) ? TFORGE_OK : TFORGE_ERR_MODE;
}

}  // namespace

extern "C" {

int tforge_linear(const tforge_linear_args *args, void *stream) {
  if (!args) return TFORGE_ERR_NULL;
  tforge_linear_args a = *args;
  const bool f8 = a.a_dtype == TFORGE_E4M3 && a.b_dtype == TFORGE_E4M3;
  int rc = f8 ? check_linear_types(a.activation, a.trans_b, TFORGE_BF16, TFORGE_BF16)
              : check_linear_types(a.activation, a.trans_b, a.a_dtype, a.b_dtype);
  if (rc) return rc;
  if (!is_float(a.out_dtype) || (a.residual && !is_float(a.residual_dtype))) return TFORGE_ERR_MODE;
  if (!f8 && (a.a_scale || a.b_scale)) return TFORGE_ERR_MODE;
  if (f8 && !a.trans_b) return TFORGE_ERR_UNSUPPORTED;
  if (!dims_ok(a.M, a.N, a.K)) return TFORGE_ERR_SHAPE;
  const int64_t brows = a.trans_b ? a.N : a.K, bcols = a.trans_b ? a.K : a.N;
  if (!pitch(a.lda, a.K) || !pitch(a.ldb, bcols) || !pitch(a.ldr, a.N, a.residual) || !pitch(a.ldo, a.N) ||
      !pitch(a.ldp, a.N, a.pre))
    return TFORGE_ERR_SHAPE;
  if (a.M == 0 || a.N == 0) return TFORGE_OK;
  if (!a.out || (a.K > 0 && (!a.A || !a.B)) || (f8 && (!a.a_scale || !a.b_scale))) return TFORGE_ERR_NULL;
  const int eo = elem_size(a.out_dtype);
  const Array ins[] = {{a.A, a.M, a.K, a.lda, elem_size(a.a_dtype)}, {a.B, brows, bcols, a.ldb, elem_size(a.b_dtype)},
                       {a.a_scale, 1, a.M, a.M, 4}, {a.b_scale, 1, a.N, a.N, 4}, {a.bias, 1, a.N, a.N, 4},
                       {a.residual, a.M, a.N, a.ldr, elem_size(a.residual_dtype)}};
  const Array outs[] = {{a.out, a.M, a.N, a.ldo, eo}, {a.pre, a.M, a.N, a.ldp, eo}};
  rc = check_arrays(ins, outs, 0, 5);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Scratch scratch(st);
  Operand A{a.A, a.M, a.K, a.lda}, B{a.B, brows, bcols, a.ldb};
  Copies copies;
  copies.add(A, a.a_dtype, scratch);
  copies.add(B, a.b_dtype, scratch);
  rc = scratch.take();
  if (!rc) rc = copies.run(scratch, st);
  if (rc) return rc;
  LinearParams p{};
  p.bias = a.bias;
  p.a_scale = a.a_scale;
  p.b_scale = a.b_scale;
  p.residual = a.residual;
  p.ldr = a.ldr;
  p.res_bf16 = a.residual_dtype == TFORGE_BF16;
  p.out = a.out;
  p.ldo = a.ldo;
  p.pre = a.pre;
  p.ldp = a.ldp;
  p.out_bf16 = a.out_dtype == TFORGE_BF16;
  p.act = a.activation;
  return product(A, false, B, !a.trans_b, f8, a.M, a.N, a.K, p, st);
}

int tforge_linear_backward(const tforge_linear_backward_args *args, void *stream) {
  if (!args) return TFORGE_ERR_NULL;
  tforge_linear_backward_args a = *args;
  int rc = check_linear_types(a.activation, a.trans_b, a.a_dtype, a.b_dtype);
  if (rc) return rc;
  if (!is_float(a.dtype) || !is_float(a.grad_dtype)) return TFORGE_ERR_MODE;
  if (!dims_ok(a.M, a.N, a.K)) return TFORGE_ERR_SHAPE;
  const int64_t brows = a.trans_b ? a.N : a.K, bcols = a.trans_b ? a.K : a.N;
  if (!pitch(a.lddo, a.N) || !pitch(a.ldp, a.N, a.pre && a.activation != TFORGE_ACT_NONE) || !pitch(a.lda, a.K, a.A && a.dB) ||
      !pitch(a.ldb, bcols, a.B && a.dA) || !pitch(a.ldda, a.K, a.dA) || !pitch(a.lddb, bcols, a.dB))
    return TFORGE_ERR_SHAPE;
  const bool want_a = a.dA && a.M > 0 && a.K > 0, want_b = a.dB && a.N > 0 && a.K > 0, want_bias = a.dbias && a.N > 0;
  if (!want_a && !want_b && !want_bias) return TFORGE_OK;
  const bool some = a.M > 0 && a.N > 0;  // else every sum is over nothing
  if (some && (!a.dout || (a.activation != TFORGE_ACT_NONE && !a.pre) || (want_a && !a.B) || (want_b && !a.A)))
    return TFORGE_ERR_NULL;
  const int ed = elem_size(a.dtype), eg = elem_size(a.grad_dtype);
  const Array ins[] = {{a.dout, a.M, a.N, a.lddo, ed},
                       {a.activation == TFORGE_ACT_NONE ? nullptr : a.pre, a.M, a.N, a.ldp, ed},
                       {want_b ? a.A : nullptr, a.M, a.K, a.lda, elem_size(a.a_dtype)},
                       {want_a ? a.B : nullptr, brows, bcols, a.ldb, elem_size(a.b_dtype)}};
  const Array outs[] = {{a.dA, a.M, a.K, a.ldda, eg}, {a.dB, brows, bcols, a.lddb, eg}, {a.dbias, 1, a.N, a.N, 4}};
  rc = check_arrays(ins, outs);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Scratch scratch(st);
  // dz and the column sums, unless dout serves as it is.
  Operand dz{a.dout, a.M, a.N, a.lddo}, A{a.A, a.M, a.K, a.lda}, B{a.B, brows, bcols, a.ldb};
  const bool need_dz = some && (want_a || want_b) &&
                       (a.activation != TFORGE_ACT_NONE || a.dtype == TFORGE_F32 || !at(a.dout, 16) || a.lddo % 8);
  const int rb = some ? grad_row_blocks(a.M, a.N) : 1;
  Copies copies;
  if (some && want_a) copies.add(B, a.b_dtype, scratch);
  if (some && want_b) copies.add(A, a.a_dtype, scratch);
  const uint64_t z_at = need_dz ? scratch.want((uint64_t)a.M * padded(a.N, 2) * 2) : 0;
  const uint64_t part_at = some && want_bias && rb > 1 ? scratch.want((uint64_t)rb * a.N * 4) : 0;
  rc = scratch.take();
  if (!rc) rc = copies.run(scratch, st);
  if (rc) return rc;
  if (need_dz) {
    dz.p = scratch.at(z_at);
    dz.ld = padded(a.N, 2);
  }
  if (some && (need_dz || want_bias)) {
    void *z = need_dz ? const_cast<void *>(dz.p) : nullptr;
    float *part = want_bias && rb > 1 ? reinterpret_cast<float *>(scratch.at(part_at)) : nullptr;
    float *sums = part ? part : (want_bias ? a.dbias : nullptr);
    cudaError_t e = a.dtype == TFORGE_BF16
                        ? launch_activation_grad<__nv_bfloat16>(a.activation, a.dout, a.lddo, a.pre, a.ldp, z, dz.ld, sums, rb, a.M, a.N, st)
                        : launch_activation_grad<float>(a.activation, a.dout, a.lddo, a.pre, a.ldp, z, dz.ld, sums, rb, a.M, a.N, st);
    if (e == cudaSuccess && part) e = launch_column_sum(part, rb, a.N, a.dbias, st);
    if (e != cudaSuccess) return cuda_failure(e, "activation gradient");
  } else if (want_bias) {
    cudaError_t e = cudaMemsetAsync(a.dbias, 0, (size_t)a.N * 4, st);
    if (e != cudaSuccess) return cuda_failure(e, "cudaMemsetAsync(dbias)");
  }
  LinearParams p{};
  p.act = TFORGE_ACT_NONE;
  p.out_bf16 = a.grad_dtype == TFORGE_BF16;
  if (want_a) {
    p.out = a.dA;
    p.ldo = a.ldda;
    rc = product(dz, false, B, a.trans_b != 0, false, a.M, a.K, a.N, p, st);
    if (rc) return rc;
  }
  if (want_b) {
    p.out = a.dB;
    p.ldo = a.lddb;
    rc = a.trans_b ? product(dz, true, A, true, false, a.N, a.K, a.M, p, st)
                   : product(A, true, dz, true, false, a.K, a.N, a.M, p, st);
    if (rc) return rc;
  }
  return TFORGE_OK;
}

int tforge_rms_norm(const tforge_rms_norm_args *args, void *stream) {
  if (!args) return TFORGE_ERR_NULL;
  tforge_rms_norm_args a = *args;
  if (!is_float(a.dtype) || (a.weight && !is_float(a.weight_dtype)) ||
      !(is_float(a.out_dtype) || a.out_dtype == TFORGE_E4M3))
    return TFORGE_ERR_MODE;
  if (!dims_ok(a.M, a.N) || !(a.eps >= 0.0f) || std::isinf(a.eps)) return TFORGE_ERR_SHAPE;
  if (!pitch(a.ldx, a.N) || !pitch(a.ldr, a.N, a.residual) || !pitch(a.lds, a.N, a.sum_out) || !pitch(a.ldo, a.N))
    return TFORGE_ERR_SHAPE;
  if (a.M == 0 || a.N == 0) return TFORGE_OK;
  if (!a.x || !a.out || (a.out_dtype == TFORGE_E4M3 && !a.scale)) return TFORGE_ERR_NULL;
  const int e = elem_size(a.dtype);
  const Array ins[] = {{a.x, a.M, a.N, a.ldx, e}, {a.residual, a.M, a.N, a.ldr, e},
                       {a.weight, 1, a.N, a.N, elem_size(a.weight_dtype)}};
  const Array outs[] = {{a.sum_out, a.M, a.N, a.lds, e}, {a.out, a.M, a.N, a.ldo, elem_size(a.out_dtype)},
                        {a.out_dtype == TFORGE_E4M3 ? a.scale : nullptr, 1, a.M, a.M, 4}, {a.rstd, 1, a.M, a.M, 4}};
  int rc = check_arrays(ins, outs, 0, 0, 1);
  if (rc) return rc;
  NormArgs p{};
  p.x = a.x;
  p.residual = a.residual;
  p.weight = a.weight;
  p.sum_out = a.sum_out;
  p.out = a.out;
  p.scale = a.scale;
  p.rstd = a.rstd;
  p.M = a.M;
  p.N = a.N;
  p.ldx = a.ldx;
  p.ldr = a.ldr;
  p.lds = a.lds;
  p.ldo = a.ldo;
  p.eps = a.eps;
  p.inv_n = 1.0f / (float)a.N;
  p.x_bf16 = a.dtype == TFORGE_BF16;
  p.w_bf16 = a.weight_dtype == TFORGE_BF16;
  p.out_kind = a.out_dtype;
  cudaError_t err = launch_rms_norm(p, true, static_cast<cudaStream_t>(stream));
  return err == cudaSuccess ? TFORGE_OK : cuda_failure(err, "rms_norm launch");
}

int tforge_rms_norm_backward(const tforge_rms_norm_backward_args *args, void *stream) {
  if (!args) return TFORGE_ERR_NULL;
  tforge_rms_norm_backward_args a = *args;
  if (!is_float(a.dtype) || (a.weight && !is_float(a.weight_dtype))) return TFORGE_ERR_MODE;
  if (!dims_ok(a.M, a.N)) return TFORGE_ERR_SHAPE;
  if (!pitch(a.lddy, a.N) || !pitch(a.lds, a.N) || !pitch(a.ldds, a.N, a.ds) || !pitch(a.lddx, a.N))
    return TFORGE_ERR_SHAPE;
  if (a.N == 0) return TFORGE_OK;
  if (a.M > 0 && (!a.dy || !a.s || !a.rstd || !a.dx)) return TFORGE_ERR_NULL;
  const int e = elem_size(a.dtype);
  const Array ins[] = {{a.dy, a.M, a.N, a.lddy, e}, {a.s, a.M, a.N, a.lds, e},
                       {a.weight, 1, a.N, a.N, elem_size(a.weight_dtype)}, {a.rstd, 1, a.M, a.M, 4}, {a.ds, a.M, a.N, a.ldds, e}};
  const Array outs[] = {{a.dx, a.M, a.N, a.lddx, e}, {a.dweight, 1, a.N, a.N, 4}};
  int rc = check_arrays(ins, outs, 0, 4);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.M == 0) {
    cudaError_t err = a.dweight ? cudaMemsetAsync(a.dweight, 0, (size_t)a.N * 4, st) : cudaSuccess;
    return err == cudaSuccess ? TFORGE_OK : cuda_failure(err, "cudaMemsetAsync(dweight)");
  }
  NormBwdArgs p{};
  p.dy = a.dy;
  p.s = a.s;
  p.weight = a.weight;
  p.ds = a.ds;
  p.rstd = a.rstd;
  p.dx = a.dx;
  p.M = a.M;
  p.N = a.N;
  p.lddy = a.lddy;
  p.lds = a.lds;
  p.ldds = a.ldds;
  p.lddx = a.lddx;
  p.inv_n = 1.0f / (float)a.N;
  p.x_bf16 = a.dtype == TFORGE_BF16;
  p.w_bf16 = a.weight_dtype == TFORGE_BF16;
  const int parts = rms_norm_bwd_blocks(p);
  Scratch scratch(st);
  const bool join = a.dweight && parts > 1;
  const uint64_t part_at = join ? scratch.want((uint64_t)parts * a.N * 4) : 0;
  rc = scratch.take();
  if (rc) return rc;
  float *part = join ? reinterpret_cast<float *>(scratch.at(part_at)) : nullptr;
  float *sums = part ? part : a.dweight;
  cudaError_t err = launch_rms_norm_bwd(p, sums, parts, st);
  if (err == cudaSuccess && part) err = launch_column_sum(part, parts, a.N, a.dweight, st);
  return err == cudaSuccess ? TFORGE_OK : cuda_failure(err, "rms_norm_backward launch");
}

int tforge_quantize_e4m3(const void *x, int dtype, uint8_t *q, float *scale, int64_t M, int64_t N, int64_t ldx,
                         int64_t ldq, void *stream) {
  if (!is_float(dtype)) return TFORGE_ERR_MODE;
  if (!dims_ok(M, N) || !pitch(ldx, N) || !pitch(ldq, N)) return TFORGE_ERR_SHAPE;
  if (M == 0 || N == 0) return TFORGE_OK;
  if (!x || !q || !scale) return TFORGE_ERR_NULL;
  const Array ins[] = {{x, M, N, ldx, elem_size(dtype)}};
  const Array outs[] = {{q, M, N, ldq, 1}, {scale, 1, M, M, 4}};
  int rc = check_arrays(ins, outs);
  if (rc) return rc;
  NormArgs p{};
  p.x = x;
  p.out = q;
  p.scale = scale;
  p.M = M;
  p.N = N;
  p.ldx = ldx;
  p.ldo = ldq;
  p.x_bf16 = dtype == TFORGE_BF16;
  p.out_kind = TFORGE_E4M3;
  cudaError_t err = launch_rms_norm(p, false, static_cast<cudaStream_t>(stream));
  return err == cudaSuccess ? TFORGE_OK : cuda_failure(err, "quantize_e4m3 launch");
}

int tforge_debug_linear_kernel(int kernel, int tile, int splits) {
  const bool tile_ok = tile == 16 || tile == 32 || tile == 64 || tile == 128 || tile == 256;
  const bool split_ok = splits == 1 || splits == 2 || splits == 4 || splits == 8;
  if (kernel < 0 || kernel > 2 || (kernel == 1 && (!tile_ok || !split_ok))) return TFORGE_ERR_MODE;
  g_force.store(kernel == 1 ? 1u | (uint32_t)tile << 8 | (uint32_t)splits << 24 : (uint32_t)kernel);
  return TFORGE_OK;
}

}  // extern "C"
