/*
 * tforge.h -- C-ABI of the B200 (sm_100a) TensorForge operator library.
 *
 * Drop-in for the kernel that TensorForge's `--tforge-gpu-pipeline` generates and that
 * runners/gpu/tforge-gpu-bench.cu launches with cuLaunchKernel. The argument order is
 * the MLIR host entry's out-param order, `entry(A, B, bias, out)`:
 *   matmul:   A (M x K), B (K x N), out (M x N)            runners/gpu/tforge-gpu-bench.cu:20-24
 *   mbr:      A, B, bias (N), out                          runners/gpu/tforge-gpu-bench.cu:209-213
 *   bias_add: X (M x N), bias (N), Y                       python/tforge_cpu.py:3-8
 *   relu:     X, Y
 * All tensors are row-major contiguous f32 in device memory, owned by the caller,
 * distinct and non-overlapping (the reference marks every kernel pointer `noalias`,
 * lib/Transforms/Gpu.cpp:453-457). The library allocates no input or output buffers
 * and never copies them. Every call is asynchronous on `stream` (a cudaStream_t; NULL
 * is the legacy default stream) and returns a status code; it never exits the process
 * (the reference runner's die() + exit(1), tforge-gpu-bench.cu:52-70, becomes a code).
 *
 * Op semantics (include/TensorForge/Dialect/TForge/TForgeOps.td:37-113):
 *   matmul   C[m,n] = sum_k A[m,k] * B[k,n], accumulator starts at +0.0, K order unspecified
 *   bias_add Y[m,n] = X[m,n] + bias[n]            (one IEEE add)
 *   relu     Y = maximum(X, +0.0)                  (IEEE-2019: NaN -> NaN, -0.0 -> +0.0)
 *   add      Z = X + Y                             (one IEEE add)
 *   mbr      relu(bias_add(matmul(A, B), bias))    fused in one kernel
 *   matmul_add  matmul(A, B) + C_res               fused in one kernel
 */
#ifndef TFORGE_H
#define TFORGE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. */
enum tforge_status {
  TFORGE_OK = 0,
  TFORGE_ERR_SHAPE = 1,       /* M, N or K negative, or a pitch smaller than its row */
  TFORGE_ERR_ALIGN = 2,       /* a pointer not 4-byte aligned (f32) */
  TFORGE_ERR_ALIAS = 3,       /* the output overlaps an input */
  TFORGE_ERR_MODE = 4,        /* unknown precision mode or workload */
  TFORGE_ERR_CUDA = 5,        /* a CUDA runtime/driver call failed; see tforge_last_error() */
  TFORGE_ERR_TIMEOUT = 6,     /* a bounded device-side wait expired (reported by tforge_device_status) */
  TFORGE_ERR_NULL = 7,        /* a required pointer is NULL */
  TFORGE_ERR_UNSUPPORTED = 8, /* no kernel for this combination (e.g. a forced config that cannot run) */
  TFORGE_ERR_NOMEM = 9        /* the library's own workspace could not be allocated */
};

/* Precision modes of the GEMM kernels. */
enum tforge_mode {
  TFORGE_MODE_FP32 = 0,       /* fp32-accurate: 3xTF32 split products on tcgen05 (default) */
  TFORGE_MODE_TF32 = 1,       /* one TF32 product on tcgen05 (inputs rounded to 10-bit mantissa) */
  TFORGE_MODE_BF16 = 2,       /* inputs rounded to bf16, fp32 accumulation on tcgen05 */
  TFORGE_MODE_FP32_EXACT = 3  /* SIMT FFMA, sequential k from +0.0: bitwise equal to the reference's
                                 generated kernels (docs/numerics.md:3,53) */
};

/* Workloads (python/tforge_cpu.py:3-8 plus matmul_add). */
enum tforge_workload {
  TFORGE_MATMUL = 0,
  TFORGE_MBR = 1,
  TFORGE_MATMUL_ADD = 2,
  TFORGE_BIAS_ADD = 3,
  TFORGE_RELU = 4,
  TFORGE_ADD = 5
};

/* Element types.  tforge_gemm takes f32 and bf16; E4M3 (8 bits: sign, 4 exponent and 3 mantissa
 * bits, largest 448) is an operand type of tforge_linear and an output type of tforge_rms_norm
 * and tforge_quantize_e4m3. */
enum tforge_dtype { TFORGE_F32 = 0, TFORGE_BF16 = 1, TFORGE_E4M3 = 2 };

/* Activations of tforge_linear.  GELU is z Phi(z) with the normal distribution's Phi; GELU_TANH its
 * tanh form, z (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3))) / 2; SILU z / (1 + exp(-z)). */
enum tforge_activation {
  TFORGE_ACT_NONE = 0,
  TFORGE_ACT_RELU = 1,
  TFORGE_ACT_GELU = 2,
  TFORGE_ACT_GELU_TANH = 3,
  TFORGE_ACT_SILU = 4
};

/* Fused GEMM.  out = epilogue(A @ B).  Replaces the generated `entry_kernel` of the
 * tforge-gpu-pipeline (lib/Transforms/Gpu.cpp:219-316) launched at
 * runners/gpu/tforge-gpu-bench.cu:292-302.  Pitches are in elements; 0 means packed
 * (lda = K, ldb = N, ldc = N; C_res shares ldc).  BF16 A/B are accepted only in
 * TFORGE_MODE_BF16 (inputs already converted, e.g. a weight converted once).
 * out_dtype TFORGE_BF16 (TFORGE_MODE_BF16 only; not in tforge_gemm_host): out holds M x N
 * bf16 values, the f32 results rounded to nearest even -- the same values tforge_convert_bf16
 * of the f32 output gives, written without the f32 round trip (a hidden layer feeding a
 * BF16-mode layer, e.g. the MLP chain's H). */
typedef struct tforge_gemm_args {
  int32_t workload;      /* TFORGE_MATMUL, TFORGE_MBR or TFORGE_MATMUL_ADD */
  int32_t mode;          /* enum tforge_mode */
  int32_t a_dtype;       /* enum tforge_dtype */
  int32_t b_dtype;       /* enum tforge_dtype */
  const void *A;         /* M x K */
  const void *B;         /* K x N */
  const float *bias;     /* N        (mbr) */
  const float *C_res;    /* M x N    (matmul_add) */
  void *out;             /* M x N, f32 (or bf16, see out_dtype) */
  int64_t M, N, K;
  int64_t lda, ldb, ldc;
  int32_t out_dtype;     /* enum tforge_dtype; 0 = TFORGE_F32 */
} tforge_gemm_args;

int tforge_gemm(const tforge_gemm_args *args, void *stream);

/* tforge_gemm on HOST buffers: args->A, B, bias / C_res and out are host pointers (pitches as in
 * tforge_gemm).  Replaces the GPU runner's host flow -- cudaMalloc, cudaMemcpy of A, B and bias
 * to the device, the launch, cudaMemcpy of C back (runners/gpu/tforge-gpu-bench.cu:198-207,
 * 292-302,327) -- with an overlapped one: device staging comes from the library's pool; B and
 * bias are copied first, then A (and C_res) in chunks of `chunk_rows` rows (0: automatic, at
 * most 8 chunks of at least 512 rows); each chunk's kernel starts on its own stream once its
 * rows have landed, and each chunk of out is copied back while later chunks compute.
 * Asynchronous with respect to the host: out is complete once `stream` has synchronized.  Copies overlap only
 * with page-locked host memory; pageable memory gives the same results without overlap.
 * Results equal tforge_gemm's on each chunk of rows (the kernel is chosen per chunk). */
int tforge_gemm_host(const tforge_gemm_args *args, int64_t chunk_rows, void *stream);

/* The three operator entries, in the reference's host-entry argument order. */
int tforge_matmul(const float *A, const float *B, float *out, int64_t M, int64_t N, int64_t K,
                  int mode, void *stream);
int tforge_mbr(const float *A, const float *B, const float *bias, float *out, int64_t M, int64_t N,
               int64_t K, int mode, void *stream);
int tforge_matmul_add(const float *A, const float *B, const float *C_res, float *out, int64_t M,
                      int64_t N, int64_t K, int mode, void *stream);

/* Elementwise ops, bit-exact (one IEEE operation per element): the GPU runner's
 * bias_add / relu workloads (runners/gpu/tforge-gpu-bench.cu:127-130) and the CPU
 * runner's add (runners/cpu/tforge-cpu-bench.cpp:214-219). */
int tforge_bias_add(const float *X, const float *bias, float *Y, int64_t M, int64_t N, void *stream);
int tforge_relu(const float *X, float *Y, int64_t M, int64_t N, void *stream);
int tforge_add(const float *X, const float *Y, float *Z, int64_t M, int64_t N, void *stream);

/* Round f32 to bf16 (round to nearest even), n elements: converts a weight once for
 * repeated TFORGE_MODE_BF16 calls with b_dtype = TFORGE_BF16. */
int tforge_convert_bf16(const float *x, uint16_t *y, int64_t n, void *stream);

/* ---- transformer-layer operators --------------------------------------------------------------
 * All asynchronous on `stream`, which belongs to the current device, as all pointers do.  Pitches
 * are in elements, 0 = packed; those of arrays that are not there are not looked at.  Any size up to 2^30, any pitch and any element-aligned pointer works;
 * rows that start on 16-byte boundaries save an operand's copy (tforge_linear) or take wider
 * accesses.  An output may not overlap another output or an input, but where its entry says so
 * (else TFORGE_ERR_ALIAS); column slices of one buffer do not overlap.  M = 0 or N = 0 is a no-op
 * but for the gradients' sums over no rows, which are zeros.  Scratch comes from the library's
 * stream-ordered pool. */

/* The linear layer with its epilogue:
 *   z = (A @ B) * a_scale[m] * b_scale[n] + bias[n];  out = act(z) + residual;  pre = z
 * A is M x K; B is K x N, or N x K with trans_b = 1 (a row per output feature).  Operands: bf16 or
 * f32 (rounded to bf16, as TFORGE_MODE_BF16 does), or both E4M3 with f32 scales a row of A and a
 * column of B, as tforge_rms_norm and tforge_quantize_e4m3 write them (then trans_b = 1).  Products
 * are accumulated and the epilogue computed in f32, and each output is rounded once.  bias, residual
 * and pre may be NULL; pre has out's type.  out may be the residual itself (same pointer, pitch and
 * type): a residual stream updated in place.  K = 0 gives z = bias. */
typedef struct tforge_linear_args {
  int32_t activation;      /* enum tforge_activation */
  int32_t trans_b;         /* 0: B is K x N; 1: N x K */
  int32_t a_dtype;         /* enum tforge_dtype */
  int32_t b_dtype;
  int32_t out_dtype;       /* TFORGE_F32 or TFORGE_BF16: out and pre */
  int32_t residual_dtype;  /* TFORGE_F32 or TFORGE_BF16 */
  const void *A;
  const void *B;
  const float *a_scale;    /* M (E4M3) */
  const float *b_scale;    /* N (E4M3) */
  const float *bias;       /* N or NULL */
  const void *residual;    /* M x N or NULL */
  void *out;               /* M x N */
  void *pre;               /* M x N or NULL */
  int64_t M, N, K;
  int64_t lda, ldb, ldr, ldo, ldp;
} tforge_linear_args;

int tforge_linear(const tforge_linear_args *args, void *stream);

/* The linear layer's gradient.  With dz = dout * act'(pre):
 *   dA = dz @ B^T (M x K);  dB = A^T @ dz (laid out as B);  dbias[n] = sum over m of dz[m, n]
 * The residual's gradient is dout itself.  dA, dB and dbias may each be NULL (not wanted).  A and B
 * are bf16 or f32 (rounded to bf16); dz is rounded to bf16 for the two products, dbias sums it
 * unrounded, in f32 and in a fixed order.  pre is needed but for TFORGE_ACT_NONE. */
typedef struct tforge_linear_backward_args {
  int32_t activation;
  int32_t trans_b;
  int32_t a_dtype;         /* TFORGE_F32 or TFORGE_BF16 */
  int32_t b_dtype;
  int32_t dtype;           /* TFORGE_F32 or TFORGE_BF16: dout and pre */
  int32_t grad_dtype;      /* TFORGE_F32 or TFORGE_BF16: dA and dB */
  const void *dout;        /* M x N */
  const void *pre;         /* M x N */
  const void *A;           /* M x K */
  const void *B;
  void *dA;
  void *dB;
  float *dbias;            /* N */
  int64_t M, N, K;
  int64_t lddo, ldp, lda, ldb, ldda, lddb;
} tforge_linear_backward_args;

int tforge_linear_backward(const tforge_linear_backward_args *args, void *stream);

/* Root-mean-square norm of rows, with the residual's addition before it:
 *   s = x + residual (sum_out = s);  r = (mean(s^2) + eps)^-1/2 (rstd = r);  out = s r weight
 * in f32 (squares beyond its range make r 0), each output rounded once.  out is f32, bf16 or E4M3;
 * E4M3 rows come with scale[m] = max(max|out| / 448, 2^-126), the f32 factor back to out's values, and
 * hold e4m3(out * (1 / scale[m])), the reciprocal and the product each rounded to f32; a row that holds
 * a NaN, or an infinity in s, has a NaN scale and NaN values.  residual, weight (1), sum_out, rstd may
 * be NULL.
 * sum_out may be x or the residual itself (same pointer and pitch). */
typedef struct tforge_rms_norm_args {
  int32_t dtype;           /* TFORGE_F32 or TFORGE_BF16: x, residual, sum_out */
  int32_t weight_dtype;    /* TFORGE_F32 or TFORGE_BF16 */
  int32_t out_dtype;
  float eps;               /* >= 0 */
  const void *x;           /* M x N */
  const void *residual;    /* M x N or NULL */
  const void *weight;      /* N or NULL */
  void *sum_out;           /* M x N or NULL */
  void *out;               /* M x N */
  float *scale;            /* M (E4M3) */
  float *rstd;             /* M or NULL */
  int64_t M, N;
  int64_t ldx, ldr, lds, ldo;
} tforge_rms_norm_args;

int tforge_rms_norm(const tforge_rms_norm_args *args, void *stream);

/* The norm's gradient, from s and rstd as the forward call gave them and out's gradient dy.  With
 * h = s rstd and g = dy weight:
 *   dx = rstd (g - h mean(g h)) + ds;  dweight[n] = sum over m of dy[m, n] h[m, n]
 * dx is the gradient of x and of the residual alike; ds (may be NULL) is what reaches s on the
 * residual stream, and dx may be ds itself (same pointer and pitch).  dweight may be NULL; it is
 * summed in f32 and in a fixed order. */
typedef struct tforge_rms_norm_backward_args {
  int32_t dtype;           /* TFORGE_F32 or TFORGE_BF16: dy, s, ds, dx */
  int32_t weight_dtype;    /* TFORGE_F32 or TFORGE_BF16 */
  const void *dy;          /* M x N */
  const void *s;           /* M x N */
  const void *weight;      /* N or NULL */
  const float *rstd;       /* M */
  const void *ds;          /* M x N or NULL */
  void *dx;                /* M x N */
  float *dweight;          /* N or NULL */
  int64_t M, N;
  int64_t lddy, lds, ldds, lddx;
} tforge_rms_norm_backward_args;

int tforge_rms_norm_backward(const tforge_rms_norm_backward_args *args, void *stream);

/* Rows of f32 or bf16 x (M x N, pitch ldx) in 8 bits: scale[m] = max(max|x[m]| / 448, 2^-126),
 * q = e4m3(x * (1 / scale[m])) (pitch ldq), the reciprocal and the product each rounded to f32.
 * Weights (N x K) are quantized once, activations before a product that tforge_rms_norm does not
 * feed.  NaN and infinities as in tforge_rms_norm. */
int tforge_quantize_e4m3(const void *x, int dtype, uint8_t *q, float *scale, int64_t M, int64_t N, int64_t ldx,
                         int64_t ldq, void *stream);

/* relu(A @ B + bias) in TFORGE_MODE_BF16 without allocating anything.  No counterpart in
 * the reference.  For callers that must not allocate device memory during a call (a
 * serving loop that reserves all of its memory up front and cannot risk an out-of-memory
 * error or an allocator synchronisation mid-request, or a host framework that owns every
 * device byte).  The f32 -> bf16 operand copies go to a 16 MiB static device array that
 * every GPU loading this library keeps until exit: bf16(A) (rounded up to 256 bytes) plus
 * bf16(B) must fit in 16 MiB (e.g. M = N = K = 2048), else TFORGE_ERR_SHAPE.  Needs K and
 * N multiples of 8 and 16-byte-aligned pointers (else TFORGE_ERR_UNSUPPORTED /
 * TFORGE_ERR_ALIGN).  Calls share the array: calls that overlap on the GPU race.  The
 * first call on a device resolves the array's address; make it before any stream capture. */
int tforge_mbr_bf16_noalloc(const float *A, const float *B, const float *bias, float *out, int64_t M,
                            int64_t N, int64_t K, void *stream);

/* Launch description: replaces the `tforge.launch = {kernel, grid, block, args}`
 * module attribute (lib/Transforms/Gpu.cpp:449-457,572-577) that python/tforge_gpu.py
 * parses into launch.json (:42-51,88-90).  Filled for the kernel the dispatch table
 * picks for (workload, M, N, K, mode) without launching anything. */
typedef struct tforge_launch {
  char kernel[64];       /* kernel family name */
  int32_t grid[3];
  int32_t block[3];
  int32_t cluster[3];
  int32_t smem_bytes;    /* dynamic shared memory per CTA */
  int32_t tile[3];       /* BM, BN, BK (K elements per pipeline stage) */
  int32_t stages;
  int32_t tmem_cols;     /* tensor-memory columns per CTA (0 for SIMT kernels) */
  int32_t mode;          /* the precision mode that will run */
  int32_t persistent;    /* 1 if CTAs loop over tiles */
  int32_t split_k;
  int32_t regs;          /* registers per thread (-1 without a device) */
  int32_t static_smem;   /* static shared memory per CTA (-1 without a device) */
  int32_t blocks_per_sm; /* resident CTAs per SM from the occupancy API (-1 without a device) */
} tforge_launch;

int tforge_describe(int workload, int64_t M, int64_t N, int64_t K, int mode, tforge_launch *out);

/* Force a kernel configuration (offline tuning sweeps); NULL restores the table. */
typedef struct tforge_config {
  int32_t kernel;        /* 0 = table, 1 = tcgen05 one CTA per tile, 2 = SIMT, 3 = tcgen05 CTA pair */
  int32_t bn;            /* 64, 128 or 256 (one-CTA kernel); 256 or 240 (CTA pair) */
  int32_t stages;
  int32_t persistent;    /* 1 with kernel = 3: persistent CTA-pair kernel (TF32 / BF16 modes,
                            256x256 tiles, two TMEM accumulators, no split-K) */
  int32_t split_k;       /* CTA-pair kernel in fp32 / TF32 mode: 0 = automatic, 1 = no split,
                            S = 2..8 pairs per tile, each over K / S */
  int32_t b_layout;      /* TF32 mode, 256-wide pair and persistent pair kernels: 0 or 1 = B as
                            given, loaded as k-group-major tiles (one 4-D box per tile) when N is
                            a multiple of 32 and K of 4, else in 128-byte column blocks; 2 = a
                            transposed, K-major copy of B (one extra pass over B); 3 = B as given
                            in column blocks.  Every form gives the same bits. */
} tforge_config;

int tforge_set_config(const tforge_config *cfg);

/* Synchronizes `stream`, then returns and clears the current device's status words that
 * bounded waits write on expiry (TFORGE_OK or TFORGE_ERR_TIMEOUT): the one of the GEMM
 * entries and the one of tforge_mbr_bf16_noalloc.  Allocates nothing.  TFORGE_ERR_CUDA if
 * the synchronization itself failed. */
int tforge_device_status(void *stream);

/* Device-side wait limit in nanoseconds (default 1e9); 0 restores the default.  The wait for one of
 * tforge_linear's sums over a long k gets it again for each 2^20 of k (bf16; 2^21 e4m3). */
int tforge_set_wait_limit_ns(uint64_t ns);

/* Test hook: 1 makes the next GEMM launches' producer skip its first stage's load, so
 * the consumer's bounded wait expires and reports TFORGE_ERR_TIMEOUT; 0 clears. */
int tforge_debug_skip_load(int on);

/* Test hook: the kernel that tforge_linear's and tforge_linear_backward's products take.  kernel 0:
 * chosen by size; 1: one CTA per 128 columns x `tile` rows (16, 32, 64, 128 or 256), `splits` CTAs
 * (1, 2, 4 or 8) sharing a tile's K; 2: persistent CTA pairs on 256 x 256 tiles.  A forced kernel that cannot take a product gives
 * TFORGE_ERR_UNSUPPORTED. */
int tforge_debug_linear_kernel(int kernel, int tile, int splits);

/* Test hook: bytes of the library's scratch pool in use now and the high-water mark since
 * the last reset (reset_high = 1 resets it after reading).  Creates the pool if the
 * device has none yet. */
int tforge_debug_pool_usage(uint64_t *used_now, uint64_t *used_high, int reset_high);

const char *tforge_status_string(int status);
const char *tforge_last_error(void);   /* text of the last TFORGE_ERR_CUDA, per thread */
const char *tforge_version(void);

/* Minimal device-memory helpers for callers without a CUDA binding (the ctypes shim). */
int tforge_malloc(void **ptr, uint64_t bytes);
int tforge_free(void *ptr);
int tforge_memcpy_h2d(void *dst, const void *src, uint64_t bytes, void *stream);
int tforge_memcpy_d2h(void *dst, const void *src, uint64_t bytes, void *stream);
int tforge_memset(void *dst, int byte, uint64_t bytes, void *stream);
int tforge_stream_sync(void *stream);
int tforge_device_count(int *n);
int tforge_set_device(int dev);

#ifdef __cplusplus
}
#endif

#endif /* TFORGE_H */
