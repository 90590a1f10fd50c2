/*
 * hipgemm -- C ABI of the MI355X (gfx950) FP8 GEMM.
 *
 *   C[M x N] = bf16_rne( (scale_a * scale_b) * sum_k A[m, k] * B_T[n, k] )
 *
 * A is M x K, row-major, e4m3 (OCP E4M3FN, one byte), row stride lda bytes.
 * B_T is N x K, row-major (K contiguous), e4m3, row stride ldb bytes.
 * C is M x N, row-major, bf16, row stride ldc elements.
 * (hipgemm_gemm generalises this: e5m2 operands, fp16 output, row / column
 * scales, bias and activation; see hipgemm_gemm_desc.)
 * Accumulation is fp32.  scale_a / scale_b are DEVICE pointers to one fp32
 * each (per-tensor scales), or NULL for 1.0; the product scale_a * scale_b is
 * formed in fp32 and applied to the fp32 accumulator before rounding.
 *
 * The reference (nirw4nna/hipgemm) exposes only a C++ kernel template,
 * fp8_gemm_4wave_256x256x128<M, N, K>(A, B_T, C) (fp8_4wave.hpp:334-338),
 * launched by its callers as <<<(M*N)/65536, 256>>> on the null stream
 * (test.cpp:79, bench.cpp:55, bench.cpp:78).  That surface is kept in
 * include/hipgemm/fp8_gemm.hpp; these entry points are the plain-pointer
 * boundary over it.  Plain pointers and sizes only.
 *
 * Errors: every entry point returns a hipError_t and never exits the
 * process.  Argument errors return hipErrorInvalidValue before any HIP call,
 * so they can be checked on a machine without a GPU.  Requirements:
 *   M, N, K >= 0;  C non-NULL, 2-byte aligned, N <= ldc <= 2^22;
 *   A, B_T non-NULL and 16-byte aligned;  K % 16 == 0;
 *   lda >= K, ldb >= K, lda % 16 == 0, ldb % 16 == 0, lda, ldb <= 2^23.
 * M == 0 or N == 0 is a no-op (nothing is checked or written).  K == 0
 * writes bf16(0 * scale) everywhere and neither reads nor checks A, B_T,
 * lda, ldb.
 * Nothing outside the M x N window of C is written.
 *
 * Threading: no global mutable state; calls on different streams may run
 * concurrently as long as their C windows do not overlap.
 */
#ifndef HIPGEMM_H
#define HIPGEMM_H

#include <hip/hip_runtime_api.h>
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HIPGEMM_VERSION 100 /* 1.0.0 */

/* Workspace layout (every schedule): the first HIPGEMM_WS_COUNTER_BYTES
 * bytes hold arrival counters that must be zero before a workspace's first
 * use; every call leaves them zero again and writes nothing else there.
 * Partial tiles follow; calls overwrite them before reading them.  So one
 * workspace serves calls of every shape and schedule in turn. */
#define HIPGEMM_WS_COUNTER_BYTES 16384

/* Schedules.  AUTO names one by shape (hipgemm_select_variant: "AUTO's choice"
 * below) and runs it, except that 8-bit operands without MX scales from 33 rows
 * up run on another tile of the 128 x 128 schedule's loop where one is estimated
 * faster (hipgemm_auto_tile: most calls from 33 to 128 rows and many above; so
 * SKINNY seldom runs but where those tiles are not built, or for fp32 and e4m3
 * outputs with few columns and long rows). */
enum {
  HIPGEMM_VARIANT_AUTO = 0,
  /* 256 threads (4 waves, one per SIMD), 256 x 256 tile, 2 LDS stages,
   * persistent grid, v_mfma_f32_32x32x64_f8f6f4. */
  HIPGEMM_VARIANT_4WAVE = 1,
  /* The same schedule on v_mfma_f32_16x16x128_f8f6f4: AUTO's choice for
   * M > 128 when the 256 x 256 tiles fill the CUs (but see TILE128 and
   * hipgemm_split_columns), and the schedule behind the drop-in
   * template. */
  HIPGEMM_VARIANT_4WAVE_MFMA16 = 2,
  /* M <= 128 only: split-K over every CU for the HBM-bound skinny shapes,
   * operands streamed straight into registers, a deterministic in-kernel
   * reduction of the K-slices.  AUTO's choice for 64 < M <= 128 only where
   * B_T exceeds 8 MiB and the 128 x 128 schedule's K-split would leave at
   * least half the CUs idle in 3 slices or more, for N >= 2048 (e.g.
   * 128 x 4096 x 4096; not 128 x 8192 x 2048).  Needs a workspace (hipgemm_workspace_size) when
   * it splits K. */
  HIPGEMM_VARIANT_SKINNY = 3,
  /* 512 threads (8 waves, two per SIMD, in two groups that alternate
   * between LDS/DMA work and MFMAs), 256 x 256 tile, each wave 128 x 64 of
   * it, persistent grid, v_mfma_f32_16x16x128_f8f6f4.  Never AUTO's
   * choice (3-7 % behind the 4-wave one from 2048 x 4096 up, behind the
   * 128 x 128 one below).  The reference's kernels are 4-wave only; no
   * reference counterpart. */
  HIPGEMM_VARIANT_8WAVE = 4,
  /* 256 threads (4 waves, one per SIMD), 128 x 128 tile, each wave 64 x 64
   * of it, 4 LDS stages, persistent grid, v_mfma_f32_16x16x128_f8f6f4: four
   * times as many tiles as the 256 x 256 schedules, for shapes whose 256 x
   * 256 tiles underfill the CUs: AUTO's choice for M > 128 when its tiles
   * fit in one round over the CUs, or in less than two where the 256 x 256
   * ones fill at most half of them (unless M or N >= 8192 and K >= 4096), or
   * for K <= 2048 on at most 128 tiles of 256 x 256, for 64 < M <= 128
   * (except as under STRIP and SKINNY), and for 16 < M <= 64 where N > 64 x
   * CUs, above 32 rows where K <= 1024 (unless N / 32 lies in (CUs / 4,
   * CUs]), or above 48 rows where K > 8192 and N >= 3072. The workgroups
   * of each XCD start their K walk at their own step (a different order of
   * the fp32 sums per XCD). Splits K into slices when its tiles fill at most a
   * quarter of the CUs and K has at least 16 steps of 128 bytes, or at most
   * half of them and K has at least 64 steps (CUs / tiles slices: 2, or 3
   * for 65-85 tiles on 256 CUs); a workspace then (hipgemm_workspace_size).
   * With a caller's workspace (or hipgemm_gemm_noalloc), the per-tensor
   * epilogue, no MX scales and at most 4 slices, the slice that finishes a
   * 64 x 64 quadrant last sums it in the same kernel (arrival counters in
   * the workspace); else a second kernel sums the slices. A call with no
   * workspace under stream capture runs unsplit (as do the split-K and strip
   * schedules' calls there). No reference counterpart (the reference has 256
   * x 256 tiles only). */
  HIPGEMM_VARIANT_TILE128 = 5,
  /* M <= 128 only: 256 threads, each workgroup a strip of 32 columns of C
   * (64 from 17 rows when 32-column strips would outnumber the CUs, and
   * for some long-K shapes above 40 rows) over all of K (over a K-slice,
   * with a workspace, when the strips alone are fewer than the CUs; at most
   * one workgroup per CU), its 4 waves each a quarter of the K-steps,
   * summed in LDS; B_T streamed by whole-line DMA into LDS, A straight into
   * registers (through LDS as well for 17-32 rows on 32-column strips).
   * AUTO's choice for M <= 64 except where TILE128 is, and for
   * 64 < M <= 128 with a B_T of at most 8 MiB.  No reference
   * counterpart. */
  HIPGEMM_VARIANT_STRIP = 6,
  HIPGEMM_VARIANT_COUNT = 7
};

/* Operand formats (OCP 8-bit floating point v1.0; OCP Microscaling v1.0
 * for E2M3, E3M2 and E2M1).  FP4_E2M1: 1 sign, 2 exponent (bias 1), 1
 * mantissa bit -- 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives -- two per
 * byte, element 2i in the low nibble of byte i of a row; A and B_T both
 * FP4_E2M1 (not mixed with the other formats), K (in elements) a multiple
 * of 32, lda / ldb in bytes (>= K / 2); schedules AUTO, TILE128 and
 * 4WAVE_MFMA16 (AUTO's choice where it takes that schedule for 8-bit
 * operands of the same byte shape).
 * FP6_E2M3 (1 sign, 2 exponent bits, bias 1, 3 mantissa bits; largest 7.5)
 * and FP6_E3M2 (1 sign, 3 exponent bits, bias 3, 2 mantissa bits; largest
 * 28), no inf or NaN: four per three bytes, packed LSB first -- element k
 * of a row is bits [6k, 6k + 6) of the row read as one little-endian bit
 * string; A and B_T both fp6 (either variant each), K (in elements) a
 * multiple of 64, lda / ldb in bytes (>= 3K / 4, multiples of 16),
 * schedules AUTO, TILE128 and 4WAVE_MFMA16 (AUTO's choice where it takes
 * that schedule for 8-bit operands of the same byte shape), no MX block
 * scales. */
enum {
  HIPGEMM_FMT_E4M3 = 0,     /* E4M3FN: bias 7, max 448, NaN 0x7F/0xFF, no inf */
  HIPGEMM_FMT_E5M2 = 1,     /* E5M2: bias 15, max 57344, IEEE inf and NaN     */
  HIPGEMM_FMT_FP6_E2M3 = 2, /* E2M3: max 7.5, no inf or NaN                   */
  HIPGEMM_FMT_FP6_E3M2 = 3, /* E3M2: max 28, no inf or NaN                    */
  HIPGEMM_FMT_FP4_E2M1 = 4  /* E2M1: max 6, no inf or NaN                     */
};

/* Output types of hipgemm_gemm.  BF16, F16: round to nearest even; F32: the
 * fp32 value itself; FP8_E4M3: OCP e4m3 of activation(v) * scale_out, round
 * to nearest even, finite magnitudes above 448 saturate to 448, Inf and NaN
 * become NaN (0x7f | sign) -- the __HIP_SATFINITE conversion of
 * amd_hip_fp8.h.  F32 and FP8_E4M3 run on schedules AUTO, 4WAVE_MFMA16,
 * SKINNY and TILE128. */
enum {
  HIPGEMM_OUT_BF16 = 0,
  HIPGEMM_OUT_F16 = 1,
  HIPGEMM_OUT_F32 = 2,
  HIPGEMM_OUT_FP8_E4M3 = 3
};

/* Activations of the fused epilogue, applied in fp32 after bias:
 *   RELU(v) = v < 0 ? 0 : v
 *   GELU_TANH(v) = v/2 (1 + tanh(sqrt(2/pi) (v + 0.044715 v^3)))
 *   SILU(v) = v / (1 + exp(-v))
 * evaluated with the hardware exponential and reciprocal (a few ulp of
 * fp32 before the rounding to the output type). */
enum {
  HIPGEMM_ACT_NONE = 0,
  HIPGEMM_ACT_RELU = 1,
  HIPGEMM_ACT_GELU_TANH = 2,
  HIPGEMM_ACT_SILU = 3
};

/*
 * Full description of one GEMM for hipgemm_gemm:
 *
 *   scale[m,n] = scale_rows[m] * (scale_cols[n] * (scale_a * scale_b))
 *   v[m,n]     = fma(acc[m,n], scale[m,n], bias[n])       (one rounding)
 *   C[m,n]     = round_out(activation(v[m,n]) [* scale_out, e4m3 only])
 *
 * acc is the fp32 sum over K of A[m,k] * B_T[n,k] with A in a_format and
 * B_T in b_format.  NULL scalars and vectors are ones, a NULL bias is
 * -0.0 (v is then exactly acc * scale).  With the defaults (e4m3 x e4m3, no
 * vectors, no bias, no activation, bf16) this is hipgemm_fp8_gemm_bf16,
 * bit for bit.  Zero-initialise the struct, set `size` to
 * sizeof(hipgemm_gemm_desc) (a different size is rejected), then the
 * fields.  Shape, stride, alignment and workspace rules are those of the
 * entry points above; vectors must be 4-byte aligned; variant
 * HIPGEMM_VARIANT_4WAVE accepts only the defaults of format and epilogue.
 */
typedef struct hipgemm_gemm_desc {
  size_t size;
  const void *A;   /* M x K, row stride lda bytes */
  const void *B_T; /* N x K, row stride ldb bytes */
  void *C;         /* M x N, row stride ldc elements of out_dtype, aligned
                    * to one element */
  int M, N, K;
  int lda, ldb, ldc;
  int a_format, b_format; /* HIPGEMM_FMT_* */
  int out_dtype;          /* HIPGEMM_OUT_* */
  int activation;         /* HIPGEMM_ACT_* */
  const float *scale_a, *scale_b;       /* device scalars or NULL */
  const float *scale_rows, *scale_cols; /* device vectors of M, N or NULL */
  const float *bias;                    /* device vector of N or NULL */
  int variant;                          /* HIPGEMM_VARIANT_* */
  void *workspace; /* as for hipgemm_fp8_gemm_bf16_ws; NULL with size 0: */
  size_t workspace_bytes; /* allocate one when needed, stream-ordered    */
  /* MX block scales (OCP Microscaling v1.0): E8M0 bytes, one per 32
   * consecutive K-elements of a row of A / B_T, 2^(e - 127), 255 = NaN,
   * in the packed device layout hipgemm_mx_pack_scales writes.  Both or
   * neither; K % 32 == 0, 16-byte aligned.  Each element is multiplied by its
   * block's scale before the products are summed; the per-tensor scales
   * still apply.  Not combined with the row / column / bias / activation /
   * output-type options; schedules AUTO (the 128 x 128 one where AUTO picks
   * it, else the 4-wave one), HIPGEMM_VARIANT_4WAVE_MFMA16 and
   * HIPGEMM_VARIANT_TILE128 (which also takes fp4 operands: MXFP4). */
  const void *mx_scale_a, *mx_scale_b;
  /* Device scalar or NULL (1.0) multiplying activation(v) before the
   * conversion; FP8_E4M3 output only (NULL otherwise), 4-byte aligned. */
  const float *scale_out;
} hipgemm_gemm_desc;

/*
 * Runtime-shape GEMM with scales and a stream.
 * Replaces: fp8_gemm_4wave_256x256x128<M, N, K><<<(M*N)/65536, 256>>>(A, B_T,
 * C) (fp8_4wave.hpp:334-338, launched at test.cpp:79 and bench.cpp:78), whose
 * shapes are template constants, strides fixed at lda = ldb = K, ldc = N, with
 * no scales and the null stream.
 */
hipError_t hipgemm_fp8_gemm_bf16(const void *A, const void *B_T, void *C,
                                 int M, int N, int K, int lda, int ldb,
                                 int ldc, const float *scale_a,
                                 const float *scale_b, int variant,
                                 hipStream_t stream);

/*
 * hipgemm_fp8_gemm_bf16 with a caller-provided workspace.  A schedule that
 * needs scratch memory (hipgemm_workspace_size(M, N, K, variant) > 0: the
 * skinny split-K and column-strip schedules' K-slices and the 128 x 128
 * schedule's keep their arrival counters and fp32 partial tiles there) uses
 * `workspace` instead of taking a stream-ordered allocation
 * (hipMallocAsync, a clear of the counters, hipFreeAsync: about 12 us of
 * host time) on `stream` for the call, as hipgemm_fp8_gemm_bf16 does.  The
 * workspace must be 256-byte aligned and at least that size, and its first
 * HIPGEMM_WS_COUNTER_BYTES bytes zero before its first use (every call
 * leaves them zero: see HIPGEMM_WS_COUNTER_BYTES).  Calls that may run
 * concurrently must not share a workspace.  Returns hipErrorInvalidValue if
 * it is missing or too small when needed.  It is not needed for AUTO's
 * 64-column tiles (hipgemm_auto_tile): where only their K-slices would use it,
 * a call with less, or none, runs them in the slices that fit, or over whole K.
 * While `stream` is being captured into a graph, an entry point given no
 * workspace allocates none: a schedule that would split K runs with one
 * K-slice (the same result within rounding, slower on the shapes that
 * split).  Pass a workspace there to keep the split.  Without a workspace
 * the strip schedule also runs one K-slice, allocating nothing, where each
 * strip then streams at most 1 MiB of A and B_T (faster than an allocation
 * per call there; the result again within rounding of the split one).
 * Replaces: the same reference launch (the reference has no workspace and no
 * split-K path).
 */
hipError_t hipgemm_fp8_gemm_bf16_ws(const void *A, const void *B_T, void *C,
                                    int M, int N, int K, int lda, int ldb,
                                    int ldc, const float *scale_a,
                                    const float *scale_b, int variant,
                                    void *workspace, size_t workspace_bytes,
                                    hipStream_t stream);

/*
 * Per-row / per-column scaled GEMM:
 *
 *   C[m, n] = bf16_rne( (scale_rows[m] * scale_cols[n]) * sum_k A[m,k] B_T[n,k] )
 *
 * scale_rows is a DEVICE vector of M fp32 (one per row of A and C),
 * scale_cols one of N fp32 (one per row of B_T, i.e. column of C); either may
 * be NULL for all ones.  The product of the two scales is formed in fp32 and
 * applied to the fp32 accumulator before rounding, as in
 * hipgemm_fp8_gemm_bf16 (which is this call with constant vectors).  Both
 * vectors must be 4-byte aligned.  Accepts every schedule but
 * HIPGEMM_VARIANT_4WAVE, which returns hipErrorInvalidValue (SKINNY and
 * STRIP for M <= 128 only).  Workspace as in
 * hipgemm_fp8_gemm_bf16_ws, except that workspace == NULL with
 * workspace_bytes == 0 takes a stream-ordered allocation when one is needed,
 * as hipgemm_fp8_gemm_bf16 does.
 * No reference counterpart: the reference applies no scales at all
 * (store_rt, fp8_4wave.hpp:214-238, converts the accumulator straight to
 * bf16).
 */
hipError_t hipgemm_fp8_gemm_bf16_rowcol(const void *A, const void *B_T, void *C,
                                        int M, int N, int K, int lda, int ldb,
                                        int ldc, const float *scale_rows,
                                        const float *scale_cols, int variant,
                                        void *workspace, size_t workspace_bytes,
                                        hipStream_t stream);

/*
 * The general entry point: operand formats (e4m3 / e5m2, mixed), output
 * type (bf16 / fp16), per-tensor and per-row / per-column scales, bias and
 * activation, fused into the one kernel (see hipgemm_gemm_desc).
 * No reference counterpart beyond the plain launch it generalises: the
 * reference's kernel is e4m3 x e4m3 -> bf16 with no scales
 * (fp8_4wave.hpp:58 passes format codes 0, 0 and zero scales to the MFMA;
 * store_rt, :214-238, converts the accumulator straight to bf16).
 */
hipError_t hipgemm_gemm(const hipgemm_gemm_desc *desc, hipStream_t stream);

/*
 * hipgemm_gemm that allocates nothing: schedules that need scratch memory
 * (the skinny schedule's split-K counters and partial tiles, the 128 x 128
 * schedule's K-slices) use a static device array of the library,
 * HIPGEMM_NOALLOC_SCRATCH_BYTES per GPU: it belongs to the code object of
 * its own translation unit, which the HIP runtime loads on a GPU at the first
 * hipgemm_gemm_noalloc call there that needs scratch, and holds until the
 * process ends (with the runtime's deferred code-object loading; without
 * it, on every GPU where the library's code is loaded).  AUTO's 64-column
 * K-slices use it too, but do not make a call need it (they run over whole K
 * where nothing else of the call would).  No call makes an
 * allocation or a memset.
 * desc->workspace must be NULL and desc->workspace_bytes 0.  Returns
 * hipErrorInvalidValue when the descriptor is invalid (as hipgemm_gemm) or
 * when the call would need more scratch than HIPGEMM_NOALLOC_SCRATCH_BYTES
 * (hipgemm_gemm_workspace_size(desc) tells; never on MI355X, whose largest
 * need is 32 MiB plus the counter region).  Every call on one GPU shares
 * that GPU's array and leaves its counters at zero: calls on one stream
 * are ordered, but calls that may overlap on one GPU (other streams,
 * threads or processes' graphs replayed concurrently) race on it.  Its
 * first call on a GPU looks the array's address up (hipGetSymbolAddress)
 * and clears its counters with a kernel on `stream`.
 * No reference counterpart (the reference's kernel needs no scratch).  For
 * callers that cannot allocate device memory: code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc.
 */
#define HIPGEMM_NOALLOC_SCRATCH_BYTES (HIPGEMM_WS_COUNTER_BYTES + (32u << 20))
hipError_t hipgemm_gemm_noalloc(const hipgemm_gemm_desc *desc,
                                hipStream_t stream);

/*
 * MX scale packing.  hipgemm_mx_scales_bytes: bytes of the packed layout for
 * an operand of `rows` rows and K columns (0 for rows or K <= 0).
 * hipgemm_mx_pack_scales: packs src, `rows` x ceil(K/32) E8M0 bytes with
 * row stride ld bytes (device), into dst (device, that many bytes),
 * stream-ordered.  The layout groups, per 128 rows and per two 128-wide
 * K-steps, what one wave's MFMA need (padding scales are 1.0).  Returns
 * hipErrorInvalidValue for K % 32 != 0, ld < K / 32 or null pointers.
 * No reference counterpart (the reference passes zero scales,
 * fp8_4wave.hpp:58).
 */
size_t hipgemm_mx_scales_bytes(int rows, int K);
hipError_t hipgemm_mx_pack_scales(const void *src, int rows, int K, int ld,
                                  void *dst, hipStream_t stream);

/*
 * Per-row e4m3 quantisation of x (M x K, device, row stride ldx elements, of
 * type HIPGEMM_IN_*): s[m] = max |x[m, :]| times fp32(1 / 448), or 1 where that
 * maximum is 0 or NaN; q[m, k] (M x K packed bytes) = e4m3 of x[m, k] / s[m]
 * clamped to +-448, round to nearest even, NaN kept.  So x ~= q * s[m], and q, s
 * are hipgemm_gemm's A and scale_rows.  x aligned to its type, s to 4 bytes,
 * ldx >= K; M == 0 or K == 0 is a no-op.  One launch on `stream` per 2^23 rows.
 * No reference counterpart (the reference takes e4m3 operands as they are).
 */
enum { HIPGEMM_IN_F32 = 0, HIPGEMM_IN_BF16 = 1, HIPGEMM_IN_F16 = 2 };
hipError_t hipgemm_quantize_rows_e4m3(const void *x, int type, int M, int K,
                                      long long ldx, void *q, float *s,
                                      hipStream_t stream);

/*
 * Products of 16-bit activations with 4-bit weights:
 *
 *   y[m, n] = round_out(activation(sum_k x[m, k] w[n, k] + bias[n]))
 *   int4: w[n, k] = (q[n, k] - z[n, k / G]) s[n, k / G]
 *   fp4:  w[n, k] = e2m1(q[n, k]) s[n, k / G]
 *
 * x is M x K, bf16 or fp16; q the N x K codes, two per byte, element 2i in the
 * low nibble of byte i of a row; one scale s (and zero point z, a byte, 8 where
 * zeros is NULL) per G = group_size neighbouring elements of a row, N x
 * ceil(K / G).  Products and sums are fp32 and the weights are not rounded: the
 * scale multiplies the fp32 sum over its group.  Results that come out infinite or
 * NaN are computed again term by term, unless their row of x holds a NaN: rows of NaN
 * cost about three times the call, rows with an infinity up to 100 times (M > 4).
 * bias: N floats or NULL.
 * Rows of x, q, scales and zeros are contiguous, with the strides given.
 * Requirements: K % 32 == 0, K <= 2^26, G % 32 == 0, x and q 16-byte aligned
 * with strides of a multiple of 16 bytes, the others aligned to their element;
 * out_dtype BF16, F16 or F32; ldw and lds up to 2^25 bytes.  M == 0 or N == 0 is a
 * no-op, K == 0 gives activation(bias).  One launch on `stream` (one per four rows
 * where K == 0 or ldx > 2^24), no workspace.  Zero-initialise the struct and set
 * `size`.  No reference counterpart (the reference has e4m3 operands only).
 */
enum { HIPGEMM_W4_INT4 = 0, HIPGEMM_W4_FP4 = 1 };
/* Scale types: HIPGEMM_IN_F32, _BF16, _F16, or E8M0 bytes, 2^(e - 127), 255 NaN. */
enum { HIPGEMM_SCALE_E8M0 = 3 };
typedef struct hipgemm_w4_desc {
  size_t size;
  const void *x, *weight, *scales;
  const unsigned char *zeros; /* or NULL */
  void *y;
  const float *bias; /* or NULL */
  int M, N, K, group_size;
  long long ldx;    /* elements */
  long long ldw;    /* bytes */
  long long lds;    /* elements, of zeros too */
  long long ldy;    /* elements */
  int x_type;       /* HIPGEMM_IN_BF16 or HIPGEMM_IN_F16 */
  int format;       /* HIPGEMM_W4_* */
  int scale_type;   /* HIPGEMM_IN_* or HIPGEMM_SCALE_E8M0 */
  int out_dtype;    /* HIPGEMM_OUT_* */
  int activation;   /* HIPGEMM_ACT_* */
} hipgemm_w4_desc;
hipError_t hipgemm_w4_gemm(const hipgemm_w4_desc *desc, hipStream_t stream);

/* The kernel that hipgemm_w4_gemm runs for a descriptor, and the rows and columns of
 * its tiles (0 for VECTORS: up to four rows of x at a time, a pass over the weights).
 * No GPU needed; no reference counterpart. */
enum {
  HIPGEMM_W4_VECTORS = 0,
  HIPGEMM_W4_SPLIT = 1, /* some rows: four waves along K */
  HIPGEMM_W4_TILES = 2  /* many: tiles of 128 x 128 */
};
typedef struct hipgemm_w4_plan {
  int kernel, tile_rows, tile_columns;
} hipgemm_w4_plan;
hipError_t hipgemm_w4_select(const hipgemm_w4_desc *desc, hipgemm_w4_plan *plan);

/*
 * The router's choice of a mixture-of-experts layer: for each of T rows of E
 * logits (device, of type HIPGEMM_IN_*, row stride ld elements) the k largest,
 * in order, equal ones by the lower index:
 *
 *   softmax: p = exp(l - max l) / sum exp(l - max l);  sigmoid: p = 1 / (1 + exp(-l))
 *   weights[t, j] = scale * p[ids[t, j]]   [ / sum over j, if renormalize ]
 *
 * weights (float) and ids (int) are T x k, packed.  A logit of -inf is never
 * chosen: where fewer than k others are left, the rest of the row gets id -1 and
 * weight 0.  A NaN ranks above +inf.  1 <= k <= min(E, 64), E <=
 * HIPGEMM_MOE_MAX_EXPERTS.  One launch, no workspace.  No reference counterpart.
 */
#define HIPGEMM_MOE_MAX_EXPERTS 1024
enum { HIPGEMM_MOE_SOFTMAX = 0, HIPGEMM_MOE_SIGMOID = 1 };
hipError_t hipgemm_moe_route(const void *logits, int type, int T, int E, int k,
                             long long ld, int scoring, int renormalize,
                             float scale, float *weights, int *ids,
                             hipStream_t stream);

/*
 * The experts of a mixture-of-experts layer for a few tokens:
 *
 *   h[t, j] = act(x[t] W13[e][:F]^T) * (x[t] W13[e][F:]^T),  e = ids[t, j]
 *   y[t]    = round_out(sum_j weights[t, j] (h[t, j] W2[e]^T))
 *
 * x: T x D, bf16 or fp16; ids (int), weights (float): T x k, packed.  W13: E x
 * 2F x D (gate rows, then up rows), W2: E x D x F, in one weight format:
 * HIPGEMM_W4_INT4 or _FP4 with scales (and zeros) per group_size elements of a
 * row as in hipgemm_w4_gemm, or HIPGEMM_W8_E4M3 with one float scale per row
 * (scale_type F32, lds 1: E x 2F and E x D).  An id outside [0, E) is skipped: a
 * token without any gives zeros.  Sums are fp32; h is held to 16 significant
 * bits between the two kernels, to fp32's 24 where out_dtype is F32.  Made for a few
 * tokens (up to 64); more go in turns of at most HIPGEMM_MOE_MAX_PAIRS / k.  In a turn
 * an expert's weights are read for each of its tokens while few are read twice
 * (pair by pair: hipgemm_moe_select), else once for up to 16 or 32 of them, W13 for
 * no more than 37120 / D.  Always pair by pair for D above 37120 or F above 65536.
 * D, F, group_size multiples of 32; matrices 16-byte aligned, with row and
 * expert strides of multiples of 16 bytes; k <= 64.  Workspace:
 * hipgemm_moe_workspace_size bytes, 16-byte aligned, of any content; calls that
 * may run concurrently must not share one.  Two launches per turn on `stream`, three
 * grouped.
 * Zero-initialise the struct and set `size`.  No reference counterpart.
 */
enum { HIPGEMM_W8_E4M3 = 2 };
#define HIPGEMM_MOE_MAX_PAIRS 512
typedef struct hipgemm_moe_matrix {
  const void *weight, *scales;
  const unsigned char *zeros;          /* or NULL */
  long long ldw, expert_w;             /* bytes: a row, an expert */
  long long lds, expert_s;             /* elements, of zeros too */
} hipgemm_moe_matrix;
typedef struct hipgemm_moe_desc {
  size_t size;
  const void *x;
  const int *ids;
  const float *weights;
  hipgemm_moe_matrix w13, w2;
  void *y;
  void *workspace;
  size_t workspace_bytes;
  long long ldx, ldy; /* elements */
  int T, k, E, D, F;
  int group_size;     /* not for e4m3 */
  int x_type;         /* HIPGEMM_IN_BF16 or HIPGEMM_IN_F16 */
  int format;         /* HIPGEMM_W4_* or HIPGEMM_W8_E4M3 */
  int scale_type;     /* HIPGEMM_IN_* or HIPGEMM_SCALE_E8M0 */
  int out_dtype;      /* HIPGEMM_OUT_BF16, _F16 or _F32 */
  int activation;     /* HIPGEMM_ACT_* */
} hipgemm_moe_desc;
size_t hipgemm_moe_workspace_size(int T, int k, int E, int D, int F);
hipError_t hipgemm_moe_experts(const hipgemm_moe_desc *desc, hipStream_t stream);

/* How hipgemm_moe_experts runs (the first turn of) a call of these sizes: all 0 pair by
 * pair; grouped, the rows (tokens) of a tile and the waves that share a row's K, up and
 * down, and the parts of F of the down product, of part_len each.  No GPU needed; no
 * reference counterpart. */
typedef struct hipgemm_moe_plan {
  int grouped, up_rows, up_waves, down_rows, down_waves, parts, part_len;
} hipgemm_moe_plan;
hipError_t hipgemm_moe_select(int T, int k, int E, int D, int F, int format,
                              int out_dtype, hipgemm_moe_plan *plan);

/*
 * Products of 16-bit activations with 16-bit weights, and what a feed-forward block
 * does with them:
 *
 *   z[m, n] = sum_k x[m, k] weight[n, k] + bias[n]
 *   y[m, n] = round_out(activation(z[m, n]) + residual[m, n])
 *
 * gated: weight holds N gate rows, then N up rows (bias likewise), and
 *
 *   y[m, n] = round_out(activation(z[m, n]) * z[m, N + n])
 *
 * x is M x K, weight N x K (gated 2N x K), both of `type`, bf16 or fp16; products and
 * sums are fp32.  bias, residual (not gated) and pre may be NULL; pre receives z (gated:
 * both halves, M x 2N) as pre_dtype, for the backward pass.  bias_type,
 * residual_type: HIPGEMM_IN_*.  Rows are contiguous, with the strides given.
 * Requirements: K % 8 == 0, gated N % 8 == 0;  x and weight 16-byte aligned with row
 * strides of a multiple of 8;  the others aligned to their element (16 bytes, strides
 * of a multiple of 16 bytes and N % 8 == 0 are faster);  M <= 2^30, K, rows of weight
 * and strides of x and weight up to 2^21.  residual may be y itself; otherwise what is
 * written overlaps nothing else.  M == 0 or N == 0 is a no-op;  K == 0 is a sum of nothing.
 * Workspace: hipgemm_linear_workspace_size bytes (0 for most calls), 256-byte aligned, of
 * any content; calls that may run concurrently must not share one.  Zero-initialise the
 * struct and set `size`.  No reference counterpart (the reference has e4m3 operands only).
 */
typedef struct hipgemm_linear_desc {
  size_t size;
  const void *x, *weight;
  const void *bias, *residual; /* or NULL */
  void *y;
  void *pre;                   /* or NULL */
  void *workspace;
  size_t workspace_bytes;
  long long ldx, ldw, ldr, ldy, ldp; /* elements */
  int M, N, K;
  int gated;                   /* 0 or 1 */
  int type;                    /* HIPGEMM_IN_BF16 or HIPGEMM_IN_F16 */
  int bias_type, residual_type; /* HIPGEMM_IN_* */
  int out_dtype, pre_dtype;    /* HIPGEMM_OUT_BF16, _F16 or _F32 */
  int activation;              /* HIPGEMM_ACT_* */
} hipgemm_linear_desc;
size_t hipgemm_linear_workspace_size(const hipgemm_linear_desc *desc);
hipError_t hipgemm_linear(const hipgemm_linear_desc *desc, hipStream_t stream);

/*
 * Its backward pass: of dy, the gradient of y (M x N, dy_type HIPGEMM_IN_*),
 *
 *   dz = dy activation'(z)     gated, z = [g | u]: [dy u activation'(g) | dy activation(g)]
 *   dx = dz weight             M x K
 *   dw = dz^T x                N x K (gated 2N x K)
 *   db[n] = sum_m dz[m, n]     N (gated 2N)
 *
 * each where its pointer is not NULL.  (The residual's gradient is dy.)  z is read from
 * pre (pre_type HIPGEMM_IN_*), as the forward pass left it; not needed where activation is
 * NONE and not gated.  dz is rounded to `type` for the products of 16-bit results, and held
 * to fp32's 24 bits for float32 ones (in parts of `type`, three of bf16 or two of fp16, with
 * a product each; values past fp16's range are infinite) and for db; sums are fp32, in an
 * order that depends on sizes and types only.  Slopes: relu'(0) = 0.  With M == 0, dw
 * and db are zeros.  Requirements as above; dy, pre: aligned to their element.  Workspace:
 * hipgemm_linear_backward_workspace_size bytes for the descriptor (its pointers, strides
 * and types matter), as above.  No reference counterpart.
 */
typedef struct hipgemm_linear_grad_desc {
  size_t size;
  const void *dy, *x, *weight;
  const void *pre;             /* or NULL */
  void *dx, *dw, *db;          /* or NULL */
  void *workspace;
  size_t workspace_bytes;
  long long lddy, ldx, ldw, ldp, lddx, lddw; /* elements */
  int M, N, K;
  int gated;
  int type;                    /* of x and weight */
  int dy_type, pre_type;       /* HIPGEMM_IN_* */
  int dx_dtype, dw_dtype, db_dtype; /* HIPGEMM_OUT_BF16, _F16 or _F32 */
  int activation;
} hipgemm_linear_grad_desc;
size_t hipgemm_linear_backward_workspace_size(const hipgemm_linear_grad_desc *desc);
hipError_t hipgemm_linear_backward(const hipgemm_linear_grad_desc *desc,
                                   hipStream_t stream);

/* The kernels that hipgemm_linear and hipgemm_linear_backward's products (dx, dw; all 0
 * where not asked for) run for a descriptor's sizes: tiles of tile_rows x tile_columns
 * results (gated: of gate and up columns together), or tile_rows 0 for the kernel of a few
 * rows; the slices along K, whose sums are added by a second kernel; and the first columns
 * (0: none) that tiles of 256 x 256 do in a launch of their own.  (dx and dw both whole in
 * tiles of 128 x 128, not more than the CUs together: one launch.  A float32 dx or dw: the
 * kernel of each part of dz, all added by a second.)  No GPU needed; no reference
 * counterpart. */
typedef struct hipgemm_linear_plan {
  int tile_rows, tile_columns, slices, first_columns;
} hipgemm_linear_plan;
hipError_t hipgemm_linear_select(const hipgemm_linear_desc *desc, hipgemm_linear_plan *plan);
hipError_t hipgemm_linear_backward_select(const hipgemm_linear_grad_desc *desc,
                                          hipgemm_linear_plan plan[2]);

/* Workspace bytes hipgemm_fp8_gemm_bf16_ws needs for this shape and variant
 * on the current device (0: none).  No GPU work.  No reference counterpart. */
size_t hipgemm_workspace_size(int M, int N, int K, int variant);

/* Workspace bytes hipgemm_gemm needs for this descriptor on the current
 * device (0: none, or an invalid descriptor); it accounts for the operand
 * formats, the output type and the schedule AUTO takes for them.  No GPU work.  No reference
 * counterpart. */
size_t hipgemm_gemm_workspace_size(const hipgemm_gemm_desc *desc);

/*
 * The reference launch with runtime shapes: packed strides (lda = ldb = K,
 * ldc = N), no scales, the 4-wave schedule (16x16x128 MFMA).
 * Replaces: fp8_gemm_4wave_256x256x128<M, N, K><<<(M*N)/65536, 256>>>(A, B_T,
 * C) at test.cpp:79 and bench.cpp:55/78.
 */
hipError_t hipgemm_fp8_gemm_4wave_256x256x128(const void *A, const void *B_T,
                                              void *C, int M, int N, int K,
                                              hipStream_t stream);

/* The schedule that AUTO names for this shape (no GPU needed); where
 * hipgemm_auto_tile returns 1, 8-bit operands run on that tile instead.  No
 * reference counterpart (the reference has one schedule). */
int hipgemm_select_variant(int M, int N, int K);

/* AUTO's column split: when the last round of 256 x 256 tiles would leave
 * most CUs idle, AUTO runs columns [0, n1) of C on the 4-wave 16x16x128
 * schedule (whole rounds) and [n1, N) on the 128 x 128 schedule, two
 * launches on the caller's stream.  Returns n1 (a multiple of 256), or 0
 * when AUTO runs one schedule, or the tile of hipgemm_auto_tile (calls that that
 * tile is not built for, extended epilogues without aligned stores, may still
 * split).  Uses the current device's CU count (256
 * without a device).  No reference counterpart (the reference's grid is
 * M*N/65536 tiles of 256 x 256, fp8_4wave.hpp:357-377). */
int hipgemm_split_columns(int M, int N, int K);

/* AUTO's tile for 8-bit operands above 32 rows, where another tile is
 * estimated faster than the schedule hipgemm_select_variant names: returns 1
 * and the tile (bm x bn), or 0 when AUTO runs that schedule as it is.  Such
 * calls run the 128 x 128 schedule's pipeline in one launch on 128 x 256, 192
 * x 192, 192 x 128 or 128 x 128 tiles (above 128 rows, no workspace) or, up to
 * 1024 rows, on 128 x 64 or 64 x 64 tiles -- those in K-slices where that is
 * faster and the call brings a workspace that holds them (what
 * hipgemm_workspace_size names for AUTO does) or runs hipgemm_gemm_noalloc, the
 * last slice to arrive at a part of a tile summing it.  For packed operands (lda =
 * ldb = K): the choice also depends on whether rows start on 128-byte lines.  No
 * reference counterpart (the reference has 256 x 256 tiles only). */
int hipgemm_auto_tile(int M, int N, int K, int *bm, int *bn);

/* Human-readable variant name, or NULL.  No reference counterpart. */
const char *hipgemm_variant_name(int variant);

/* HIPGEMM_VERSION of the built library.  No reference counterpart. */
int hipgemm_version(void);

/*
 * Host-side view of the workgroup -> output-tile order a launch of `grid`
 * workgroups uses over a tiles_m x tiles_n tile grid: fills tile_m[i],
 * tile_n[i] for the i-th tile processed (workgroup-major: the tiles of
 * workgroup b are b's first, second, ... tile).  Returns the number of
 * entries written (at most cap).  For tests of the order's bijectivity; no
 * GPU needed.  group_m <= 0 selects the library default.  Replaces the
 * in-kernel remap at fp8_4wave.hpp:357-377 (not callable there).
 */
int hipgemm_tile_order(int grid, int tiles_m, int tiles_n, int group_m,
                       int *tile_m, int *tile_n, int cap);

/*
 * Host-side view of the LDS tile layout: the 16-byte slot (0..7) at which
 * K-chunk `chunk` (0..7) of tile row `row` sits inside its 128-byte LDS row.
 * For tests of the bank-conflict-freedom of the layout; no GPU needed.
 * Returns -1 for out-of-range arguments.  Replaces the swizzle helpers at
 * fp8_4wave.hpp:136-177 (not callable there).
 */
int hipgemm_lds_slot(int row, int chunk);

/*
 * The same for the instruction K order (MX block scales on the 4-wave
 * schedule, and the skinny schedule's A): the MFMA's lane group g holds
 * K-chunks g
 * and g + 4 of its row, stored where the plain order above keeps chunks 2g
 * and 2g + 1, so both fetch the same LDS addresses.  -1 for out-of-range
 * arguments.  No reference counterpart (its kernel has one K order).
 */
int hipgemm_lds_slot_kpair(int row, int chunk);

/*
 * The 8-byte slot (0-15) of the 8-byte piece `piece` (0-15) of row `row` of
 * the 4-wave schedule's epilogue stage (128-byte rows of bf16 C, staged
 * between the accumulators and the 16-byte stores of whole 128-byte lines).
 * -1 for out-of-range arguments.  No reference counterpart (its epilogue
 * stores from the accumulators).
 */
int hipgemm_lds_stage_slot(int row, int piece);

#ifdef __cplusplus
}
#endif

#endif /* HIPGEMM_H */
