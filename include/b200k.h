/*
 * b200k.h -- C ABI of the B200 (sm_100a) kernel backend for Emmy Kernel IR.
 *
 * The reference compiler turns each recognised Kernel-IR kernel into PTX text
 * (compile.py:9628-9724 compile_path) which a runner assembles and launches
 * with cuLaunchKernel, passing positional arguments in meta.json's arg_order
 * (tools/local_runner.py:246-342, launch at :309-324).  This library replaces
 * that emitted PTX: a front end recognises the kernel and calls one of the
 * entry points below with the same device buffers.
 *
 * Conventions shared by every entry point:
 *   - Plain C types only: device pointers, 64-bit extents, a cudaStream_t
 *     passed as void* (NULL = the legacy default stream).
 *   - The caller owns every buffer; the library only reads inputs and writes
 *     outputs.  Scratch memory (the GEMM's TF32 operand split) belongs to the
 *     context and is reused across calls.
 *   - Return value: B2K_OK, a positive validation code (nothing was
 *     launched), or a negative device-side code.  b2k_last_error() gives a
 *     human-readable reason.
 *   - A context is not thread-safe: use one per (host thread, device).
 */
#ifndef B200K_H
#define B200K_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define B2K_OK 0
#define B2K_EINVAL 1       /* invalid argument; nothing launched */
#define B2K_EUNSUPPORTED 2 /* valid request outside this build's kernels */
#define B2K_ECUDA (-1)     /* CUDA runtime/driver error */
#define B2K_ETIMEOUT (-2)  /* a device-side bounded wait expired (kernel error flag) */
#define B2K_ESCRATCH 3     /* problem needs more than the fixed no-alloc scratch array */
#define B2K_ENCCL (-3)     /* NCCL error; the multi-GPU handle is aborted and must be destroyed */
#define B2K_EINDEX (-4)    /* a kernel met an index from device memory outside its bounds */

typedef struct b2k_ctx b2k_ctx;

/* ABI version of this header (major*100 + minor). */
int b2k_version(void);

/* Create a context on CUDA device `device_ordinal` (makes it current on this
 * thread).  Replaces the runner's per-worker context set-up
 * (tools/local_runner.py:258-280). */
int b2k_init(int device_ordinal, b2k_ctx **out);
int b2k_destroy(b2k_ctx *ctx);
/* Reason for the last non-OK return on this context ("" if none). */
const char *b2k_last_error(const b2k_ctx *ctx);
/* Streaming multiprocessor count of the context's device. */
int b2k_sm_count(const b2k_ctx *ctx);

/* --- device memory helpers for callers without their own allocator ------
 * (the runner's cuMemAlloc / cuMemcpyHtoD / cuMemcpyDtoH / cuMemsetD8 calls,
 * tools/local_runner.py:287-300, 320-322, 333-338). */
int b2k_malloc(b2k_ctx *ctx, void **ptr, size_t bytes);
int b2k_free(b2k_ctx *ctx, void *ptr);
int b2k_memcpy_htod(b2k_ctx *ctx, void *dst, const void *src, size_t bytes, void *stream);
int b2k_memcpy_dtoh(b2k_ctx *ctx, void *dst, const void *src, size_t bytes, void *stream);
int b2k_memset(b2k_ctx *ctx, void *dst, int value, size_t bytes, void *stream);
/* Page-locked host memory, so host<->device copies run asynchronously at
 * full PCIe/C2C bandwidth. */
int b2k_host_alloc(b2k_ctx *ctx, void **ptr, size_t bytes);
int b2k_host_free(b2k_ctx *ctx, void *ptr);
int b2k_stream_sync(b2k_ctx *ctx, void *stream);
/* Failure-detection self test: launches one kernel whose mbarrier wait can
 * never complete and gives up after `budget_cycles` SM cycles (at most the
 * kernels' own ~2 s budget), exactly as a stalled tensor-core kernel would.
 * The following b2k_stream_sync returns B2K_ETIMEOUT and clears the device
 * error word; the context stays usable.  No counterpart in the reference
 * (its runner retires a worker process on any CUDA error,
 * tools/local_runner.py:246-342). */
int b2k_selftest_wait_timeout(b2k_ctx *ctx, int64_t budget_cycles, void *stream);

/* --- per-phase timing -------------------------------------------------------
 * When enabled, every entry point brackets the kernels of each of its phases
 * with CUDA events recorded on the caller's stream (the runner's event
 * timing, tools/local_runner.py:318-332, per kernel instead of per launch
 * request).  b2k_timing_read synchronises and sums the recorded intervals of
 * one phase (`launches` = intervals: one per entry-point call of the phase,
 * which may cover more than one kernel); b2k_timing_reset forgets them.
 * b2k_kernel_launches returns how many kernels the context has enqueued
 * since b2k_init (every launch is counted, timing enabled or not). */
#define B2K_PHASE_SPLIT 0     /* 3xTF32 operand split pre-pass */
#define B2K_PHASE_MMA 1       /* tcgen05 GEMM main kernel */
#define B2K_PHASE_POINTWISE 2 /* pointwise programs */
#define B2K_PHASE_SOFTMAX 3   /* row softmax */
#define B2K_PHASE_ATTENTION 4 /* attention (all of its passes) */
#define B2K_PHASE_ROWS 5      /* row reductions / norms */
#define B2K_PHASE_FLASH 6     /* fused attention kernel */
#define B2K_PHASE_ROTARY 7    /* rotary positions */
#define B2K_PHASE_APPEND 8    /* append to a paged cache */
#define B2K_PHASE_PAGED 9     /* attention over a paged cache (all of its kernels) */
#define B2K_PHASE_VERIFY 10   /* verification of drafted tokens */
#define B2K_PHASE_COUNT 11
int b2k_timing_enable(b2k_ctx *ctx, int on);
/* Restrict timing to the phases whose bit (1 << B2K_PHASE_*) is set in
 * `phase_mask` (default: all).  Each timed phase costs two event records
 * per call, and an event between two kernels of one call serialises them
 * (see b2k_set_pdl), so a caller timing one kernel should select only its
 * phase. */
int b2k_timing_select(b2k_ctx *ctx, uint32_t phase_mask);
int b2k_timing_read(b2k_ctx *ctx, int phase, double *total_ms, int64_t *launches);
int b2k_timing_reset(b2k_ctx *ctx);
int b2k_kernel_launches(b2k_ctx *ctx, int64_t *count);

/* --- launch overlap -----------------------------------------------------------
 * Process-wide switch (default on): the kernels of a split-then-multiply
 * operation (GEMM, fused attention) are launched with programmatic
 * dependent launch, so the tensor-core kernel's CTAs are scheduled and run
 * their set-up while the split kernel drains, and the next call's split
 * overlaps this call's tail.  Results are identical either way; the switch
 * exists for comparisons.  No counterpart in the reference. */
int b2k_set_pdl(int on);

/* --- pointwise programs ---------------------------------------------------
 * Replaces the SIMT Emitter's pointwise lowering: Tile decode
 * (compile.py:8473-8585), 16-byte vector load/store groups
 * (compile.py:1425-1600, 5865-5942, 8586-8661) and scalar arithmetic
 * (compile.py:2645-2965).  A program is a straight-line list of FP32
 * operations over up to B2K_PW_MAX_INPUTS input streams; register r < n_inputs
 * holds input r's element, later registers hold instruction results. */
#define B2K_PW_MAX_INPUTS 8
#define B2K_PW_MAX_INSNS 48
#define B2K_PW_MAX_REGS (B2K_PW_MAX_INPUTS + B2K_PW_MAX_INSNS)

enum b2k_pw_opcode {
  B2K_OP_CONST = 0,      /* dst = imm */
  B2K_OP_COPY = 1,       /* dst = a */
  B2K_OP_ADD = 2,        /* dst = a + b (round to nearest) */
  B2K_OP_SUB = 3,
  B2K_OP_MUL = 4,
  B2K_OP_DIV = 5,        /* IEEE division, round to nearest */
  B2K_OP_MAX = 6,
  B2K_OP_MIN = 7,
  B2K_OP_NEG = 8,
  B2K_OP_RCP = 9,        /* 1/a, round to nearest */
  B2K_OP_SQRT = 10,      /* round to nearest */
  B2K_OP_RSQRT = 11,     /* 1/sqrt(a) */
  B2K_OP_EXP = 12,       /* selective subnormal-preserving exp (compile.py:2953-2965) */
  B2K_OP_RELU = 13,      /* max(a, 0) */
  B2K_OP_ABS = 14,
  B2K_OP_FMA = 15,       /* dst = a * b + c, single rounding */
  B2K_OP_GT = 16,        /* dst = (a > b) ? 1 : 0 */
  B2K_OP_GE = 17,
  B2K_OP_LT = 18,
  B2K_OP_LE = 19,
  B2K_OP_WHERE = 20,     /* dst = (a != 0) ? b : c */
  B2K_OP_LOG = 21,       /* natural log via lg2.approx * ln2 (compile.py:2938-2942) */
  B2K_OP_COUNT = 22
};

typedef struct b2k_pw_insn {
  int32_t op;       /* enum b2k_pw_opcode */
  int32_t a, b, c;  /* source registers (unused ones ignored) */
  float imm;        /* B2K_OP_CONST value */
} b2k_pw_insn;

typedef struct b2k_pw_program {
  int32_t n_inputs;                        /* input streams, registers 0..n_inputs-1 */
  int32_t n_insns;                         /* instructions; insn i writes register n_inputs+i */
  int32_t result;                          /* register stored to the output */
  int32_t broadcast[B2K_PW_MAX_INPUTS];    /* 1: input is a scalar buffer read at element 0 */
  int32_t offset[B2K_PW_MAX_INPUTS];       /* >= 0: input i is read at element i + offset[i]
                                              (a shifted window; ignored for broadcast inputs) */
  b2k_pw_insn insns[B2K_PW_MAX_INSNS];
} b2k_pw_program;

/* out[i] = program(inputs[0][i + offset[0]], inputs[1][i + offset[1]], ...)
 * for i in [0, n).  Non-broadcast input r must hold n + offset[r] FP32
 * elements, out n; 16-byte vector accesses are used when every stream (its
 * base plus offset) is 16-byte aligned, element accesses otherwise -- the
 * runtime alignment fallback of the reference's vector groups
 * (compile.py:1425-1600, 8586-8661). */
int b2k_pointwise_f32(b2k_ctx *ctx, const b2k_pw_program *program, const float *const *inputs,
                      float *out, int64_t n, void *stream);

/* --- row softmax ----------------------------------------------------------
 * Replaces the Emitter's row-reduction softmax passes: online/two-pass
 * max+sum (compile.py:1656-1711, 6492-6644), warp-shuffle and shared-tree
 * combine (compile.py:8958-9035, 9175-9268), selective exp
 * (compile.py:2953-2965) and the reciprocal-multiply normalisation.
 * y[r, :] = exp(x[r, :] - max_r) / sum_r for a row-major rows x cols matrix
 * with leading dimensions ld_x / ld_y (elements). */
int b2k_row_softmax_f32(b2k_ctx *ctx, const float *x, float *y, int64_t rows, int64_t cols,
                        int64_t ld_x, int64_t ld_y, void *stream);

/* --- row reductions and row norms -------------------------------------------
 * Replaces the Emitter's merged vector row reduction (compile.py:4987-5165,
 * shuffles and trees 8958-9268) and row-map reuse (compile.py:5511-5665) for
 * the reduction / rmsnorm / l2norm kernels:
 *   B2K_ROW_SUM      y[r]    = (sum_c x[r,c]) / div                 (div = *sum_div_ptr or sum_div)
 *   B2K_ROW_RMSNORM  y[r,c]  = x[r,c] * w[c] / sqrt(sum_c x^2 / count + eps)
 *   B2K_ROW_L2NORM   y[r,c]  = x[r,c] * w[c] / sqrt(sum_c x^2 + eps)
 *   B2K_ROW_MAX      y[r]    = max_c x[r,c]    (IEEE maxNum: a NaN loses to a number)
 *   B2K_ROW_MIN      y[r]    = min_c x[r,c]    (IEEE minNum)
 *   B2K_ROW_PROD     y[r]    = prod_c x[r,c]   (FP32 products in a fixed tree order)
 * count = *ms_div_ptr or ms_div, eps = *eps_ptr or eps; w may be NULL (1).
 * A single row longer than 65,536 (a whole-array sum) is reduced by many CTAs
 * and a fixed-order second pass. */
#define B2K_ROW_SUM 0
#define B2K_ROW_RMSNORM 1
#define B2K_ROW_L2NORM 2
#define B2K_ROW_MAX 3
#define B2K_ROW_MIN 4
#define B2K_ROW_PROD 5
typedef struct b2k_row_params {
  int32_t op;
  float sum_div;
  const float *sum_div_ptr;
  float ms_div;
  const float *ms_div_ptr;
  float eps;
  const float *eps_ptr;
  const float *w;
} b2k_row_params;
/* Fold over the middle axis of x [batch][s][cols] (contiguous):
 *   y[b][j] = fold_{i < s} x[b][i][j]      (y [batch][cols], contiguous)
 * op: B2K_ROW_SUM (the sum divided by *div_ptr when non-NULL, else by div:
 * a mean for div = s), B2K_ROW_MAX, B2K_ROW_MIN (IEEE maxNum / minNum) or
 * B2K_ROW_PROD.  Each output folds i = 0, 1, ... in order, as the IR's serial
 * Loop + Accum over that axis (the reference interpreter,
 * tests/test_research_cases.py:103-160).  s = 0 gives the fold's identity. */
int b2k_axis_reduce_f32(b2k_ctx *ctx, int32_t op, const float *x, float *y, int64_t batch, int64_t s, int64_t cols,
                        float div, const float *div_ptr, void *stream);
int b2k_row_op_f32(b2k_ctx *ctx, const b2k_row_params *params, const float *x, float *y, int64_t rows,
                   int64_t cols, int64_t ld_x, int64_t ld_y, void *stream);

/* Elementwise selective exponential (compile.py:2953-2965); exposed for the
 * subnormal-range accuracy tests. */
int b2k_selective_exp_f32(b2k_ctx *ctx, const float *x, float *y, int64_t n, void *stream);

/* --- 3xTF32 GEMM -----------------------------------------------------------
 * Replaces the reference's dense-contraction back ends: the 3xTF32
 * mma.sync emitter tf32_emitter.production_ptx (tf32_emitter.py:291-710,
 * arithmetic model :22-96) and the exact-FP32 SIMT plan emitter
 * compile.plan_simt_ptx (compile.py:9326-9611) selected for proven plans
 * (compile.py:9614-9625, tensor_core.py MatmulPlan :232-330).
 *
 * C[m, n] = relu?(A[m, k] * B + bias[n]) with every product expanded as
 * hi*hi + hi*lo + lo*hi of TF32 halves and FP32 accumulation.
 * A is row-major with leading dimension lda.  b_layout B2K_B_KN: B is
 * row-major [k, n] (ldb >= n); B2K_B_NK: B is stored transposed, row-major
 * [n, k] (ldb >= k).  Or-ing B2K_A_KM into b_layout says A is stored
 * transposed, row-major [k, m] (lda >= m; the pre-pass split transposes it;
 * not accepted by the host-array and batched calls).  bias may be NULL; relu
 * is 0 or 1.  C is row-major (ldc >= n).  Uses 2 * (m + n) * round_up(k, 32)
 * * 4 bytes of context scratch for the split operands, and, when the call
 * takes the K-chunk split (b2k_gemm_set_chunk_split, b2k_gemm_plan), a
 * second context arena of chunks * m * round_up(n, 4) * 4 bytes (chunks =
 * round_up(k, 32) / 256 rounded up) for the chunks' raw accumulators.  Both
 * arenas grow on first need (a synchronising cudaMalloc) and are then
 * reused. */
#define B2K_B_KN 0
#define B2K_B_NK 1
#define B2K_A_KM 2
int b2k_gemm_tf32x3(b2k_ctx *ctx, const float *a, const float *b, float *c, int64_t m, int64_t n, int64_t k,
                    int64_t lda, int64_t ldb, int64_t ldc, int32_t b_layout, const float *bias, int32_t relu,
                    void *stream);

/* b2k_gemm_tf32x3 with the product divided before the epilogue:
 *   C = relu?((A B) / div + bias),  div = *div_ptr (a one-element device
 *   buffer, read on the device) when div_ptr is non-NULL, else div_value.
 * The division is FP32 round-to-nearest of each accumulated element, as the
 * IR's `divide` of a contraction result (the scaled-score kernel of an
 * attention pipeline: scores = x @ y / scale[0]).  Takes the pre-pass split
 * path.  K = 0 returns B2K_EUNSUPPORTED. */
int b2k_gemm_tf32x3_scaled(b2k_ctx *ctx, const float *a, const float *b, float *c, int64_t m, int64_t n, int64_t k,
                           int64_t lda, int64_t ldb, int64_t ldc, int32_t b_layout, const float *bias, int32_t relu,
                           const float *div_ptr, float div_value, void *stream);

/* A batch of independent GEMMs with the arithmetic and epilogue of
 * b2k_gemm_tf32x3: C[i] = relu?(A[i] B[i] + bias) for i < batch, A[i] at
 * a + i * stride_a (elements), B[i] at b + i * stride_b, C[i] at
 * c + i * stride_c; bias (optional, n columns) is shared by the batch.  Each
 * stride must cover its matrix (stride_a >= m * lda, ...).  Replaces the
 * batched contractions the reference's tensor-core plan rejects
 * (tensor_core.py:284).  batch <= 65535; takes the pre-pass split path. */
int b2k_gemm_tf32x3_batched(b2k_ctx *ctx, const float *a, const float *b, float *c, int64_t batch, int64_t m,
                            int64_t n, int64_t k, int64_t lda, int64_t ldb, int64_t ldc, int64_t stride_a,
                            int64_t stride_b, int64_t stride_c, int32_t b_layout, const float *bias, int32_t relu,
                            void *stream);

/* --- attention ----------------------------------------------------------------
 * Replaces the reference's fused SIMT attention lowering (compile.py:7009-7966:
 * hoisted score rows, selective-exp softmax, P.V fold) for every head of a
 * batch: O[h] = softmax(Q[h] K[h]^T / scale) V[h] for h < bh, both contractions
 * as 3xTF32 on the tensor cores.  Q is [bh][s_q][d], V is [bh][s_kv][dv], O
 * is [bh][s_q][dv] (all row-major, contiguous).  k_layout B2K_K_SD: K is
 * [bh][s_kv][d]; B2K_K_DS: K is given transposed as [bh][d][s_kv] (the IR's
 * `kt`).  The divisor is *scale_div_ptr when that device pointer is non-NULL
 * (the IR's one-element `div_c1` buffer), else scale_div.  Head dims up to
 * 128 (d and dv) run one fused kernel (S and P never leave the SM); larger
 * ones run three batched passes through context scratch. */
#define B2K_K_SD 0
#define B2K_K_DS 1
int b2k_attention_tf32x3(b2k_ctx *ctx, const float *q, const float *k, const float *v, float *o, int64_t bh,
                         int64_t s_q, int64_t s_kv, int64_t d, int64_t dv, float scale_div,
                         const float *scale_div_ptr, int32_t k_layout, void *stream);
/* Process-wide choice of attention path where head dims allow the fused
 * kernel: 1 (default) the fused kernel with one CTA per query tile; 0 the
 * three-pass path (for comparisons).  Other values return B2K_EINVAL. */
int b2k_attention_set_fused(int mode);

/* --- rotary positions ----------------------------------------------------------
 * Rotates pairs (a, b) of a head's first `rot` elements by position * f_i:
 *   y_a = g (x_a cos - x_b sin),  y_b = g (x_b cos + x_a sin),  i < rot / 2,
 * with (a, b) = (i, i + rot / 2), or (2i, 2i + 1) when interleaved; the other
 * d - rot elements are copied.  f_i = theta^(-2i / rot) radians a position,
 * changed for contexts longer than the one a model was trained on by
 *   B2K_ROPE_NONE      nothing
 *   B2K_ROPE_LINEAR    f / factor
 *   B2K_ROPE_BASE      theta * factor^(rot / (rot - 2)) for theta: the slowest
 *                      pair is slowed by `factor`, the fastest not at all
 *   B2K_ROPE_RAMP      f (w + (1 - w) / factor), w = (t - low) / (high - low)
 *                      held to [0, 1], t = context * f / 2 pi: the turns the
 *                      pair makes over the trained context
 *   B2K_ROPE_LOG_RAMP  the same with log t, log low and log high
 * and g = magnitude.  No table bounds the positions: the plan holds f_i / 2 pi
 * as a 64-bit binary fraction of a turn, and position * turn modulo 2^64 is the
 * angle.  That is off by less than |position| * 2^-62 turns (the fraction's
 * error, with theta >= 1, factor >= 1 and, for the ramps, high >= 2 low), plus
 * 2^-32 turns and the rounding to FP32.  No counterpart in the reference. */
#define B2K_F32 0 /* element types of the operators below */
#define B2K_F16 1
#define B2K_BF16 2
#define B2K_ROPE_NONE 0
#define B2K_ROPE_LINEAR 1
#define B2K_ROPE_BASE 2
#define B2K_ROPE_RAMP 3
#define B2K_ROPE_LOG_RAMP 4
#define B2K_ROPE_MAX_PAIRS 128
#define B2K_MAX_HEAD_DIM 256
typedef struct b2k_rope_params {
  int32_t rot;         /* rotated elements of a head: even, 2 .. 256 */
  int32_t interleaved; /* 0: pairs (i, i + rot / 2); 1: pairs (2i, 2i + 1) */
  int32_t scaling;     /* B2K_ROPE_* */
  double theta;        /* > 0 */
  double factor;       /* > 0; unused by B2K_ROPE_NONE */
  double context;      /* ramps: trained context, tokens, > 0 */
  double low, high;    /* ramps: turns at or below `low` are slowed, at or above `high` kept; low < high */
  double magnitude;    /* g */
} b2k_rope_params;
typedef struct b2k_rope {
  int32_t rot, interleaved;
  float magnitude;
  int32_t reserved;
  uint64_t turn[B2K_ROPE_MAX_PAIRS]; /* f_i / 2 pi * 2^64, modulo 2^64 */
} b2k_rope;
/* Fill `out` from `params`: host arithmetic only (no device, no context).
 * B2K_EINVAL for parameters outside the ranges above. */
int b2k_rope_plan(const b2k_rope_params *params, b2k_rope *out);

/* A tensor [tokens][heads][d] whose d elements are contiguous: strides in
 * elements.  An input may repeat one token (stride_token < d); an output's
 * tokens and heads may not overlap, nor may an output and another operand
 * (B2K_EINVAL; b2k_heads_overlap is the test), but for those that an entry point
 * names. */
typedef struct b2k_heads {
  void *data;
  int64_t stride_token, stride_head;
  int32_t heads;
} b2k_heads;
/* 1 where rows of x and y ([tokens][heads][d] of `dtype` both), or two rows of
 * x (y == NULL), share an element, 0 where none do.  Exact where tokens lie the
 * same stride apart in x and y with a token's heads within it, or where x and y
 * have the same strides; of other tensors whose extents cross, 1.  Host
 * arithmetic on the addresses; -1 for extents below zero or an unknown type. */
int b2k_heads_overlap(const b2k_heads *x, const b2k_heads *y, int64_t tokens, int32_t d, int32_t dtype);
/* y[i] = rotary(x[i]) for i < count (1 .. 3) tensors of the same tokens, one
 * launch (queries and keys, say); positions [tokens], any sign.  transpose
 * = 1 applies the transposed rotation, with the same g: given the gradient
 * of the outputs it returns the gradient of the inputs.  y[i] may be x[i]
 * (the same data and strides), but may not overlap it or another tensor of the
 * call otherwise.  Products
 * and sums are FP32, rounded once to `dtype`.  tokens may be 0. */
int b2k_rotary(b2k_ctx *ctx, const b2k_rope *rope, int32_t dtype, int32_t count, const b2k_heads *x,
               const b2k_heads *y, const int64_t *positions, int64_t tokens, int32_t d, int32_t transpose,
               void *stream);

/* --- paged key / value cache -----------------------------------------------------
 * Keys and values live in pages of `page_size` tokens; element (page, row,
 * head, i) of k is at k + page * k_page + row * k_row + head * k_head + i
 * (strides in elements), so pages may be token-major [pages][page_size][heads][d],
 * head-major [pages][heads][page_size][d] or part of a larger buffer.
 *
 * A batch is `sequences` sequences whose new tokens are packed one after the
 * other: sequence b's are rows first[b] .. first[b + 1] - 1 (first does not
 * fall; none is allowed).  lengths[b] counts its own cached tokens with the
 * new ones, so new token j of n has own position lengths[b] - n + j, which
 * lies in page table[b * table_stride + position / page_size], row position %
 * page_size.  All sequences may share a prefix of prefix_len tokens, cached
 * once, in the pages of prefix_table in order; own positions follow it.
 * first, lengths, table and prefix_table are device memory, read when the
 * kernels run (a captured graph sees their values at replay); the other
 * members are host values.
 *
 * Indexes from device memory are checked on the device: a page outside [0,
 * pages), a position outside the table, a sequence with more new tokens than
 * max_new (or fewer than none) or a length above max_len touches no memory (the token is not
 * written, the key is left out, the row not computed) and the next
 * b2k_stream_sync of the context returns B2K_EINDEX.  No counterpart in the
 * reference. */
typedef struct b2k_paged_cache {
  void *k, *v;
  int32_t dtype;     /* B2K_F32, B2K_F16 or B2K_BF16; every operand's */
  int32_t page_size; /* tokens, >= 1 */
  int64_t pages;
  int32_t heads, d;  /* key / value heads; head dim, 1 .. B2K_MAX_HEAD_DIM */
  int64_t k_page, k_row, k_head;
  int64_t v_page, v_row, v_head;
} b2k_paged_cache;
typedef struct b2k_paged_batch {
  int32_t sequences;
  int32_t table_width;         /* pages in a row of the table */
  int64_t tokens;              /* rows of the packed tensors; rows from first[sequences] on are left alone */
  const int32_t *first;        /* [sequences + 1] */
  const int32_t *lengths;      /* [sequences] */
  const int32_t *table;        /* [sequences][table_width] */
  int64_t table_stride;        /* >= table_width */
  int32_t max_new, max_len;    /* upper bounds of the new tokens and of lengths[b]; sizes of the launches.
                                  Attention splits the keys by max_len: fastest near the longest length */
  int32_t prefix_len;
  const int32_t *prefix_table; /* [ceil(prefix_len / page_size)] */
} b2k_paged_batch;
/* The cache row of own position `position` under a table row of `table_width`
 * pages: page * page_size + row, or -1 where the kernels would refuse it.
 * Host arithmetic on host memory, by the kernels' own function. */
int64_t b2k_paged_slot(const int32_t *table_row, int32_t table_width, int64_t pages, int32_t page_size,
                       int64_t position);
/* Write the batch's new keys and values k, v [tokens][cache heads][d] into
 * the cache.  With a rope, keys are rotated on the way to position prefix_len
 * + own position, and, when q is not NULL, q [tokens][heads][d] is rotated
 * into q_out (which may be q) by the same launch.  Without one, k is copied
 * (q must be NULL).  No two new tokens may share a cache row, nor keys and
 * values an element. */
int b2k_paged_append(b2k_ctx *ctx, const b2k_rope *rope, const b2k_paged_cache *cache, const b2k_paged_batch *batch,
                     const b2k_heads *k, const b2k_heads *v, const b2k_heads *q, const b2k_heads *q_out,
                     void *stream);
/* Attention of the new tokens over the cache, with the prefix read once for
 * all sequences: new token j of sequence b sees the whole prefix and own
 * positions up to its own,
 *   o = sum_s softmax_s(q . k_s / scale_div) v_s,   0 < scale_div < inf, 1.45 / scale_div finite in FP32.
 * Query head h reads cache head h / (q heads / cache heads).  A row that sees
 * no key is zero.  FP32 softmax and sums; f16 and bf16 operands run on the
 * tensor cores, with the probabilities rounded to the operands' type.  Rows of a
 * page that hold no token may hold anything.  A later token's value that an
 * earlier one may not see is multiplied by zero there, so it has to be finite.
 * `workspace` (device memory of the caller's, `workspace_bytes` at least what
 * b2k_paged_attention_workspace says, 16-byte aligned; may be NULL when that
 * is 0) holds what parts of one row's keys have summed; calls that may run at
 * the same time need one each.  o may not overlap q. */
int b2k_paged_attention_workspace(b2k_ctx *ctx, const b2k_paged_cache *cache, const b2k_paged_batch *batch,
                                  int32_t q_heads, size_t *bytes);
int b2k_paged_attention(b2k_ctx *ctx, const b2k_paged_cache *cache, const b2k_paged_batch *batch, const b2k_heads *q,
                        const b2k_heads *o, float scale_div, void *workspace, size_t workspace_bytes, void *stream);
/* What a call with these operands launches on a GPU of `sms` SMs, under the
 * current setting below: host arithmetic only (no GPU; no pointer is
 * dereferenced, addresses are read for their alignment).  B2K_EINVAL and
 * B2K_EUNSUPPORTED where the call is refused. */
typedef struct b2k_paged_attention_plan_info {
  int32_t own_kernel, prefix_kernel; /* 0 plain cores, 1 warp MMAs, 2 tensor memory; prefix -1: no part of its own */
  int32_t own_splits, own_chunk;     /* splits of the sequences' own keys, keys of each */
  int32_t prefix_splits, prefix_chunk;
  int32_t joined;                    /* 1: each sequence reads the prefix with its own keys */
  int32_t streaming;                 /* plain cores: 1 the own part, 2 the prefix by the kernel that streams f32 (3: both) */
  int64_t workspace_bytes;           /* as b2k_paged_attention_workspace says */
} b2k_paged_attention_plan_info;
int b2k_paged_attention_plan(int32_t sms, const b2k_paged_cache *cache, const b2k_paged_batch *batch, const b2k_heads *q,
                             const b2k_heads *o, b2k_paged_attention_plan_info *out);
/* Process-wide choice of b2k_paged_attention's kernels, kept for comparisons
 * and tests: 0 (default) by operands and sizes; 1 the plain cores always; 2
 * warp MMAs, 3 tensor memory, wherever the operands (and for 3 with head dims
 * above 128 the page size: 8 to 128 that divides 128, or a multiple of it)
 * allow, and 1 or 2 elsewhere.  Other values return B2K_EINVAL.  A
 * workspace is asked for under the setting it is used with. */
int b2k_paged_attention_set_kernel(int mode);

/* --- verification of drafted tokens ------------------------------------------------
 * For each of `batch` sequences with `drafts` drafted tokens x_0 .. x_{n-1},
 * the target's probabilities p_0 .. p_n ([batch][drafts + 1][vocab]) and the
 * drafter's q_0 .. q_{n-1} ([batch][drafts][vocab]), contiguous FP32 as
 * b2k_row_softmax_f32 writes them (row strides ld_target, ld_draft >= vocab):
 * x_i is taken while u_accept[b][i] * q_i(x_i) < p_i(x_i); at the first i
 * that is not, one token is drawn from max(p_i - q_i, 0) (from p_i should
 * that be zero everywhere), and with all taken one from p_n.  Drawn from r:
 * the smallest t with r_0 + .. + r_t > u_sample[b] * sum(r), in 64 bits (the
 * last t with r_t > 0 should rounding leave none).  draft == NULL: the drafts
 * were certain (q_i(x_i) = 1, 0 elsewhere).  counts (may be NULL) holds each
 * sequence's own number of drafts, 0 .. drafts.  accepted [batch]; tokens
 * [batch][drafts + 1]: the taken drafts, the drawn token, then -1; neither may
 * overlap another array (from its first element to its last: B2K_EINVAL).  A drafted token outside [0, vocab) is never taken.  Every
 * draw follows its target distribution exactly.  No counterpart in the
 * reference. */
typedef struct b2k_drafts {
  const float *target, *draft;
  int64_t ld_target, ld_draft;
  const int32_t *drafted;      /* [batch][drafts] */
  const int32_t *counts;       /* [batch] or NULL */
  const float *u_accept;       /* [batch][drafts], in [0, 1) */
  const float *u_sample;       /* [batch], in [0, 1) */
  int64_t batch, vocab;
  int32_t drafts;
} b2k_drafts;
int b2k_verify_drafts(b2k_ctx *ctx, const b2k_drafts *drafts, int32_t *accepted, int32_t *tokens, void *stream);

/* --- launch by descriptor ----------------------------------------------------
 * The reference's runner launches a compiled kernel with
 * cuLaunchKernel(fn, grid, block, smem, stream, params, NULL), `params` being
 * pointers to the values of the positional meta.json arguments in arg_order
 * (tools/local_runner.py:296-324; Emitter ABI binding compile.py:1995-2213).
 * b2k_launch takes that same `args` array -- a device-pointer argument's slot
 * points at its 64-bit address, an f32 scalar's slot at its value -- plus a
 * descriptor naming the B200 kernel and which positional arguments feed it.
 * The front end (frontend.py) fills the descriptor when it recognises an IR
 * kernel; meta's grid/block are validated there, not obeyed (the sm_89
 * geometry is not a B200 geometry).  zero_outputs stay with the caller, as in
 * the reference's runner.  Every failure is reported before launching. */
#define B2K_KIND_POINTWISE 1
#define B2K_KIND_ROW_SOFTMAX 2
#define B2K_KIND_ROW_OP 3
#define B2K_KIND_GEMM_3XTF32 4
#define B2K_KIND_ATTENTION_3XTF32 5
#define B2K_KIND_AXIS_REDUCE 6
#define B2K_KIND_GEMM_BATCHED 7
#define B2K_MAX_ROLES 12
#define B2K_NO_ARG (-1)
#define B2K_ROLE_PW_OUT 8
typedef struct b2k_kernel_desc {
  int32_t kind;
  /* Positional argument index of each operand role (B2K_NO_ARG if absent):
   *   POINTWISE   roles 0..n_inputs-1 input streams, B2K_ROLE_PW_OUT output
   *   ROW_SOFTMAX 0 x, 1 y
   *   ROW_OP      0 x, 1 y, 2 weight, 3 sum-divisor buffer,
   *               4 mean-square-divisor buffer, 5 epsilon buffer
   *   GEMM_3XTF32 0 A, 1 B, 2 C, 3 bias, 4 divisor buffer (b2k_gemm_tf32x3_scaled)
   *   ATTENTION   0 Q, 1 K, 2 V, 3 O, 4 divisor buffer
   *   AXIS_REDUCE 0 x, 1 y, 3 divisor buffer
   *   GEMM_BATCHED 0 A, 1 B, 2 C, 3 bias (contiguous [batch][rows][cols] operands) */
  int32_t role[B2K_MAX_ROLES];
  /* POINTWISE: n | ROW_*: rows, cols, ld_x, ld_y | GEMM: m, n, k, lda, ldb, ldc |
   * ATTENTION: bh, s_q, s_kv, d, dv | AXIS_REDUCE: batch, s, cols | GEMM_BATCHED: batch, m, n, k */
  int64_t dims[6];
  /* GEMM, GEMM_BATCHED: b_layout, relu | ATTENTION: k_layout | ROW_OP, AXIS_REDUCE: op */
  int32_t flags[4];
  /* ROW_OP: sum_div, ms_div, eps | ATTENTION: scale_div (when no buffer) |
   * AXIS_REDUCE: sum divisor (when no buffer) */
  float values[4];
  const b2k_pw_program *program; /* POINTWISE */
} b2k_kernel_desc;
int b2k_launch(b2k_ctx *ctx, const b2k_kernel_desc *desc, void *const *args, int32_t nargs, void *stream);

/* The same GEMM for callers that cannot allocate device memory: embedders
 * whose device memory belongs to another allocator or a pre-sized pool,
 * runtimes that plan every buffer up front, and code in a host callback or
 * library hook where a synchronising cudaMalloc is not allowed.  No
 * counterpart in the reference.  It takes no context and
 * allocates nothing: the operand split goes to a fixed scratch array inside
 * the library image (B2K_NOALLOC_SCRATCH_BYTES per device that loads the
 * library, kept until exit).  Problems with 2 * (m + n) * round_up(k, 32) * 4
 * bytes of split operands above that size return B2K_ESCRATCH and launch
 * nothing; extents beyond the 32-bit limits of b2k_gemm_tf32x3 return
 * B2K_EINVAL; K = 0 returns B2K_EUNSUPPORTED.  Runs on the calling thread's
 * current device and the given stream.  The first call on a device looks up
 * the scratch array's device address (cudaGetSymbolAddress) and keeps it;
 * make that first call on each device before any stream capture begins.
 * Every call on a device shares the one
 * array, so calls that overlap on the GPU (different streams, no ordering)
 * race and corrupt each other's results; calls on one stream are safe.  Each
 * call rewrites all the scratch it reads, so nothing needs clearing.  A
 * device-side bounded-wait expiry is not returned by this entry point (its
 * kernels are still running when it returns): the kernels record it in a
 * per-device word that b2k_gemm_noalloc_status reads.
 * Other return codes as b2k_gemm_tf32x3 (B2K_EINVAL, B2K_ECUDA). */
#define B2K_NOALLOC_SCRATCH_BYTES (32u << 20)
int b2k_gemm_tf32x3_noalloc(const float *a, const float *b, float *c, int64_t m, int64_t n, int64_t k,
                            int64_t lda, int64_t ldb, int64_t ldc, int32_t b_layout, const float *bias,
                            int32_t relu, void *stream);

/* Read and clear the device error word of b2k_gemm_tf32x3_noalloc on
 * `device`: B2K_ETIMEOUT when a bounded wait of one of its kernels expired
 * since the last query (the word is then cleared), B2K_OK when none did,
 * B2K_EINVAL for a device index out of range, B2K_ECUDA on a CUDA error.
 * Synchronise the streams of the calls to be checked first; the calling
 * thread's current device is left as it was.  No counterpart in the
 * reference (its runner retires a worker on any CUDA error). */
int b2k_gemm_noalloc_status(int32_t device);

/* --- multi-GPU: one problem over the GPUs of a node -------------------------
 * One process per GPU, each with its own b2k_ctx and one NCCL communicator
 * (NCCL is opened at run time; without it these calls return
 * B2K_EUNSUPPORTED and everything else works).  The reference is single-GPU
 * (tools/local_runner.py:246-342 drives one device); each workload of its hot
 * path splits into independent units, so a call takes this rank's shard of
 * the inputs and returns the whole output on every rank:
 *   shard of `units` for rank r = b2k_mgpu_partition(units, world, r, align):
 *   contiguous, every shard but the last a multiple of `align`, the last
 *   taking the remainder (4097 rows over 8 ranks: seven of 512, one of 513).
 * Collectives run on a stream of the handle's own and overlap the compute on
 * the caller's stream; the caller's stream waits for them at the end of each
 * call.  Calls on one handle are ordered like any other stream work.  Every
 * rank must make the same calls in the same order.  Returns B2K_ENCCL after
 * an NCCL error and B2K_ETIMEOUT when a bounded wait expires; the handle is
 * then aborted and only b2k_mgpu_destroy remains valid. */
typedef struct b2k_mgpu b2k_mgpu;
#define B2K_MGPU_ID_BYTES 128
int b2k_mgpu_partition(int64_t units, int32_t world, int32_t rank, int64_t align, int64_t *start, int64_t *count);
/* Rendezvous token: one rank makes it; the caller hands the 128 bytes to
 * every rank by its own channel (a file, a socket, a process-group broadcast). */
int b2k_mgpu_unique_id(void *id);
/* Join the communicator of `world` ranks as `rank` on ctx's device.  Returns
 * B2K_ETIMEOUT (nothing left behind) if the ranks have not all joined within
 * timeout_ms. */
int b2k_mgpu_init(b2k_ctx *ctx, int32_t world, int32_t rank, const void *id, int64_t timeout_ms, b2k_mgpu **out);
int b2k_mgpu_destroy(b2k_mgpu *mg);
/* Wait for the work issued on `stream` (the calls' collectives included),
 * at most timeout_ms: a collective whose peer has gone (a rank that exited
 * or stopped calling) ends in B2K_ETIMEOUT or B2K_ENCCL, not a hang. */
int b2k_mgpu_sync(b2k_mgpu *mg, void *stream, int64_t timeout_ms);
/* C = relu?(A B + bias) for C [m][n] (row-major, complete on every rank).
 * a_rows: this rank's rows of A, partition(m, world, rank, align), row-major
 * [rows][k] contiguous.  b: B on rank 0 only (other ranks may pass NULL),
 * [k][n] (B2K_B_KN) or [n][k] (B2K_B_NK), contiguous.  bias: [n] on every
 * rank, or NULL.  B is broadcast in `panels` column panels (1..16): panel
 * p's GEMM waits only for panel p, and panel p's C is gathered while panel
 * p + 1 computes; with one panel rank 0 broadcasts from `b` itself (read
 * only, never written).  Replaces a launch of the reference's GEMM plan
 * (tensor_core.py:232-330) by its row-partitioned form. */
int b2k_mgpu_gemm_tf32x3(b2k_mgpu *mg, const float *a_rows, const float *b, float *c, int64_t m, int64_t n,
                         int64_t k, int64_t align, int32_t b_layout, const float *bias, int32_t relu, int32_t panels,
                         void *stream);
/* Row softmax of a [rows][cols] matrix: x_rows is this rank's rows
 * (partition(rows, world, rank, 1)), y the whole output.  The gathers run
 * per piece (1..16; equal shards only, else one piece), piece i while piece
 * i + 1 computes. */
int b2k_mgpu_row_softmax_f32(b2k_mgpu *mg, const float *x_rows, float *y, int64_t rows, int64_t cols,
                             int32_t pieces, void *stream);
/* A pointwise program over n elements: non-broadcast input r holds this
 * rank's elements, partition(n, world, rank, align) (plus offset[r] elements
 * of window), broadcast inputs their one element; out is the whole output. */
int b2k_mgpu_pointwise_f32(b2k_mgpu *mg, const b2k_pw_program *program, const float *const *inputs, float *out,
                           int64_t n, int64_t align, int32_t pieces, void *stream);
/* Attention over bh heads: q, k ([heads][s_kv][d]) and v are this rank's
 * heads, partition(bh, world, rank, 1); o [bh][s_q][dv] the whole output. */
int b2k_mgpu_attention_tf32x3(b2k_mgpu *mg, const float *q, const float *k, const float *v, float *o, int64_t bh,
                              int64_t s_q, int64_t s_kv, int64_t d, int64_t dv, float scale_div, int32_t pieces,
                              void *stream);

/* Select the GEMM kernel variant for subsequent calls (process-wide; for
 * tuning and benchmarking): 0 = 128x256 tile, 128-byte swizzle, 2 stages;
 * 1 (default) = 128x256, 64-byte swizzle, 4 stages, or the tile of variant 3
 * or 2 when its tiles cover the output in clearly less estimated time (fewer
 * waves over the SMs: a row shard of a multi-GPU GEMM); every width gives the
 * same bits; 2 = 128x128, 128-byte
 * swizzle, 3 stages; 3 = 128x192, 64-byte swizzle, 5 stages.  Outputs at
 * most 128 columns wide always use 2.  For the in-kernel split kernels
 * (b2k_gemm_set_fused_split) variant 2 selects 128-wide tiles and every
 * other variant 192-wide ones.  No counterpart in the reference, whose plan
 * geometry comes from the IR. */
int b2k_gemm_set_variant(int variant);

/* Chunk split of the pre-pass GEMM kernel (process-wide; for tuning and
 * tests): 1 (default) = where the estimate says it is faster, 0 = never,
 * 2 = wherever it applies.  It applies to single (not batched) calls with at
 * least two 256-wide K chunks, made through a context: every 128 x 128 output
 * tile is computed as one CTA per K chunk, each storing its chunk's raw
 * accumulator in a context-owned arena, and a second kernel folds the chunks
 * in order and applies the epilogue -- the fold the unsplit kernel makes --
 * so the result is the same bits.  It fills the GPU when the output has few
 * tiles and K is long (a row shard of the ragged GEMM on eight GPUs, a
 * 256 x 512 x 4096 product).  The allocation-free entry point and the
 * host-array calls never take it.  No counterpart in the reference (its
 * split-K variant uses atomics, whose order is not fixed). */
int b2k_gemm_set_chunk_split(int mode);

/* Which kernel path b2k_gemm_tf32x3 takes for a call with these operands on
 * a GPU of `sms` SMs, under the current settings (variant, split modes,
 * chunk split), decided by the dispatch's own functions.  Host arithmetic
 * only: it touches no GPU and dereferences no pointer (a and b are read for
 * their alignment).  A divided product (b2k_gemm_tf32x3_scaled) always takes
 * split mode 0.  B2K_EINVAL for the arguments b2k_gemm_tf32x3 refuses, and
 * for m, n or k of 0 (nothing is launched then). */
typedef struct {
  int32_t split_mode;  /* 0 both operands pre-split, 1 A split in the kernel,
                          2 B split in the kernel (C^T = B^T A^T) */
  int32_t tile_width;  /* the kernel's tile width: output columns, or output
                          rows in mode 2 */
  int32_t chunk_split; /* 1: one CTA per (128 x 128 tile, 256-wide K chunk),
                          then the in-order fold */
  int32_t chunks;      /* 256-wide K chunks of the call */
} b2k_gemm_plan_info;
int b2k_gemm_plan(int32_t sms, const float *a, const float *b, int64_t m, int64_t n, int64_t k, int64_t lda,
                  int64_t ldb, int32_t b_layout, b2k_gemm_plan_info *out);
/* Process-wide choice of where b2k_gemm_tf32x3 (and the no-alloc variant)
 * split operands into TF32 hi/lo halves:
 *   3            direct: A is staged raw by TMA and split inside the
 *                tensor-core kernel into tensor memory, which the MMAs read A
 *                from (128 x 192 tiles, 128 x 128 for n <= 128); B is split
 *                once by a pre-pass.  Needs A 16-byte aligned, not stored
 *                transposed, with a row stride that is a multiple of 4
 *                elements, and K >= 16.
 *   2            transposed: the kernel computes C^T = B^T A^T, so B is staged
 *                raw and split inside the kernel into tensor memory (a [K, N]
 *                B read in 128-column boxes, a [N, K] B by rows) and only A is
 *                split by the pre-pass; the epilogue writes C transposed back
 *                into row-major C.  For short, wide outputs (a row shard of a
 *                large GEMM) it splits the small operand and tiles the output
 *                128 columns by 128 or 192 rows.  Needs B 16-byte aligned with
 *                a row stride that is a multiple of 4 elements, K >= 16 and,
 *                for a [K, N] B, N >= 128.
 *   1 (default)  whichever of 0, 2 and 3 the operands allow and an estimate
 *                of (waves of tiles over the SMs) x (tile time) + (pre-pass
 *                bytes) says is fastest.
 *   0            both operands split by the pre-pass (128 x 256 tiles).
 * Calls whose operands do not meet a mode's conditions take the pre-pass
 * path.  Every path runs the same three TF32 products per 8-wide K step with
 * the same 256-wide chunked FP32 accumulation.  Returns B2K_EINVAL for other
 * values.  No counterpart in the reference. */
int b2k_gemm_set_fused_split(int mode);

/* --- pipelined host-array calls ----------------------------------------------
 * The runner's per-request host flow -- copy every input in, launch, copy
 * every output out (tools/local_runner.py:287-338) -- as one call that
 * overlaps the three.  Arguments are HOST pointers with the meaning of the
 * device entry point of the same name.  Inputs are cut into slabs (rows of
 * the softmax or of A, element ranges, batch*heads); slab i is copied in on
 * a context-owned host-to-device stream, its kernels run on `stream` once it
 * has landed, and its output is copied out on a device-to-host stream while
 * later slabs compute and copy in.  Device staging memory belongs to the
 * context.  Asynchronous like the device entry points: the host outputs are
 * complete once `stream` is synchronised (b2k_stream_sync).  Host buffers
 * should be page-locked (b2k_host_alloc); pageable buffers work with less
 * overlap.  Results equal the device entry points' bit for bit. */
int b2k_row_softmax_f32_host(b2k_ctx *ctx, const float *x, float *y, int64_t rows, int64_t cols, int64_t ld_x,
                             int64_t ld_y, void *stream);
int b2k_pointwise_f32_host(b2k_ctx *ctx, const b2k_pw_program *program, const float *const *inputs, float *out,
                           int64_t n, void *stream);
int b2k_gemm_tf32x3_host(b2k_ctx *ctx, const float *a, const float *b, float *c, int64_t m, int64_t n, int64_t k,
                         int64_t lda, int64_t ldb, int64_t ldc, int32_t b_layout, const float *bias, int32_t relu,
                         void *stream);
/* Host variant of b2k_attention_tf32x3 with the scale divisor by value. */
int b2k_attention_tf32x3_host(b2k_ctx *ctx, const float *q, const float *k, const float *v, float *o, int64_t bh,
                              int64_t s_q, int64_t s_kv, int64_t d, int64_t dv, float scale_div, int32_t k_layout,
                              void *stream);

#ifdef __cplusplus
}
#endif

#endif /* B200K_H */
