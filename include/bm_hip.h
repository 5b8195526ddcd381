/*
 * bm_hip.h -- C ABI of the MI355X (gfx950) BitLinear backend.
 *
 * Drop-in for the ternary BitLinear hot path of jserv/bitmamba.c.  The
 * backend takes the slot the Metal backend fills in the reference
 * (src/metal/bm_metal.h:14-99) and registers its kernels in the reference's
 * plugin table kernel_dispatch_t g_kernels (src/dispatch.h:86-100).
 *
 * Every entry point takes plain pointers and sizes.  Functions whose names
 * start with hip_ have exactly the function-pointer types of the dispatch
 * table and take HOST pointers (synchronous, like the CPU kernels they
 * replace).  Functions ending in _dev take DEVICE pointers and a HIP stream
 * (void *, NULL = the library's stream) and are asynchronous.
 *
 * Errors: contract violations (dimension mismatch, non-BitNet weights) exit
 * the process like BITLINEAR_CHECK (src/bitmamba.h:219-231); a HIP runtime
 * failure inside a hip_ kernel entry point also prints and exits -- outputs
 * are never silently zeroed (contrast src/metal/bm_metal.c:549-553).
 * Lifecycle and _dev functions return false / a negative code instead, with
 * the reason in bm_hip_last_error().
 */
#pragma once

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The reference's tensor view (src/bitmamba.h:65-74).  The layout below is
 * the one the reference compiles; define BM_HIP_HAVE_TENSOR_T when the
 * reference's own bitmamba.h is already included. */
#ifndef BM_HIP_HAVE_TENSOR_T
struct tensor {
    const float *data;          /* float32 weights */
    const uint8_t *packed_data; /* packed 2-bit weights, [rows][ceil(cols/4)] */
    int rows;
    int cols;
    size_t n_elements;
    bool is_bitnet;
    float scale;
};
#endif

/* ------------------------------------------------------------------ */
/* Lifecycle -- mirrors src/metal/bm_metal.h:14-24, 44-45               */
/* ------------------------------------------------------------------ */

/* bm_metal_init (src/metal/bm_metal.h:15): selects device 0, creates the
 * library stream.  false if no gfx950 device is usable. */
bool bm_hip_init(void);
/* bm_metal_available (src/metal/bm_metal.h:18) */
bool bm_hip_available(void);
/* bm_metal_set_mmap (src/metal/bm_metal.h:24): registers a model image.
 * When the image parses as BIT2 (src/model.c:477-932 layout) every packed
 * tensor is copied once into its own 256-byte-aligned device buffer with
 * the 2-bit code 11 rewritten to 10 (same value, src/quantization.c:27-31),
 * and every float tensor is copied too; hip_* calls then find them by host
 * pointer.  Tensors outside a registered image are uploaded on every call
 * (their host memory may be reused for other data).  Registered host memory
 * must not change afterwards. */
bool bm_hip_set_mmap(const void *base, size_t size);
/* bm_metal_cleanup (src/metal/bm_metal.h:45) */
void bm_hip_cleanup(void);
/* Reason for the last false / negative return. */
const char *bm_hip_last_error(void);

/* ------------------------------------------------------------------ */
/* Dispatch-table kernels (host pointers, synchronous)                  */
/* ------------------------------------------------------------------ */

/* rms_norm_fn_t (src/dispatch.h:20-23); semantics of scalar_rms_norm
 * (src/kernel.c:72-129), bit-exact. */
float hip_rms_norm(const float *x, int size, const float *weight, float *out);

/* bitlinear_forward_fn_t (src/dispatch.h:25-31); semantics of
 * scalar_bitlinear_forward (src/kernel.c:346-448), bit-exact fp32 output.
 * x_norm_buf[n] and x_quant_buf[n] receive what the scalar kernel leaves
 * there. */
void hip_bitlinear_forward(const float *x,
                           int n,
                           const struct tensor *w,
                           const struct tensor *norm_w,
                           float *out,
                           float *x_norm_buf,
                           int8_t *x_quant_buf);

/* bitlinear_forward_batch_fn_t (src/dispatch.h:33-42); semantics of
 * scalar_bitlinear_forward_batch (src/kernel.c:322-338).  x_norm_buf holds
 * the last token's normalized input afterwards, as in the reference. */
void hip_bitlinear_forward_batch(const float *x_batch,
                                 int n_tokens,
                                 int n,
                                 const struct tensor *w,
                                 const struct tensor *norm_w,
                                 float *out_batch,
                                 float *x_norm_buf,
                                 int8_t *x_quant_batch,
                                 int quant_stride);

/* Layout mirror of kernel_dispatch_t (src/dispatch.h:87-95). */
typedef struct {
    void *rms_norm;
    void *bitlinear_forward;
    void *bitlinear_forward_batch;
    void *bitlinear_prepare;
    void *bitlinear_row_worker;
    void *ssm_inner;
    const char *name;
} bm_hip_dispatch_t;

/* The GPU branch of dispatch_init (src/dispatch.c:15-52): sets rms_norm,
 * bitlinear_forward and bitlinear_forward_batch to the hip_ entries,
 * bitlinear_prepare and bitlinear_row_worker to NULL (so block_step takes
 * its unfused path, src/block.c:280, 361-371, and the LM head calls
 * bitlinear_forward, src/model.c:1258-1262), keeps ssm_inner, and sets
 * name = "hip".  Returns false (table untouched) if the backend is not
 * available. */
bool bm_hip_register(bm_hip_dispatch_t *table);

/* bm_metal_bitlinear_forward_batch (src/metal/bm_metal.h:31-42): the same
 * computation as hip_bitlinear_forward_batch from raw tensor fields. */
void bm_hip_bitlinear_forward_batch(const float *x_batch,
                                    int n_tokens,
                                    int n,
                                    const uint8_t *packed_data,
                                    int rows,
                                    int cols,
                                    float w_scale,
                                    const float *norm_weight,
                                    float *out_batch,
                                    float *x_norm_buf,
                                    int8_t *x_quant_batch,
                                    int quant_stride);

/* ------------------------------------------------------------------ */
/* Batch context: the Metal backend's prefill batching                  */
/* (src/metal/bm_metal.h:57-99), driven as model_prefill_metal drives   */
/* it (src/model.c:934-1041).                                           */
/* ------------------------------------------------------------------ */

/* Buffer ids (BM_BUF_X .. BM_BUF_OUT, src/metal/bm_metal.h:58-63) */
enum {
    BM_HIP_BUF_X = 0,    /* n_tokens * d_model floats */
    BM_HIP_BUF_PROJ = 1, /* n_tokens * max_proj floats */
    BM_HIP_BUF_Y = 2,    /* n_tokens * d_inner floats */
    BM_HIP_BUF_OUT = 3,  /* n_tokens * d_model floats */
};
typedef struct bm_hip_batch_ctx bm_hip_batch_ctx_t;

/* bm_metal_batch_begin: the four buffers, zeroed.  NULL before bm_hip_init
 * or on a failed allocation (the caller falls back to the CPU). */
bm_hip_batch_ctx_t *bm_hip_batch_begin(int n_tokens,
                                       int d_model,
                                       int max_proj,
                                       int d_inner,
                                       int quant_stride);
/* bm_metal_batch_ptr: host pointer to a buffer (NULL for another id).  The
 * buffers live on the device with a pinned host copy: what the caller
 * writes there before bm_hip_submit_and_wait reaches the steps of that
 * submit, and what the steps write is there when it returns. */
float *bm_hip_batch_ptr(bm_hip_batch_ctx_t *ctx, int buf_id);
/* bm_metal_encode_bitlinear: queue RMSNorm + int8 + the blocked product of
 * the n_tokens rows of src (X or Y, row stride input_dim) into dst (PROJ or
 * OUT, row stride rows), bit-exact with scalar_bitlinear_forward_batch
 * (src/kernel.c:322-338).  Runs nothing.  False, as in Metal, for a bad id,
 * cols % 16 != 0, no image registered by bm_hip_set_mmap, packed_data or
 * norm_weight outside it; also when input_dim != cols or the rows do not
 * fit the buffers. */
bool bm_hip_encode_bitlinear(bm_hip_batch_ctx_t *ctx,
                             int src_id,
                             int input_dim,
                             const uint8_t *packed_data,
                             int rows,
                             int cols,
                             float w_scale,
                             const float *norm_weight,
                             int dst_id);
/* bm_metal_encode_residual: queue X[i] += OUT[i] for i < count. */
void bm_hip_encode_residual(bm_hip_batch_ctx_t *ctx, int count);
/* bm_metal_submit_and_wait: run the queued steps in order and wait; a
 * failure is reported on stderr ("[HIP] Batch submit error") and in
 * bm_hip_last_error(). */
void bm_hip_submit_and_wait(bm_hip_batch_ctx_t *ctx);
/* bm_metal_batch_end */
void bm_hip_batch_end(bm_hip_batch_ctx_t *ctx);

/* ------------------------------------------------------------------ */
/* Device memory helpers (for callers without a HIP runtime of their    */
/* own; no counterpart in the reference)                                */
/* ------------------------------------------------------------------ */
void *bm_hip_malloc(size_t bytes);
void bm_hip_free(void *dev);
int bm_hip_memcpy_h2d(void *dev, const void *host, size_t bytes);
int bm_hip_memcpy_d2h(void *host, const void *dev, size_t bytes);
int bm_hip_memset(void *dev, int value, size_t bytes);
int bm_hip_synchronize(void);
/* Rewrites 2-bit code 11 to 10 in place (device buffer of `bytes`). */
int bm_hip_canonicalize_dev(uint8_t *packed, size_t bytes, void *stream);

/* Timing and calibration (no reference counterpart; the reference times
 * with CLOCK_MONOTONIC, src/utils.c:90-95): HIP events on a stream (NULL =
 * the library's stream), and a plain 16-byte copy kernel whose HBM counters
 * calibrate traffic measurements. */
void *bm_hip_stream(void);
void *bm_hip_event_create(void);
void bm_hip_event_destroy(void *ev);
int bm_hip_event_record(void *ev, void *stream);
float bm_hip_event_elapsed_ms(void *start, void *stop);
int bm_hip_copy_dev(void *dst, const void *src, size_t bytes, void *stream);
/* int8 MFMA ceiling: `blocks` blocks of 256 threads, each wave `iters` x 16
 * v_mfma_i32_32x32x32_i8 (65536 ops each); ternary != 0 uses hashed int8
 * activations against codes 0..2 like the prefill GEMM.  `sink` (one int,
 * device) is written only on an impossible value. */
int bm_hip_mfma_peak_dev(int blocks, int iters, int ternary, int *sink, void *stream);

/* ------------------------------------------------------------------ */
/* Device-pointer kernels (asynchronous on `stream`)                    */
/* ------------------------------------------------------------------ */

/* Per-token RMSNorm + absmax int8 quantization, bit-exact with
 * src/kernel.c:72-129 + 356-386, for M tokens of n values (row stride
 * x_stride floats).  Writes x_quant[m*quant_stride + i] and scale_x[m];
 * x_norm (nullable) gets [m*n + i].  Also fills the activation workspace
 * `act` (bm_hip_act_bytes(M, n) bytes) used by the _dev products below. */
size_t bm_hip_act_bytes(int M, int n);
int bm_hip_quantize_dev(const float *x,
                        int M,
                        int n,
                        int x_stride,
                        const float *norm_w,
                        float *x_norm,
                        int8_t *x_quant,
                        int quant_stride,
                        float *scale_x,
                        void *act,
                        void *stream);

/* Fast mode of the same (opt-in; not the reference's bits): the sum of
 * squares as one pairwise tree over the n values -- the reduction class of
 * the Metal backend's rms_norm_quantize (src/metal/bm_shaders.metal:40-60)
 * -- instead of the scalar kernel's four sequential chains
 * (src/kernel.c:77-89).  For n = 1024, 2048, 4096; other n give the
 * sequential sum. */
int bm_hip_quantize_fast_dev(const float *x,
                             int M,
                             int n,
                             int x_stride,
                             const float *norm_w,
                             float *x_norm,
                             int8_t *x_quant,
                             int quant_stride,
                             float *scale_x,
                             void *act,
                             void *stream);

/* Ternary BitLinear product on quantized activations (the act workspace
 * from bm_hip_quantize_dev): out[m*N + r] (fp32) with the scalar kernel's
 * 1024-column block epilogue (src/kernel.c:255-256, 407-447), bit-exact.
 * `canonical` != 0 promises the packed bytes hold no code 11. */
int bm_hip_bitlinear_act_dev(const void *act,
                             const float *scale_x,
                             int M,
                             const uint8_t *packed,
                             int N,
                             int K,
                             float w_scale,
                             int canonical,
                             float *out,
                             void *stream);

/* Quantize + product in one call (device pointers): scalar_bitlinear_
 * forward_batch semantics for M tokens. `act` as above.  One token on
 * canonical weights (K % 64 == 0, K <= 8192) runs as a single launch that
 * leaves `act` untouched. */
int bm_hip_bitlinear_dev(const float *x,
                         int M,
                         int K,
                         const float *norm_w,
                         const uint8_t *packed,
                         int N,
                         float w_scale,
                         int canonical,
                         float *out,
                         int8_t *x_quant,
                         int quant_stride,
                         float *scale_x,
                         void *act,
                         void *stream);

/* No counterpart in the reference: bm_hip_bitlinear_dev without any
 * allocation, for callers that cannot allocate (code under HIP stream
 * capture, tight serving loops).  The per-token scale and the activation
 * workspace (or int8 copy) live in a device array of the library's own,
 * bm_hip_noalloc_scratch_bytes() = 8 MiB per GPU, held until the process
 * ends; a call needing more (M * (K-row workspace) beyond it) returns -2.
 * Needs bm_hip_init() first (-1 otherwise).  Calls that overlap on one GPU
 * share the array and race.  Same semantics and output as
 * bm_hip_bitlinear_dev (out[m*N + r], bit-exact). */
int bm_hip_bitlinear_noalloc_dev(const float *x,
                                 int M,
                                 int K,
                                 const float *norm_w,
                                 const uint8_t *packed,
                                 int N,
                                 float w_scale,
                                 int canonical,
                                 float *out,
                                 void *stream);
size_t bm_hip_noalloc_scratch_bytes(void);

/* Exact int32 product of int8 activations and ternary weights:
 * out[m*N + r] = sum_k xq[m*ldx + k] * decode(W[r][k]) (stress shape;
 * activations need no quantization).  M = 1 (K % 64 == 0, K <= 8192) runs
 * as one GEMV launch that reads xq itself and leaves `act` untouched; few
 * tokens (K % 128 == 0, rows of xq on 16 bytes) one int8 MFMA launch that
 * also reads xq itself; other shapes prepare `act` first and run the int8
 * MFMA GEMM.  Needs bm_hip_i8_act_bytes(M, K) bytes of `act`. */
size_t bm_hip_i8_act_bytes(int M, int K);
int bm_hip_ternary_gemm_i32_dev(const int8_t *xq,
                                int M,
                                int ldx,
                                const uint8_t *packed,
                                int N,
                                int K,
                                int canonical,
                                int32_t *out,
                                void *act,
                                void *stream);

/* ------------------------------------------------------------------ */
/* Batched recurrence on device buffers (asynchronous on `stream`): the */
/* short causal convolution and the selective scan between in_proj and  */
/* out_proj, for many sequences at once, and the slots that hold their  */
/* state.  The mathematics of scalar_ssm_inner (src/kernel.c:34-70) and */
/* ssm_batch_worker (src/block.c:127-160) with d_state values per       */
/* channel and B, C shared by groups of heads; n_groups = n_heads and   */
/* d_state = 1 are the reference's block.  Sums run in another order    */
/* than the scalar kernels': results agree to fp32 rounding, they are   */
/* not the reference's bits (the device-resident model below keeps      */
/* those).                                                              */
/*                                                                      */
/* Common to the calls:                                                 */
/* - Tensors of the descriptor's `type` are read and written at any     */
/*   row stride (in elements, below 2^24) and any element alignment;    */
/*   everything is computed in fp32 or more, y is rounded once.  For a  */
/*   bf16 y of prompts with d_state > 8 two operands of its sums carry  */
/*   16 bits (2^-17 of each term) and the gate is good to 2^-20, from   */
/*   |z| = 8 on to |z| 2^-23; its own rounding is up to 2^-8.           */
/* - At most 2^20 sequences and 2^30 - 1 rows; 2^16 sequences with a    */
/*   list of slots, whose search for repeated entries grows with their  */
/*   square (it is small up to about a thousand).                       */
/* - Prompts are joined rows: sequence b has rows seq_start[b] ..       */
/*   seq_start[b + 1] - 1 (device, n_seqs + 1 ascending entries;        */
/*   NULL for one sequence of n_tokens rows).  Entries are clamped to   */
/*   0..n_tokens.  Rows that belong to no sequence are not touched.     */
/*   A call without rows still starts fresh sequences' slots; x, y and  */
/*   the other tensors with a row per token may then be NULL.           */
/* - Single tokens (_step): row b is the next token of sequence b;      */
/*   seq_start, fresh and n_tokens are not read.                        */
/* - The state of sequence b is slot slots[b] of the pool (device;      */
/*   NULL: slot b), carried from call to call: read, and replaced by    */
/*   the state after the sequence's last token.  A sequence whose entry */
/*   is outside 0..n_slots-1, or that an earlier sequence of the call   */
/*   also names, is padding: its rows of y and every slot stay as they  */
/*   are.  fresh[b] != 0 (device, nullable) starts sequence b from      */
/*   zeros whatever its slot holds.  state = NULL starts every sequence */
/*   from zeros and keeps nothing (slots and fresh are not read).       */
/* - y must not overlap the inputs or the pool; the step calls may      */
/*   write y over x itself (same address and stride).                   */
/* - Calls allocate nothing and may be captured into a graph; a replay  */
/*   reads seq_start, slots and fresh as they are then.  Calls on       */
/*   different streams need workspaces and slots of their own.          */
/* - 0, -2 for arguments that do not fit (nothing is launched), -1 for  */
/*   a HIP error; the reason is in bm_hip_last_error().                 */
/* ------------------------------------------------------------------ */
enum { BM_HIP_F32 = 0, BM_HIP_BF16 = 1, BM_HIP_F16 = 2 };

/* y[t][c] = act(bias[c] + sum_k w[k][c] * x[t - (width - 1) + k][c]), per
 * sequence; rows before its first token are the slot's rows. */
typedef struct {
    int type;                 /* of x and y */
    int channels, width;      /* width 2..4 taps */
    int silu;                 /* act(v) = v / (1 + exp(-v)), else v */
    int n_seqs, n_tokens;
    const int32_t *seq_start; /* device [n_seqs + 1], or NULL */
    const int32_t *slots;     /* device [n_seqs], or NULL */
    const uint8_t *fresh;     /* device [n_seqs], or NULL */
    const void *x;
    int64_t x_stride;
    const float *w;           /* [width][channels], the last row is the token's own tap */
    const float *bias;        /* [channels], or NULL */
    float *state;             /* slot i at state + i * state_stride: [width - 1][channels], oldest row first */
    int64_t state_stride;
    int n_slots;
    void *y;
    int64_t y_stride;
} bm_hip_conv_t;

int bm_hip_conv_dev(const bm_hip_conv_t *op, void *stream);
int bm_hip_conv_step_dev(const bm_hip_conv_t *op, void *stream);

/* Per head h of group g = h / (n_heads / n_groups), with d = dt[t][h] +
 * dt_bias[h], taken through log(1 + exp(d)) if dt_softplus, and a =
 * exp(A[h] * d).  A channel whose x is infinite or NaN is one of the two
 * from that row on; earlier rows, other channels and sequences are not
 * reached.  With d_state > 8, fp32 values of 2^128 - 2^119 and more count
 * as infinite.
 *   S[p][n] = a * S[p][n] + d * x[t][h][p] * B[t][g][n]
 *   y[t][h][p] = (sum_n C[t][g][n] * S[p][n] + D[h][p] * x[t][h][p])
 *                * z[t][h][p] / (1 + exp(-z[t][h][p])) */
typedef struct {
    int type;                      /* of x, B, C, dt, z, y */
    int n_heads, head_dim;         /* x, z, y rows: [n_heads][head_dim] */
    int n_groups, d_state;         /* B, C rows: [n_groups][d_state]; n_groups divides n_heads, d_state <= 256 */
    int dt_softplus;
    int n_seqs, n_tokens;
    const int32_t *seq_start;      /* device [n_seqs + 1], or NULL */
    const int32_t *slots;          /* device [n_seqs], or NULL */
    const uint8_t *fresh;          /* device [n_seqs], or NULL */
    const void *x, *B, *C, *dt, *z; /* z: NULL for no gate */
    int64_t x_stride, B_stride, C_stride, dt_stride, z_stride;
    const float *A;                /* [n_heads]; at most 0 for states that stay bounded */
    const float *dt_bias;          /* [n_heads], or NULL */
    const float *D;                /* [n_heads][head_dim], or NULL */
    float *state;                  /* slot i at state + i * state_stride: [n_heads][head_dim][d_state] */
    int64_t state_stride;
    int n_slots;
    void *y;
    int64_t y_stride;
} bm_hip_ssm_t;

/* Prompts.  workspace: bm_hip_ssm_workspace_bytes(op) bytes of device
 * memory on 256 bytes with any contents (NULL where that is 0; it depends
 * on the sizes of op alone, not on the pointers).  A workspace of an op
 * serves every call whose n_seqs and n_tokens are both no larger, with the
 * same n_heads, head_dim and d_state. */
size_t bm_hip_ssm_workspace_bytes(const bm_hip_ssm_t *op);
int bm_hip_ssm_dev(const bm_hip_ssm_t *op, void *workspace, void *stream);
/* One token of each sequence. */
int bm_hip_ssm_step_dev(const bm_hip_ssm_t *op, void *stream);

/* The gated delta rule (no counterpart in the reference), for blocks whose
 * state is a table from keys to values: per head h of group g = h / (n_heads
 * / n_groups), with d = dt[t][h] + dt_bias[h], taken through log(1 + exp(d))
 * if dt_softplus, a = exp(min(A[h] * d, 0)), b = beta[t][h], taken through
 * 1 / (1 + exp(-b)) if beta_sigmoid, and q, k the rows of the group, each
 * divided by sqrt(sum of its squares + norm_eps) if qk_norm,
 *   S[p][n] = a * S[p][n]
 *   w[p] = b * (v[t][h][p] - sum_n S[p][n] * k[t][g][n])
 *   S[p][n] = S[p][n] + w[p] * k[t][g][n]
 *   y[t][h][p] = scale * sum_n S[p][n] * q[t][g][n]
 *                * z[t][h][p] / (1 + exp(-z[t][h][p]))
 * Rows, sequences, slots and streams as above; frozen != 0 reads the slots
 * and leaves them as they are: drafted tokens are scored, and the accepted
 * ones given again (bm_hip_verify_dev's split_start).
 *
 * Sequences of more than 32 rows are worked out 64 rows at a time, with
 * products of operands of 22 bits: S[p] and what is read from it are then
 * good to 2^-13 of the largest that S[p] and b * v[p] * k (as vectors) are
 * within such a chunk, 64 times better where the errors are independent.
 *
 * A key with b * (sum of k's squares) above 2 makes the rule grow without
 * end; qk_norm with b in 0..2 cannot.  Where such a growth passes fp32, the
 * head's rows of the sequence from up to 15 before on are infinite, NaN or
 * undefined.  Shorter sequences and single tokens take the sums of S[p] * k,
 * S[p] * q and k * q, and w[p] / |k|, in fp32 before anything is divided by
 * a length: these must not pass its range either.
 *
 * Where a head's a or b is NaN or b infinite, or the sum of k's squares is
 * either (in fp32), the head is NaN from that row on, y and state; where that
 * of q is, its y in that row.  An infinite or NaN v[p] or S[p][n] makes y[p]
 * and S[p] infinite or NaN from its row on.  Earlier rows, other p, other heads
 * and other sequences are not reached. */
typedef struct {
    int type;                      /* of q, k, v, dt, beta, z, y */
    int n_heads, head_dim;         /* v, z, y rows: [n_heads][head_dim] */
    int n_groups, d_state;         /* q, k rows: [n_groups][d_state]; n_groups divides n_heads, d_state <= 256 */
    int dt_softplus, beta_sigmoid, qk_norm, frozen;
    float norm_eps, scale;         /* norm_eps 2^-100 and more, read with qk_norm */
    int n_seqs, n_tokens;
    const int32_t *seq_start;      /* device [n_seqs + 1], or NULL */
    const int32_t *slots;          /* device [n_seqs], or NULL */
    const uint8_t *fresh;          /* device [n_seqs], or NULL */
    const void *q, *k, *v, *dt, *beta, *z; /* dt: NULL without A; beta: NULL for 1; z: NULL for no gate */
    int64_t q_stride, k_stride, v_stride, dt_stride, beta_stride, z_stride;
    const float *A;                /* [n_heads], or NULL for a = 1 */
    const float *dt_bias;          /* [n_heads], or NULL */
    float *state;                  /* slot i at state + i * state_stride: [n_heads][head_dim][d_state] */
    int64_t state_stride;
    int n_slots;
    void *y;
    int64_t y_stride;
} bm_hip_delta_t;

/* Prompts.  The workspace as bm_hip_ssm_dev's: any contents, on 256 bytes,
 * one of an op serves every call of no more sequences and rows with the same
 * type, n_heads, n_groups and d_state. */
size_t bm_hip_delta_workspace_bytes(const bm_hip_delta_t *op);
int bm_hip_delta_dev(const bm_hip_delta_t *op, void *workspace, void *stream);
/* One token of each sequence; y may be written over v itself. */
int bm_hip_delta_step_dev(const bm_hip_delta_t *op, void *stream);

/* A pool of slots: slot i of layer l is slot_bytes bytes at base +
 * l * layer_stride + i * slot_stride (strides in bytes). */
typedef struct {
    void *base;
    int n_slots, n_layers;
    int64_t slot_bytes, slot_stride, layer_stride;
} bm_hip_slots_t;

/* Slot dst[i] takes over slot src[i] of every layer of every pool, for all
 * pairs at once (device lists): each pair reads what stood there before the
 * call, so lists may fork (one src, many dst), swap, rotate or reorder.
 * src[i] = -1 clears the slot to zero bytes.  Pairs with another src or a
 * dst outside the pool do nothing; of several pairs with one dst the first
 * such pair counts.  At most 1024 pairs and 8 pools (of equal n_slots). */
int bm_hip_slots_copy_dev(const bm_hip_slots_t *pools, int n_pools,
                          const int32_t *src, const int32_t *dst, int n, void *stream);

/* Moves the slots that a table of n entries (device) names to the front:
 * with `live` different slots named, those below `live` stay and the others
 * go, in ascending order, to the free slots below it.  new_slots (may be
 * slots itself) gets the table after the moves; entries outside the pool
 * (ended sequences) are copied as they are.  Freed slots keep their bytes.
 * n_live (device, nullable) gets `live`.  At most 65536 slots and 8 pools
 * (of equal n_slots).  workspace: bm_hip_slots_compact_workspace_bytes
 * bytes of device memory on 16 bytes with any contents. */
size_t bm_hip_slots_compact_workspace_bytes(int n_slots);
int bm_hip_slots_compact_dev(const bm_hip_slots_t *pools, int n_pools,
                             const int32_t *slots, int32_t *new_slots, int n,
                             int32_t *n_live, void *workspace, void *stream);

/* ------------------------------------------------------------------ */
/* Verification of drafted tokens (no counterpart in the reference;     */
/* asynchronous on `stream`, allocates nothing, may be captured).       */
/* Sequence b has rows row_start[b] .. row_start[b + 1] - 1 (device,    */
/* n_seqs + 1 ascending entries, clamped to 0..n_rows; NULL for one     */
/* sequence of n_rows rows): one per drafted token and a last one.      */
/* Row i's target distribution p_i is that of the token that tokens[i]  */
/* drafts, the last row's that of the token behind all drafts.  Drafts  */
/* are taken in order while u[i] * q_i(tokens[i]) < p_i(tokens[i]).     */
/* The token after those taken is drawn from max(p_i - q_i, 0) of the   */
/* first row refused (p_i where that is zero everywhere), or from the   */
/* last row's p, with the last row's u: the first token at which the    */
/* running sum exceeds u times the whole.  So with u uniform in 0..1    */
/* (1 excluded) and drafts drawn from q, tokens are distributed as if   */
/* drawn from p one by one.                                             */
/*                                                                      */
/* - A row is logits, p = softmax(row / temp), or with target_weights   */
/*   (draft_weights) numbers p is proportional to, whose negative,      */
/*   infinite and NaN ones count as 0.  With temp below 0.05 (as the    */
/*   sampler's greedy branch) a row of logits is 1 at its largest, the  */
/*   first of equal ones.  -inf and NaN logits have p = 0, +inf ones    */
/*   share everything equally.                                          */
/* - draft NULL: the drafts were not drawn, q is 1 at tokens[i].        */
/* - A draft outside the vocabulary is refused (p = 0 and q = 0).       */
/*   A target row without any p > 0 refuses, and has next_token -1 if   */
/*   it is the one drawn from.                                          */
/* - Sums and exponentials are in 64 bits; nothing depends on an order. */
/* - Outputs and workspace must not overlap the inputs or each other.   */
/* - A sequence without rows gets n_accepted 0 and next_token -1.       */
/* - 0, -2 for arguments that do not fit (nothing is launched), -1 for  */
/*   a HIP error; the reason is in bm_hip_last_error().                 */
/* ------------------------------------------------------------------ */
typedef struct {
    int type;                   /* of target and draft */
    int vocab;                  /* 1..256000 */
    int n_seqs, n_rows;         /* up to 2^20, below 2^30 */
    const int32_t *row_start;   /* device [n_seqs + 1], or NULL */
    const void *target;         /* rows of vocab values */
    int64_t target_stride;      /* in elements, below 2^24 */
    int target_weights;
    const void *draft;          /* rows of vocab values (a sequence's last is not read), or NULL */
    int64_t draft_stride;
    int draft_weights;
    float temp;                 /* finite, read for rows of logits */
    const int32_t *tokens;      /* device [n_rows] (a sequence's last is not read) */
    const float *u;             /* device [n_rows] */
    int32_t *n_accepted;        /* device [n_seqs]: drafts taken */
    int32_t *next_token;        /* device [n_seqs] */
    float *ratio;               /* device [n_rows], or NULL: min(1, p / q) of each draft; last rows keep what they hold */
    int32_t *split_start;       /* device [2 * n_seqs + 1], or NULL: see below */
} bm_hip_verify_t;

/* split_start holds the rows of 2 n_seqs sequences: 2b is sequence b's rows
 * whose tokens stand (its first and one per draft taken), 2b + 1 its others.
 * Given as seq_start, with slots -1 for the odd ones, to bm_hip_conv_dev,
 * bm_hip_ssm_dev or bm_hip_delta_dev it advances each state by the tokens
 * that stand and no more, without a round trip to the host.
 * workspace: bm_hip_verify_workspace_bytes(op) bytes of device memory on 256
 * bytes with any contents; one of an op serves every call of no more
 * sequences, rows and vocabulary. */
size_t bm_hip_verify_workspace_bytes(const bm_hip_verify_t *op);
int bm_hip_verify_dev(const bm_hip_verify_t *op, void *workspace, void *stream);

/* ------------------------------------------------------------------ */
/* Device-resident model: the reference's model API (src/bitmamba.h:    */
/* 282-294, src/model.c:477-1314) with weights, activations and the    */
/* recurrent state in HBM.  Greedy or sampled next tokens              */
/* (src/model.c:132-361) with the repetition penalty.                  */
/* ------------------------------------------------------------------ */
typedef struct bm_hip_model bm_hip_model_t;

/* model_load (src/model.c:477-932) from a BIT2 image in memory: same
 * validation; weights copied to one device arena (packed tensors with code
 * 11 rewritten to 10), A = -expf(A_log) and the conv transpose computed at
 * load.  NULL on failure (reason in bm_hip_last_error()). */
bm_hip_model_t *bm_hip_model_load(const void *image, size_t size);
/* model_free (src/model.c:1316-1372) */
void bm_hip_model_free(bm_hip_model_t *m);
/* 0 vocab, 1 d_model, 2 n_layers, 3 n_heads, 4 d_inner */
int bm_hip_model_config(const bm_hip_model_t *m, int which);
/* zero recurrent state and ring position (block_init_cache,
 * src/block.c:11-26) */
int bm_hip_model_reset(bm_hip_model_t *m);
/* model_prefill (src/model.c:1045-1153): n tokens through every layer,
 * batched BitLinear + token-serial SSM; no LM head.  0 or -1. */
int bm_hip_model_prefill(bm_hip_model_t *m, const int32_t *tokens, int n);
/* model_forward_step (src/model.c:1175-1314) with the sampler set by
 * bm_hip_model_set_sampler: returns the next token; history[history_len]
 * as the reference's caller keeps it (the last 256 tokens are used);
 * -1 for a negative length. */
int bm_hip_model_step(bm_hip_model_t *m,
                      int token,
                      const int *history,
                      int history_len,
                      float penalty);
/* Fast mode (on != 0; off by default): every later prefill, step,
 * generate and decode sums the squares of each RMSNorm of d_model 1024,
 * 2048 or 4096 (and d_inner of the same) as a pairwise tree, as
 * bm_hip_quantize_fast_dev does, instead of the reference's sequential
 * chains.  Results then differ from the reference in the last bits of
 * 1/rms and occasionally by one int8 step.  0. */
int bm_hip_model_set_fast(bm_hip_model_t *m, int on);
/* Measurement (no counterpart in the reference; for benchmarks and
 * profiles): one kernel of the decode step, launched reps times back to
 * back on the model's stream after two untimed launches, timed with events
 * on that stream.  which: 0 = in_proj + SSM step of `layer`, 1 = out_proj
 * (+ residual) of `layer`, 2 = the LM head (greedy candidates); layer -1
 * takes the layers in turn (0, 1, .., n_layers - 1, 0, ..), so that each
 * launch reads weights that the previous launches did not.  Writes the
 * average microseconds per launch to *avg_us.  The recurrent state and the
 * activations change: reset the model (or load a saved state) afterwards.
 * 0, or -1 (bm_hip_last_error) for bad arguments or widths that take the
 * generic kernels. */
int bm_hip_model_time_kernel(bm_hip_model_t *m, int which, int layer, int reps, float *avg_us);
/* Sampling parameters of every later step, generate and decode: the
 * temp, min_p, top_p, top_k arguments of model_forward_step
 * (src/model.c:1175-1183), sampled on the device by sample_advanced
 * (src/model.c:132-361).  temp < 0.05 is greedy (the default). */
int bm_hip_model_set_sampler(bm_hip_model_t *m,
                             float temp,
                             float min_p,
                             float top_p,
                             int top_k);
/* sample_advanced (src/model.c:132-361) on its own: one token from
 * logits[vocab] (device memory, 16-byte aligned; scaled in place by 1/temp
 * as the reference leaves them), advancing the XorShift64* state *rng
 * (device memory, src/utils.c:117-140); temp < 0.05 is the greedy branch.
 * workspace: bm_hip_sample_workspace_bytes(vocab) bytes of device memory, on
 * any alignment and with any contents (the reference's probs buffer, candidate
 * lists and partial sums: no multiple of the vocabulary, ask the function).
 * The token goes to token_out[0]
 * (device memory); enqueued on `stream`, no synchronization.  0, or -1 for
 * vocab outside 1..256000, misaligned logits or a null pointer. */
size_t bm_hip_sample_workspace_bytes(int vocab);
int bm_hip_sample_advanced(float *logits,
                           int vocab,
                           float temp,
                           float min_p,
                           float top_p,
                           int top_k,
                           uint64_t *rng,
                           void *workspace,
                           int32_t *token_out,
                           void *stream);
/* rng_seed (src/utils.c:121-124) for the model's device generator; the
 * model starts with the reference's default state. */
int bm_hip_model_seed(bm_hip_model_t *m, uint64_t seed);
/* Recurrent state as a BMST image (state_save / state_load,
 * src/chat.c:1160-1271): u32 magic 0x424D5354, n_layers, d_inner, d_conv,
 * then per layer conv_state[(d_conv-1)*d_inner], ssm_state[d_inner] (fp32)
 * and conv_pos (int).  File I/O stays with the caller.  save returns the
 * bytes written (bm_hip_model_state_bytes) or -1; load returns 0, or -1
 * leaving the state untouched on a bad magic or dimensions and reset to
 * zero on a truncated image or a bad ring position, as the reference does.
 * Layers at different ring positions are rejected (the device model keeps
 * one position; the reference's layers always share it). */
size_t bm_hip_model_state_bytes(const bm_hip_model_t *m);
int bm_hip_model_state_save(const bm_hip_model_t *m, void *out, size_t len);
int bm_hip_model_state_load(bm_hip_model_t *m, const void *in, size_t len);
/* copies the logits of the last step (after the penalty; divided by the
 * temperature when the step sampled, like the reference's) */
int bm_hip_model_logits(const bm_hip_model_t *m, float *out);
/* copies one layer's conv_state [3][d_inner] and ssm_state [d_inner];
 * returns the ring position */
int bm_hip_model_layer_state(const bm_hip_model_t *m,
                             int layer,
                             float *conv_state,
                             float *ssm_state);
/* The inverse: one layer's conv ring [3][d_inner], ssm state [d_inner] and
 * ring position (the block cache fields of src/bitmamba.h:84-87) into the
 * device model.  The device keeps one ring position for all layers, as the
 * reference's layers advance together.  With bm_hip_model_layer_state this
 * is the prefill hook for model_prefill (the Metal spot, src/model.c:
 * 1050-1055): push the blocks' state, bm_hip_model_prefill, pull it back.
 * 0, or -1 with bm_hip_last_error(). */
int bm_hip_model_set_layer_state(bm_hip_model_t *m,
                                 int layer,
                                 const float *conv_state,
                                 const float *ssm_state,
                                 int conv_pos);
/* The decode loop of src/main.c:443-500 on the device: prefill
 * prompt[0..n-2], history = prompt, then n_steps steps (greedy or sampled,
 * bm_hip_model_set_sampler) from
 * prompt[n-1], each step one replay of a captured hipGraph with no host
 * synchronization.  Writes the tokens; *decode_ms = device time of the
 * steps (prefill excluded, as the reference's tok/s).  Returns the number of
 * tokens (cut after the first 50256 or 0 when stop_on_eos), -1 on error.
 * With stop_on_eos the step that picks the end token is the last that
 * changes anything, as in the reference's loop (src/main.c:473-500): the
 * recurrent state, ring position, history, logits and sampler state stay
 * where that step left them although the device replays the step graph
 * n_steps times (a done word in the control block turns the later steps'
 * stores off).  This holds for d_model and d_inner multiples of 64 up to
 * 8192 (the fused step kernels); other widths run all n_steps and only the
 * returned list is cut.  bm_hip_model_decode and bm_hip_model_step then
 * continue from the end token. */
int bm_hip_model_generate(bm_hip_model_t *m,
                          const int32_t *prompt,
                          int n_prompt,
                          int n_steps,
                          float penalty,
                          int stop_on_eos,
                          int32_t *out_tokens,
                          double *decode_ms);
/* n_steps more steps from the current device state (also after a
 * generate that stopped at an end token); tokens readable with
 * bm_hip_model_tokens. */
int bm_hip_model_decode(bm_hip_model_t *m,
                        int n_steps,
                        float penalty,
                        double *decode_ms);
int bm_hip_model_tokens(const bm_hip_model_t *m, int32_t *out, int n);

/* Diagnostic (no reference counterpart): evaluates the device scalar
 * functions of the SSM step on n device floats, for checks against the host:
 * fn 0 = expf, 1 = logf (restatements of glibc's), 2 = fp32 division of each
 * even/odd input pair in both orders (out[i] = in[i] / in[i ^ 1]; a last
 * unpaired input is divided by itself), 3 = silu, x / (1 + expf(-x)),
 * 4 = sqrt.  Returns -1 for any other fn. */
int bm_hip_libm_eval_dev(int fn,
                         const float *in,
                         float *out,
                         size_t n,
                         void *stream);

/* ------------------------------------------------------------------ */
/* Synthetic BIT2 images (counterpart: the writer scripts/export-bin.py  */
/* :99-199; no libm, bit-reproducible on any host)                      */
/* ------------------------------------------------------------------ */
enum {
    BM_SYNTH_UNIFORM = 0,   /* p(-1)=p(0)=p(+1)=1/3 */
    BM_SYNTH_P0_40 = 1,     /* p(0)=0.4, p(+-1)=0.3 */
    BM_SYNTH_P0_60 = 2,     /* p(0)=0.6, p(+-1)=0.2 */
    BM_SYNTH_RAW_BYTES = 3, /* all four 2-bit codes, 11 included */
};

typedef struct {
    int vocab;
    int d_model;
    int n_layers;
    int n_heads;
    int in_proj_rows; /* 0: 2*d_inner + 3*n_heads (src/model.c:683-701) */
    int ternary_dist; /* BM_SYNTH_* */
    float fp_sigma;   /* std of every float tensor */
    float ternary_scale;
    uint64_t seed;
} bm_synth_config_t;

size_t bm_bit2_synth_size(const bm_synth_config_t *c);
int bm_bit2_synth_write(const bm_synth_config_t *c, void *dst, size_t len);
void bm_synth_ternary(uint64_t seed,
                      int tensor,
                      int rows,
                      int cols,
                      int dist,
                      uint8_t *packed);
void bm_synth_normal(uint64_t seed,
                     int tensor,
                     size_t n,
                     float sigma,
                     float *out);
void bm_synth_int8(uint64_t seed, int tensor, size_t n, int8_t *out);
void bm_synth_prompt(uint64_t seed, int vocab, int n, int32_t *tokens);

#ifdef __cplusplus
}
#endif
