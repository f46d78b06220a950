/*
 * dion_lm.h -- C ABI of the training operators around the Dion optimizer (libdion_lm.so, gfx950).
 *
 * The optimizer consumes gradients; these operators make those of the parameters that its
 * elementwise branch updates: the output layer (linear cross entropy) and the norms (residual
 * RMS norm), and the dropout between them.
 *
 * Conventions (those of dion_codec.h, whose DION_OK / DION_E_* / DION_DTYPE_* codes are used):
 *  - every function returns DION_OK (0) or a negative DION_E_* code; the text of the last
 *    failure on the calling thread is dion_lm_last_error(); a refused call enqueues nothing;
 *  - no allocation and no host synchronisation inside; everything is enqueued on `stream`, by
 *    kernels only (a call can be captured into a graph), on the current device;
 *  - stateless and re-entrant; the caller owns every buffer.  A workspace is used by one call at
 *    a time: calls (or captured graphs) that may run together need one each;
 *  - row-major tensors, unit stride along the last axis, row strides (`ld_*`) in elements;
 *  - sums, softmax statistics and norms are held in fp32; results are rounded once, to nearest
 *    even, when they are stored; all results are bitwise reproducible (no atomics on floats).
 */
#ifndef DION_LM_H_
#define DION_LM_H_

#include "dion_codec.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DION_LM_ABI_VERSION 1

#define DION_DTYPE_E4M3 3 /* 8-bit float, OCP e4m3fn (largest value 448) */

/* ABI version of the loaded library (== DION_LM_ABI_VERSION). */
int dion_lm_abi_version(void);
/* First 16 hex digits of the SHA-256 of the sources the library was compiled from. */
const char* dion_lm_build_id(void);
/* Text of the last error raised on this thread ("" if none). */
const char* dion_lm_last_error(void);

/* ------------------------------------------------------------------ random numbers
 * Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3",
 * SC 2011): key = seed (low word first), counter = (e / 4, offset) as two 64-bit numbers (low
 * words first), and element e = row * cols + col of the tensor takes word e % 4.  The element is
 * kept iff its word is >= floor(p 2^32 + 1/2); a kept x becomes x * fp32(1 / (1 - p)), a dropped
 * one 0 whatever it held.  The mask depends on (seed, offset, e) alone: the backward pass, another
 * stride or another device makes it again.
 */
typedef struct DionRng {
  uint64_t seed;
  uint64_t offset;        /* one number for each use of a seed (layer, step, rank) */
  const uint64_t* device; /* not NULL: {seed, offset} are read from this device memory when the
                             kernel runs (a captured graph then draws a new mask at each replay) */
} DionRng;

/*
 * out = residual + D(x)  (residual == NULL: out = D(x)), all rows x cols of `dtype` (F32 or BF16).
 * The product and the sum are rounded to fp32 each, then to `dtype`.  The backward pass of x is
 * the same call on the gradient without a residual.  `out` may be x or residual (same strides).
 * 0 <= p <= 1.
 */
int dion_dropout_add(int64_t rows, int64_t cols, int32_t dtype, const void* x, int64_t ld_x,
                     const void* residual, int64_t ld_residual, void* out, int64_t ld_out, double p,
                     const DionRng* rng, dion_stream_t stream);

/* ------------------------------------------------------------------ residual RMS norm */
typedef struct DionNormDesc {
  int64_t rows;
  int32_t cols;        /* 1 .. 16384 */
  int32_t dtype;       /* x, residual, h, y, their gradients: F32 or BF16                     */
  int32_t w_dtype;     /* weight: F32 or BF16                                                 */
  int32_t gw_dtype;    /* grad_weight: F32 or BF16                                            */
  int32_t y_dtype;     /* `dtype`, or E4M3 (8 bits with scales)                               */
  int32_t scale_block; /* E4M3: columns that share a scale, min(8, cols) .. cols (cols: one a row) */
  int32_t accumulate;  /* backward: grad_weight += instead of =                               */
  float eps;
  double p;            /* dropout of x, 0 <= p <= 1                                           */
  int64_t ld_x, ld_residual, ld_h, ld_y;       /* forward                                     */
  int64_t ld_grad_y, ld_grad_h, ld_grad_x, ld_grad_residual; /* backward (and ld_h)           */
} DionNormDesc;

/*
 * h = round(residual + D(x));  rstd = (mean_c h^2 + eps)^(-1/2);  y = h rstd w
 * `residual` may be NULL.  `h` may be NULL iff residual is NULL and p == 0 (h is x).  The norm is
 * of h as it is stored.  y_dtype E4M3: y holds round_e4m3(y / s) and scale (rows x
 * ceil(cols / scale_block) fp32) holds s = max(max_block |y| / 448, 2^-126).
 */
int dion_rms_norm_add(const DionNormDesc* desc, const void* x, const void* residual, const void* weight,
                      void* h, void* y, float* scale, float* rstd, const DionRng* rng, dion_stream_t stream);

/* Scratch of dion_rms_norm_add_backward (its partial weight gradients). */
int dion_rms_norm_add_workspace_bytes(const DionNormDesc* desc, size_t* bytes);

/*
 * d = rstd (w gy - h rstd mean_c(w gy h rstd)) + grad_h   (grad_h: the gradient that reaches h past
 *     the norm; NULL: none)
 * grad_residual = d (NULL: not wanted); grad_x = D(d) with the forward's mask (NULL: not wanted);
 * grad_weight = sum_rows gy h rstd (NULL: not wanted).  desc->y_dtype is not read: through an
 * 8-bit y the gradient is passed as if y had not been rounded.
 */
int dion_rms_norm_add_backward(const DionNormDesc* desc, const void* grad_y, const void* h, const void* weight,
                               const float* rstd, const void* grad_h, void* grad_x, void* grad_residual,
                               void* grad_weight, const DionRng* rng, void* ws, size_t ws_bytes,
                               dion_stream_t stream);

/* ------------------------------------------------------------------ linear cross entropy */
typedef struct DionXentDesc {
  int64_t tokens;
  int32_t hidden;
  int32_t vocab;       /* rows of `weight` that take part (this rank's shard)                  */
  int32_t dtype;       /* hidden states, weight and grad_hidden: BF16 or F32                   */
  int32_t gw_dtype;    /* grad_weight: BF16 or F32                                             */
  int32_t accumulate;  /* backward: grad_weight += instead of =                                */
  int32_t pack_weight; /* 1: weight is not 16-byte aligned and is read through the workspace   */
  int64_t vocab_start; /* the word that weight's first row stands for                          */
  int64_t vocab_total; /* words over all shards: targets are below it                          */
  int64_t ignore_index;
  int64_t ld_hidden, ld_weight, ld_grad_hidden, ld_grad_weight;
  int64_t piece_bytes; /* backward: most scratch for the gradient of a piece's logits, 0: 1 GiB
                          (a piece is 256 words at least)                                      */
} DionXentDesc;

#define DION_XENT_FORWARD 1
#define DION_XENT_BACKWARD 2

/* Scratch of one call (`op`: DION_XENT_FORWARD or DION_XENT_BACKWARD). */
int dion_xent_workspace_bytes(const DionXentDesc* desc, int op, size_t* bytes);

/*
 * z_tv = sum_k hidden_tk weight_vk over this shard's words;  lse_t = log sum_v exp(z_tv);
 * tlogit_t = z_t,target_t if the target is this shard's, else 0;  loss_t = lse_t - tlogit_t
 * (loss == NULL: not wanted; right only where one shard holds the vocabulary).
 * A token whose target is ignore_index has lse = tlogit = loss = 0 and its hidden state is not
 * read; any other target outside 0 .. vocab_total - 1 gives loss = tlogit = NaN.  The logits are
 * never stored.
 */
int dion_xent_forward(const DionXentDesc* desc, const void* hidden, const void* weight, const int64_t* target,
                      float* loss, float* lse, float* tlogit, void* ws, size_t ws_bytes, dion_stream_t stream);

/*
 * g_tv = (exp(z_tv - lse_t) - [v is t's target]) grad_loss_t;
 * grad_hidden_tk = sum_v g_tv weight_vk (this shard's share; NULL: not wanted);
 * grad_weight_vk = sum_t g_tv hidden_tk (NULL: not wanted).
 * `lse` is that of the whole vocabulary.  A token that is ignored, or whose grad_loss is 0, gets a
 * zero grad_hidden and adds nothing to grad_weight, whatever its hidden state holds.  g is computed
 * a piece of the vocabulary at a time, in the workspace.  tokens == 0 is refused: there is no
 * gradient to add, and the caller knows it.
 * Roundings before the products: g to bf16 (2^-8) for bf16 results, for grad_weight of up to 256 tokens
 * to two (2^-16); where the inputs or grad_weight are fp32, g to 2^-22 of itself or 2^-49 of grad_loss_t,
 * whichever is more, and hidden_t grad_loss_t for grad_weight to 2^-39 (bf16 inputs) or 2^-50 (fp32) of the
 * largest of them; fp32 hidden and weight, here and in dion_xent_forward, to 2^-22 of the value or 2^-50 of
 * the largest.
 */
int dion_xent_backward(const DionXentDesc* desc, const void* hidden, const void* weight, const int64_t* target,
                       const float* lse, const float* grad_loss, void* grad_hidden, void* grad_weight, void* ws,
                       size_t ws_bytes, dion_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* DION_LM_H_ */
