/*
 * zluda_ffn.h -- what stands beside the matmuls in the feed-forward half of a transformer block: a gated feed-forward layer,
 * the layer norm in front of it, and activation checkpoints in 8 bits, which the forward passes of both write and the
 * backward passes read.  The down projection is an ordinary cublasLtMatmul.  The reference has no counterpart.
 * For layers in 8 bits and for layers of experts: RMS norm with the residual's addition, packing of activations and weights with a scale for
 * each 128 (the operands of a cublasLtMatmul with such scales), and products grouped by expert.
 *
 * Conventions of the library: plain pointers to device memory, sizes and enum numbers in, a cublasStatus_t out; work is
 * enqueued on `stream` (a hipStream_t) and nothing is allocated, synchronised or kept; all calls may be captured into a
 * graph.  CUBLAS_STATUS_INVALID_VALUE (7): a pointer that is missing, misaligned for its element type, or sizes and pitches
 * that contradict each other; CUBLAS_STATUS_NOT_SUPPORTED (15): types or sizes that no kernel takes;
 * CUBLAS_STATUS_ALLOC_FAILED (3): a workspace that is too small; CUBLAS_STATUS_NOT_INITIALIZED (1): no HIP device.  What is
 * refused launches nothing.
 *
 * Matrices are row-major: element (r, c) at data[r * ld + c], ld >= columns.  A row is a token.
 */
#ifndef ZLUDA_AMD_FFN_H
#define ZLUDA_AMD_FFN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif
/* the declarations below are the library's exported symbols (it is built with -fvisibility=hidden) */
#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* A row-major matrix; data == NULL: absent.
 *
 * type CUDA_R_16F, CUDA_R_16BF, CUDA_R_32F: plain elements, aligned to their size (16-byte aligned rows are the fast case).
 *
 * type CUDA_R_8F_E4M3: a checkpoint.  Each 32 neighbours of a row share a power of two 2^e, e the smallest integer with
 * |v| <= 448 * 2^e for every finite v of the 32, and at least -126; scales holds e + 127 (UE8M0) at
 * scales[r * ld_scales + c / 32].  data holds the OCP E4M3 code of v / 2^e, rounded to nearest, ties to even; what is not
 * finite is stored as NaN (of either sign) and does not count for e.  ld is a multiple of 32 and data is 16-byte aligned; a row's last block
 * is filled up with zeros, so that rows hold 32 * ceil(columns / 32) codes.  ld_scales >= ceil(columns / 32).
 *
 * Rounding to E4M3 can take a finite value near the top of its type to the power of two behind it, 65536 for 16F (from 63488 on), 2^128 for 16BF and
 * 32F: checkpoint_load rounds that to the type, which makes it an infinity; what the backward passes read of a checkpoint counts as the largest finite
 * number there (x of the gated layer of its type, the others of 32F), so that only what was not finite spoils a sum.
 *
 * type CUDA_R_8F_E4M3 where an operator below says "packed": data holds E4M3 codes, scales floats.  Each 128 neighbours of a row (of a weight:
 * each block of 128 rows and 128 columns) share a scale s, the largest finite magnitude of them divided by 448, and at least 2^-126; the
 * code is that of v / s, rounded to nearest, ties to even; what is not finite is stored as NaN and does not count for s.  The scale of
 * element (r, c) is at scales[c / 128 * ld_scales + r], ld_scales >= rows (blocks of 128 rows: at scales[r / 128 * ld_scales + c / 128],
 * ld_scales >= ceil(columns / 128)): with ld_scales the rows what CUBLASLT_MATMUL_MATRIX_SCALE_VEC128_32F takes, with
 * ceil(columns / 128) rounded up to four what BLK128x128_32F takes.  data may lie anywhere (rows on 16 bytes are the fast case); nothing behind a
 * row's last column is written.  Products multiply by the product of two scales, held in 32 bits: finite, and a
 * normal number wherever the result is to keep its precision (a block of zeros has the scale 2^-126: its products are zeros all the same). */
typedef struct zluda_ffn_matrix {
  void *data;
  void *scales;      /* checkpoints and what is packed */
  int64_t ld;        /* elements */
  int64_t ld_scales; /* bytes, of a checkpoint; floats, of what is packed */
  uint32_t type;     /* cudaDataType */
} zluda_ffn_matrix;

#define ZLUDA_FFN_SILU 0u /* g / (1 + exp(-g)) */
#define ZLUDA_FFN_GELU 1u /* the tanh form, as the library's GELU epilogues */
#define ZLUDA_FFN_RELU 2u

/* G = X Wg^T + bg, U = X Wu^T + bu, H = act(G) * U.
 * x: tokens x model, w: 2 * features x model, Wg's rows in front of Wu's, h: tokens x features, all of one 16-bit type;
 * bias: 2 * features elements of that type or NULL; up to 2^20 features.  gate and up (both or neither; data == NULL: not kept) receive G and U,
 * in the same type or as checkpoints.  Products and sums in 32 bits; H comes from the 32-bit G and U, not from what is kept. */
typedef struct zluda_ffn_gated {
  uint32_t activation;
  uint64_t tokens, features, model;
  zluda_ffn_matrix x, w, h, gate, up;
  const void *bias;
} zluda_ffn_gated;

uint32_t zluda_ffn_gated_forward(const zluda_ffn_gated *p, void *workspace, size_t workspace_size, void *stream);
uint32_t zluda_ffn_gated_forward_workspace(const zluda_ffn_gated *p, size_t *bytes);

/* The gradients, from dH and what was kept:
 *   dU = dH * act(G), dG = dH * U * act'(G)   (computed in 32 bits, rounded to the type for the products)
 *   dx = dG Wg + dU Wu, dw = [dG dU]^T X (2 * features x model), dbias = sums of [dG dU] over the tokens (2 * features)
 * gate, up and x are plain (dh's type) or checkpoints.  Outputs that are absent are not computed: dx, dw, dbias; h
 * (tokens x features) receives H again, from the kept G and U; dz (tokens x 2 * features) receives [dG dU], which otherwise
 * goes through the workspace.  w is needed for dx, x for dw.  No output may overlap an input or another output. */
typedef struct zluda_ffn_gated_grad {
  uint32_t activation;
  uint64_t tokens, features, model;
  zluda_ffn_matrix dh, gate, up, x, w;
  zluda_ffn_matrix dx, dw, h, dz;
  void *dbias;
} zluda_ffn_gated_grad;

uint32_t zluda_ffn_gated_backward(const zluda_ffn_gated_grad *p, void *workspace, size_t workspace_size, void *stream);
/* (of the structure's sizes, types, pitches and which matrices are present; pointers are only compared with NULL) */
uint32_t zluda_ffn_gated_backward_workspace(const zluda_ffn_gated_grad *p, size_t *bytes);

/* Layer norm over rows: y = (x - mean) * rstd * weight + bias, rstd = 1 / sqrt(variance + eps), the variance that of the row
 * (divided by cols).  x, y: rows x cols of one type (16F, 16BF, 32F), cols up to 16384; weight, bias: cols elements of
 * weight_type (x's or 32F), NULL: 1 and 0; mean, rstd: rows floats each or NULL; kept (data == NULL: not kept): a checkpoint of
 * x, written in the same pass.  y may be x itself, with its pitch. */
#define ZLUDA_FFN_NORM_MAX_COLS 16384u
typedef struct zluda_ffn_norm {
  uint64_t rows, cols;
  float eps;
  uint32_t weight_type;
  zluda_ffn_matrix x, y, kept;
  const void *weight, *bias;
  float *mean, *rstd;
} zluda_ffn_norm;

uint32_t zluda_ffn_norm_forward(const zluda_ffn_norm *p, void *stream);

/* The gradients, with xhat = (x - mean) * rstd and x plain (dy's type) or a checkpoint:
 *   dx = rstd * (dy * weight - mean_c(dy * weight) - xhat * mean_c(dy * weight * xhat)) + add
 *   dweight = sum over rows of dy * xhat, dbias = sum over rows of dy   (weight_type; the order of the sums is fixed)
 * dweight and dbias: both or neither; add may be absent, dx too.  dx may be add or dy itself, with its pitch. */
typedef struct zluda_ffn_norm_grad {
  uint64_t rows, cols;
  uint32_t weight_type;
  zluda_ffn_matrix x, dy, add, dx;
  const void *weight;
  const float *mean, *rstd;
  void *dweight, *dbias;
} zluda_ffn_norm_grad;

uint32_t zluda_ffn_norm_backward(const zluda_ffn_norm_grad *p, void *workspace, size_t workspace_size, void *stream);
uint32_t zluda_ffn_norm_backward_workspace(const zluda_ffn_norm_grad *p, size_t *bytes);

/* rows x cols between a plain matrix and a checkpoint. */
uint32_t zluda_ffn_checkpoint_store(uint64_t rows, uint64_t cols, const zluda_ffn_matrix *x, const zluda_ffn_matrix *checkpoint, void *stream);
uint32_t zluda_ffn_checkpoint_load(uint64_t rows, uint64_t cols, const zluda_ffn_matrix *checkpoint, const zluda_ffn_matrix *x, void *stream);

/* Root-mean-square norm over rows, behind the residual's addition:
 *   h = x + residual, rounded once to the type (residual absent: h = x);  rstd = 1 / sqrt(mean(h^2) + eps);  y = h * rstd * weight
 * The norm takes the rounded h, which is what the backward pass reads.  x, residual, sum (receives h), y: rows x cols of one type (16F, 16BF, 32F), cols up
 * to 16384; packed receives y packed, from its 32-bit values; sum, y and packed are absent or wanted (data == NULL), one of them at least wanted;
 * weight: cols elements of weight_type (x's or 32F), NULL: 1; rstd: rows floats or NULL.  sum or y may be x or residual itself, with its
 * pitch, but sum is not y.  Squares and their sum are held in 32 bits: a row whose sum of squares passes 2^128 has rstd 0. */
typedef struct zluda_ffn_rms {
  uint64_t rows, cols;
  float eps;
  uint32_t weight_type;
  zluda_ffn_matrix x, residual, sum, y, packed;
  const void *weight;
  float *rstd;
} zluda_ffn_rms;

uint32_t zluda_ffn_rms_forward(const zluda_ffn_rms *p, void *stream);

/* The gradients, with xhat = h * rstd:
 *   dx = rstd * (dy * weight - xhat * mean_c(dy * weight * xhat)) + add     (of x, and of residual)
 *   dweight = sum over rows of dy * xhat   (weight_type; the order of the sum is fixed)
 * add, dx and dweight may be absent, dx and dweight not both; dx may be add or dy itself, with its pitch. */
typedef struct zluda_ffn_rms_grad {
  uint64_t rows, cols;
  uint32_t weight_type;
  zluda_ffn_matrix h, dy, add, dx;
  const void *weight;
  const float *rstd;
  void *dweight;
} zluda_ffn_rms_grad;

uint32_t zluda_ffn_rms_backward(const zluda_ffn_rms_grad *p, void *workspace, size_t workspace_size, void *stream);
uint32_t zluda_ffn_rms_backward_workspace(const zluda_ffn_rms_grad *p, size_t *bytes);

/* h = act(gate) * up, or act(gate) where up is absent; ZLUDA_FFN_COPY: h = gate (up absent).  gate, up, y: rows x cols of one type (16F, 16BF, 32F);
 * y and packed receive h (either may be absent), the packed one from the 32-bit values, with scales for 128 of a row (block_rows 1) or for blocks of
 * 128 x 128 (block_rows 128).  gate and up may be the halves of one matrix.  y may be gate or up itself, with its pitch. */
#define ZLUDA_FFN_COPY 3u
typedef struct zluda_ffn_activation {
  uint32_t activation, block_rows;
  uint64_t rows, cols;
  zluda_ffn_matrix gate, up, y, packed;
} zluda_ffn_activation;

uint32_t zluda_ffn_activate(const zluda_ffn_activation *p, void *stream);

/* What is packed, as plain values: code times scale, rounded to y's type (a value beyond its largest is that one). */
uint32_t zluda_ffn_unpack(uint64_t rows, uint64_t cols, uint32_t block_rows, const zluda_ffn_matrix *packed, const zluda_ffn_matrix *y, void *stream);

/* Products grouped by expert.  Rows are sorted by expert: those of expert e are offsets[e] .. offsets[e + 1] - 1, offsets being experts + 1 numbers in device
 * memory that do not decrease, from 0 to rows; an expert may have none, and rows that no expert has stay as they are in y and dx.
 *   y[r] = W_e x[r]      x: rows x model, w: experts * features x model (expert e: rows e * features and on), y: rows x features
 * x, w and y of one 16-bit type; or x packed, w packed in blocks of 128 x 128 that start anew at each expert (scales of expert e from block row
 * e * ceil(features / 128) on), and y 16F, 16BF or 32F.  y is none of the operands.  Numbers in offsets that break the rule give wrong results, but nothing outside
 * the matrices is touched.
 * Sums in 32 bits.  Packed operands with a 16-bit y are multiplied by the 8-bit instruction, which drops of each eight neighbouring products what lies 2^13 below the
 * largest: 1.4e-5 of a result (2-norm), below its rounding.  For y of 32F they are multiplied by the 16-bit one, which does not, at half the rate.
 * model a multiple of eight (packed: of 16), x and w with their rows on 16 bytes: tiles on the matrix units.  Anything else, and pitches of 2^22 and more: a kernel on
 * the vector units, 13 to 29 times as long (1001 rows of eight, 1024 x 2816: 241 us for 15.5). */
#define ZLUDA_FFN_MAX_EXPERTS 4096u
typedef struct zluda_ffn_grouped {
  uint64_t rows, experts, features, model;
  const int32_t *offsets;
  zluda_ffn_matrix x, w, y;
} zluda_ffn_grouped;

uint32_t zluda_ffn_grouped_forward(const zluda_ffn_grouped *p, void *workspace, size_t workspace_size, void *stream);
uint32_t zluda_ffn_grouped_forward_workspace(const zluda_ffn_grouped *p, size_t *bytes);

/* The gradients, all matrices of one 16-bit type:
 *   dx[r] = W_e^T dy[r] (rows x model)      dw: dW_e = sum over the rows of e of dy[r]^T x[r] (experts * features x model), zeros for an expert without rows
 * dx or dw may be absent; w is needed for dx, x for dw.  Neither may be one of the operands.  Few rows share out dx's sums, which takes a workspace, 16-byte
 * aligned: it is asked for with the sizes, the pitches and which of dx and dw there will be (dx alone can take more than both), and does not depend on addresses.
 * Sums are taken in a fixed order: the same bits in every call.  model, features and all pitches multiples of eight, addresses of 16 bytes, and rows x the pitch of
 * dy and of x below 2 GiB (features x the pitch of w too): tiles on the matrix units.  Anything else: the vector units (eight experts, 1024 x 28672: 37000 rows 3.4 ms,
 * 40000, beyond 2 GiB, 135 ms). */
typedef struct zluda_ffn_grouped_grad {
  uint64_t rows, experts, features, model;
  const int32_t *offsets;
  zluda_ffn_matrix dy, x, w, dx, dw;
} zluda_ffn_grouped_grad;

uint32_t zluda_ffn_grouped_backward(const zluda_ffn_grouped_grad *p, void *workspace, size_t workspace_size, void *stream);
uint32_t zluda_ffn_grouped_backward_workspace(const zluda_ffn_grouped_grad *p, size_t *bytes);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif
#ifdef __cplusplus
}
#endif
#endif
