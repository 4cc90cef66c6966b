/*
 * zluda_ffn.h -- what stands beside the matmuls in the feed-forward half of a transformer block: a gated feed-forward layer,
 * the layer norm in front of it, and activation checkpoints in 8 bits, which the forward passes of both write and the
 * backward passes read.  The down projection is an ordinary cublasLtMatmul.  The reference has no counterpart.
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
 * number there (x of the gated layer of its type, the others of 32F), so that only what was not finite spoils a sum. */
typedef struct zluda_ffn_matrix {
  void *data;
  void *scales;      /* checkpoints only */
  int64_t ld;        /* elements */
  int64_t ld_scales; /* bytes; checkpoints only */
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

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif
#ifdef __cplusplus
}
#endif
#endif
