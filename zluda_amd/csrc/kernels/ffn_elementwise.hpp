// Element by element: storing and loading checkpoints, and the gradients of the gated activation (include/zluda_ffn.h).
// All memory bound.  A thread owns eight neighbouring columns (16 bytes of a 16-bit type, eight codes) and walks rows; 64
// threads side by side, four rows at a time in a workgroup.
#pragma once
#include "ffn_common.hpp"

namespace zluda_amd {

struct CheckpointParams {
  void *x;
  uint8_t *codes, *scales;
  int64_t rows, ldx, ld_codes, ld_scales;
  int32_t cols;
};

// One piece a thread (the loops are for more rows than a grid has) (8192 x 14336 bf16, us, store and load: 65.5 and 59.9; with 16 workgroups a CU that
// walk the rows 72.2 and 71.5, with two or four rows of a thread in flight no better)
template <class E>
__global__ __launch_bounds__(256) void checkpoint_store_kernel(CheckpointParams p) {
  const int col = 8 * (blockIdx.x * 64 + (threadIdx.x & 63)), cols32 = (p.cols + 31) & ~31;
  for (int64_t row = blockIdx.y * 4 + (threadIdx.x >> 6); row < p.rows; row += gridDim.y * 4) {  // (whole waves)
    const typename E::Raw8 r = load8<E>((const typename E::raw *)p.x + row * p.ldx + col, p.cols - col);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = E::get(r, e);
    ckpt_store8(p.codes + row * p.ld_codes, p.scales + row * p.ld_scales, col, cols32, v);
  }
}

// FINITE: for a product's operand; otherwise values are rounded to the type as they are
template <class E, bool FINITE>
__device__ __forceinline__ void checkpoint_load(const CheckpointParams &p, int strip) {
  const int col = 8 * (strip * 64 + (threadIdx.x & 63));
  if (col >= p.cols) return;
  for (int64_t row = blockIdx.y * 4 + (threadIdx.x >> 6); row < p.rows; row += gridDim.y * 4) {
    float v[8];
    const Ckpt8 c = ckpt_load8(p.codes + row * p.ld_codes, p.scales + row * p.ld_scales, col);
    if constexpr (FINITE) ckpt_get8_finite<E>(c, v);
    else ckpt_get8(c, v);
    store8<E>((typename E::raw *)p.x + row * p.ldx + col, v, p.cols - col);
  }
}

template <class E>
__global__ __launch_bounds__(256) void checkpoint_load_kernel(CheckpointParams p) {
  checkpoint_load<E, false>(p, blockIdx.x);
}

struct RoundParams {
  const float *x;
  void *y;
  int64_t rows, ldx, ldy, plane;
  int32_t cols, shares;
};

// Sums held in 32 bits to their type: the shares of x, `plane` elements apart, added in order (rows of x on 16 bytes and padded to whole pieces)
template <class E>
__device__ __forceinline__ void round_rows(const RoundParams &p, int64_t first, int64_t end) {
  const int col = 8 * (blockIdx.x * 64 + (threadIdx.x & 63));
  if (col >= p.cols) return;
  for (int64_t row = first + blockIdx.y * 4 + (threadIdx.x >> 6); row < end; row += gridDim.y * 4) {
    const float *x = p.x + row * p.ldx + col;
    float v[8] = {};
#pragma unroll 4
    for (int z = 0; z < p.shares; z++, x += p.plane) {
      const typename ElemF32::Raw8 r = load8<ElemF32>(x, 8);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += ElemF32::get(r, e);
    }
    store8<E>((typename E::raw *)p.y + row * p.ldy + col, v, p.cols - col);
  }
}
template <class E>
__global__ __launch_bounds__(256) void round_rows_kernel(RoundParams p) { round_rows<E>(p, 0, p.rows); }

struct GatedGradParams {
  const void *dh, *gate, *up;              // gate, up: elements or codes
  const uint8_t *gate_scales, *up_scales;  // of checkpoints
  void *dz, *h;                            // dz: [dG dU]; h or NULL
  float *part;                             // [gridDim.y][2 * features]: partial sums of dz over the rows, or NULL
  int64_t tokens, lddh, ldg, ldu, ldgs, ldus, lddz, ldh;
  int32_t features;
  uint32_t activation;
  CheckpointParams load;                   // a checkpoint to decode beside it: the workgroups behind the features' strips; x == NULL: none
};

// dU = dH act(G), dG = dH U act'(G); H = act(G) U on request.  CK: gate and up are checkpoints.
//
// [dG dU] are rounded once, to the type of the operands that they meet in the two products: the matrix cores take both factors in one 16-bit type, and a
// second part for the bits below would double the products' operations.  The rounding adds to dx and dw as much as their own last one does: against 64 bits
// 2.35e-3 instead of 1.66e-3 (bf16, 2-norm; 8192 tokens, 2048 x 8192) and 2.93e-4 instead of 2.07e-4 (f16; 1001, 1024 x 2816), which is what the 32-bit products of
// the same rounded factors have, too.  The sums of the bias gradient take the values in front of it.
template <class E, bool CK, int ACT>
__global__ __launch_bounds__(256) void gated_grad_kernel(GatedGradParams p) {
  using raw = typename E::raw;
  const int strips = (p.features + 511) / 512;
  if ((int)blockIdx.x >= strips) {
    checkpoint_load<E, true>(p.load, blockIdx.x - strips);
    return;
  }
  const int lane = threadIdx.x & 63, phase = threadIdx.x >> 6, col = 8 * (blockIdx.x * 64 + lane), n = p.features - col;
  float sg[8], su[8];
#pragma unroll
  for (int e = 0; e < 8; e++) sg[e] = su[e] = 0.0f;
  if (n > 0) {
    for (int64_t row = blockIdx.y * 4 + phase; row < p.tokens; row += gridDim.y * 4) {
      float g[8], u[8], dg[8], du[8];
      const typename E::Raw8 rd = load8<E>((const raw *)p.dh + row * p.lddh + col, n);
      if constexpr (CK) {
        const Ckpt8 cg = ckpt_load8((const uint8_t *)p.gate + row * p.ldg, p.gate_scales + row * p.ldgs, col);
        const Ckpt8 cu = ckpt_load8((const uint8_t *)p.up + row * p.ldu, p.up_scales + row * p.ldus, col);
        ckpt_get8(cg, g);
        ckpt_get8(cu, u);
        if (__builtin_expect(max(cg.scale, cu.scale) >= ElemF32::top_scale, 0)) {  // (one branch, behind all loads: 82 us for 4096 x 14336, 87 with two)
          ckpt_finite8<ElemF32>(g);
          ckpt_finite8<ElemF32>(u);
        }
      } else {
        const typename E::Raw8 rg = load8<E>((const raw *)p.gate + row * p.ldg + col, n), ru = load8<E>((const raw *)p.up + row * p.ldu + col, n);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          g[e] = E::get(rg, e);
          u[e] = E::get(ru, e);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; e++) {
        float a, da;
        ffn_act_grad<ACT>(g[e], a, da);
        const float d = E::get(rd, e);
        dg[e] = d * u[e] * da;
        du[e] = d * a;
        g[e] = a * u[e];
        sg[e] += dg[e];
        su[e] += du[e];
      }
      store8<E>((raw *)p.dz + row * p.lddz + col, dg, n);
      store8<E>((raw *)p.dz + row * p.lddz + p.features + col, du, n);
      if (p.h) store8<E>((raw *)p.h + row * p.ldh + col, g, n);
    }
  }
  if (!p.part) return;
  __shared__ float fold[4][2][8][64];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    fold[phase][0][e][lane] = sg[e];
    fold[phase][1][e][lane] = su[e];
  }
  __syncthreads();
  for (int o = threadIdx.x; o < 2 * 8 * 64; o += 256) {
    const int which = o >> 9, e = (o >> 6) & 7, l = o & 63, c = 8 * (blockIdx.x * 64 + l) + e;
    if (c < p.features)
      p.part[(int64_t)blockIdx.y * 2 * p.features + which * p.features + c] =
          (fold[0][which][e][l] + fold[1][which][e][l]) + (fold[2][which][e][l] + fold[3][which][e][l]);
  }
}

// zeros where a sum has no terms (no memset node: those have replayed wrongly in captured graphs)
struct ZeroParams {
  void *p;
  int64_t rows, row_bytes, pitch_bytes;  // multiples of 2
};
static __global__ __launch_bounds__(256) void zero_rows_kernel(ZeroParams z) {
  const int64_t words = z.row_bytes / 2;
  for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < z.rows * words; i += (int64_t)gridDim.x * 256)
    ((uint16_t *)((char *)z.p + i / words * z.pitch_bytes))[i % words] = 0;
}

} // namespace zluda_amd
