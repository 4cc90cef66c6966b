// Root-mean-square norm over the rows of a matrix, behind the residual's addition, and its gradients (include/zluda_ffn.h).
//
//   h = round(x + residual), rstd = 1 / sqrt(mean(h^2) + eps), y = h rstd w;   dx = rstd (v - xhat mean(v xhat)) + add, v = dy w, xhat = h rstd
//
// Memory bound: a group of T threads holds a whole row in registers (NV times eight elements a thread), so everything is read once and written
// once; the next row travels while the one before is summed up.  One sum over the row and no second pass: h^2 has no cancellation.  A
// workgroup has neighbouring rows, whose scales of a packed output share cache lines.  16384 x 8192, bf16, residual and packed output: 193 us, 5.0 TB/s, the rate of a
// copy (4.9); four rows of 4096: 3.0 us, a launch and a round trip.  Gradients of 777 x 1001, f16, with an addend: 6.4 us and 2.9 for the sums
// of dweight in a second kernel, in one order, where atomics would add them in any.
#pragma once
#include "ffn_norm.hpp"
#include "ffn_pack.hpp"

namespace zluda_amd {

struct RmsParams {
  const void *x, *residual;  // residual or NULL
  void *sum, *y;             // or NULL
  uint8_t *codes;            // or NULL
  float *scales;
  const void *weight;        // or NULL
  float *rstd;               // or NULL
  int64_t rows, ldx, ldr, lds, ldy, ldc, ld_scales;
  float eps;
  int32_t cols, per_group;   // per_group: rows of a workgroup
  uint32_t weight_type;
};

// (Eight waves a SIMD, so that the workgroups a launch counts on are there at once: f32 has registers for seven otherwise, 2000 x 4096 29.0 us, 27.7.  Groups of fewer lanes
// would spill for it, a workgroup more or less of theirs is not seen.)
template <class E, int T, int R, int NV>
__global__ __launch_bounds__(T *R, NV == 1 && T >= 256 ? 8 : 4) void rms_forward_kernel(RmsParams p) {
  using raw = typename E::raw;
  __shared__ float words[2][R][T / 64][2];
  const int lane = threadIdx.x % T, group = threadIdx.x / T;
  int slot = 0;
  struct Row { typename E::Raw8 x[NV], r[NV]; };
  const int64_t first = (int64_t)blockIdx.x * p.per_group, last = min(p.rows, first + p.per_group);
  auto fetch = [&](Row &q, int64_t row) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int col = 8 * (lane + T * i), n = row < last ? p.cols - col : 0;
      q.x[i] = load8<E>((const raw *)p.x + row * p.ldx + col, n);
      if (p.residual) q.r[i] = load8<E>((const raw *)p.residual + row * p.ldr + col, n);
    }
  };
  Row next;
  fetch(next, first + group);
  float w[NV][8];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int col = 8 * (lane + T * i);
    norm_vector8<E>(p.weight, p.weight_type, col, p.cols - col, 1.0f, w[i]);
  }
  const float inv_n = 1.0f / (float)p.cols;
  for (int64_t r0 = first; r0 < last; r0 += R) {
    const int64_t row = r0 + group;
    const bool live = row < last;  // (a dead group of the last round keeps the barriers company)
    float h[NV][8], s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        h[i][e] = E::get(next.x[i], e);
        // (rounded as the sum that is kept: the backward pass has no other)
        if (p.residual) h[i][e] = E::dec(E::enc(h[i][e] + E::get(next.r[i], e)));
        s[0] = __builtin_fmaf(h[i][e], h[i][e], s[0]);
      }
    fetch(next, row + R);
    group_sum<T, R>(s, words, slot, group);
    const float rstd = 1.0f / __builtin_sqrtf(s[0] * inv_n + p.eps);
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int col = 8 * (lane + T * i), n = p.cols - col;
        if (p.sum) store8<E>((raw *)p.sum + row * p.lds + col, h[i], n);
#pragma unroll
        for (int e = 0; e < 8; e++) h[i][e] = h[i][e] * rstd * w[i][e];
        if (p.y) store8<E>((raw *)p.y + row * p.ldy + col, h[i], n);
        if (p.codes) {
          // (elements past the row's end are zeros)
          const float scale = pack_scale(pack_max16(pack_mag8(h[i])));
          pack_put8(p.codes + row * p.ldc + col, pack_encode8(h[i], scale), n);
          if ((lane & 15) == 0 && n > 0) p.scales[(int64_t)(col >> 7) * p.ld_scales + row] = scale;
        }
      }
      if (lane == 0 && p.rstd) p.rstd[row] = rstd;
    }
  }
}

struct RmsGradParams {
  const void *h, *dy, *add;  // add or NULL
  void *dx;                  // or NULL
  const void *weight;        // or NULL
  const float *rstd;
  float *part;               // [gridDim.x][cols]: partial sums of dweight; NULL: not wanted, or
  void *dweight;             // the sum itself, of a single workgroup
  int64_t rows, ldh, lddy, ldadd, lddx;
  int32_t cols;
  uint32_t weight_type;
};

// As norm_backward_kernel: the weight's sums stay in registers over the rows of a group and leave a workgroup once.
template <class E, int T, int R, int NV>
__global__ __launch_bounds__(T *R) void rms_backward_kernel(RmsGradParams p) {
  using raw = typename E::raw;
  __shared__ float words[2][R][T / 64][2];
  __shared__ float fold[R > 1 ? R : 1][R > 1 ? T * 8 : 1];
  const int lane = threadIdx.x % T, group = threadIdx.x / T;
  int slot = 0;
  constexpr bool AHEAD = NV == 1;
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int col = 8 * (lane + T * i);
    if constexpr (AHEAD) norm_vector8<E>(p.weight, p.weight_type, col, p.cols - col, 1.0f, w[i]);
#pragma unroll
    for (int e = 0; e < 8; e++) dw[i][e] = 0.0f;
  }
  const float inv_n = 1.0f / (float)p.cols;
  struct Row { typename E::Raw8 h[NV], dy[NV], add[NV]; float rstd; };
  auto fetch = [&](Row &q, int64_t row) __attribute__((always_inline)) {
    const bool live = row < p.rows;
    q.rstd = live ? p.rstd[row] : 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int col = 8 * (lane + T * i), n = live ? p.cols - col : 0;
      q.dy[i] = load8<E>((const raw *)p.dy + row * p.lddy + col, n);
      q.h[i] = load8<E>((const raw *)p.h + row * p.ldh + col, n);
      if (AHEAD && p.add) q.add[i] = load8<E>((const raw *)p.add + row * p.ldadd + col, p.dx ? n : 0);
    }
  };
  const int64_t step = (int64_t)gridDim.x * R;
  Row next;
  if constexpr (AHEAD) fetch(next, (int64_t)blockIdx.x * R + group);
  for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < p.rows; r0 += step) {
    const int64_t row = r0 + group;
    Row q;
    if constexpr (AHEAD) {
      q = next;
      fetch(next, row + step);
    } else {
      fetch(q, row);
    }
    float x[NV][8], d[NV][8], s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
      if constexpr (!AHEAD) norm_vector8<E>(p.weight, p.weight_type, 8 * (lane + T * i), p.cols - 8 * (lane + T * i), 1.0f, w[i]);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        x[i][e] = E::get(q.h[i], e) * q.rstd;
        d[i][e] = E::get(q.dy[i], e);
        dw[i][e] = __builtin_fmaf(d[i][e], x[i][e], dw[i][e]);
        d[i][e] *= w[i][e];
        s[0] = __builtin_fmaf(d[i][e], x[i][e], s[0]);
      }
    }
    if (!p.dx) continue;  // (uniform)
    group_sum<T, R>(s, words, slot, group);
    const float m = s[0] * inv_n;
    if (row < p.rows) {
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int col = 8 * (lane + T * i);
#pragma unroll
        for (int e = 0; e < 8; e++) d[i][e] = q.rstd * (d[i][e] - x[i][e] * m);
        if (p.add) {
          if constexpr (!AHEAD) q.add[i] = load8<E>((const raw *)p.add + row * p.ldadd + col, p.cols - col);
#pragma unroll
          for (int e = 0; e < 8; e++) d[i][e] += E::get(q.add[i], e);
        }
        store8<E>((raw *)p.dx + row * p.lddx + col, d[i], p.cols - col);
      }
    }
  }
  if (!p.part && !p.dweight) return;
  float *part = p.part + (int64_t)blockIdx.x * p.cols;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int col = 8 * (lane + T * i);
    if constexpr (R == 1) {
      const int n = p.cols - col;
      if (p.part) store8<ElemF32>(part + col, dw[i], n);
      else if (p.weight_type == CUDA_R_32F) store8<ElemF32>((float *)p.dweight + col, dw[i], n);
      else store8<E>((raw *)p.dweight + col, dw[i], n);
    } else {
      // the groups' sums meet in LDS, group after group
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; e++) fold[group][e * T + lane] = dw[i][e];  // (lane-contiguous: no bank conflicts)
      __syncthreads();
      for (int o = threadIdx.x; o < T * 8; o += T * R) {
        float t = 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) t += fold[r][o];
        const int c = 8 * (o % T + T * i) + o / T;
        if (c >= p.cols) continue;
        if (p.part) part[c] = t;
        else store_elem(p.dweight, p.weight_type, c, t);
      }
    }
  }
}

} // namespace zluda_amd
