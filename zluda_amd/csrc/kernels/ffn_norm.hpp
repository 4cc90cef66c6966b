// Layer norm over the rows of a matrix and its gradients (include/zluda_ffn.h).
//
// Memory bound: a group of T threads holds a whole row in registers (NV times eight elements a thread), so x -- and dy for the
// gradients -- are read once and y or dx written once.  The variance is summed from the differences to the mean, which takes
// a second reduction but no second read.  The groups walk rows gridDim.x * R apart; weights (and the gradients' sums over
// rows) stay in a thread's registers, because its columns are the same in every row.  The sums of dweight and dbias leave a
// workgroup once, as one partial row each, and norm_finish_kernel adds the partial rows up in their order: no atomics, the
// same bits in every call.
#pragma once
#include "ffn_common.hpp"

namespace zluda_amd {

struct NormParams {
  const void *x;
  void *y;
  uint8_t *codes, *scales;   // the checkpoint of x, or NULL
  const void *weight, *bias; // or NULL
  float *mean, *rstd;        // or NULL
  int64_t rows, ldx, ldy, ld_codes, ld_scales;
  float eps;
  int32_t cols;
  uint32_t weight_type;
};

struct NormGradParams {
  const void *x, *dy, *add;  // x: elements or codes; add or NULL
  const uint8_t *scales;     // of a checkpoint
  void *dx;                  // or NULL
  const void *weight;        // or NULL
  const float *mean, *rstd;
  float *part;               // [2][gridDim.x][cols]: partial sums of dweight, of dbias; NULL: not wanted, or
  void *dweight, *dbias;     // the sums themselves, of a single workgroup; NULL: not wanted, or by way of `part`
  int64_t rows, ldx, ld_scales, lddy, ldadd, lddx;
  int32_t cols;
  uint32_t weight_type;
};

// eight entries of a vector of `type` (the matrix's own or 32F), `miss` where there is no vector
template <class E>
__device__ __forceinline__ void norm_vector8(const void *vec, uint32_t type, int col, int n, float miss, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = miss;
  if (!vec || n <= 0) return;
  if (type == CUDA_R_32F) {
    const ElemF32::Raw8 r = load8<ElemF32>((const float *)vec + col, n);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = ElemF32::get(r, e);
  } else {
    const typename E::Raw8 r = load8<E>((const typename E::raw *)vec + col, n);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = E::get(r, e);
  }
}

// The sums of N values over a group of T threads (whole waves).  `slot` alternates between calls: with two sets of words one
// barrier a call keeps a fast wave's next sums off the words that a slow one still reads.
template <int T, int R, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float (*words)[R][T / 64][2], int &slot, int group) {
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = wave_sum(v[i]);
  if constexpr (T > 64) {
    const int wave = (threadIdx.x % T) / 64;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; i++) words[slot][group][wave][i] = v[i];
    }
    // (not __syncthreads: the next row's loads stay in flight)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < T / 64; w++) s += words[slot][group][w][i];
      v[i] = s;
    }
    slot ^= 1;
  }
}

template <class E, int T, int R, int NV>
__global__ __launch_bounds__(T *R) void norm_forward_kernel(NormParams p) {
  __shared__ float words[2][R][T / 64][2];
  const int lane = threadIdx.x % T, group = threadIdx.x / T;
  int slot = 0;
  // a row a round ahead: the first one travels beside the weights, the others while the row before is summed up
  struct Row { typename E::Raw8 x[NV]; };
  auto fetch = [&](Row &q, int64_t row) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int col = 8 * (lane + T * i);
      q.x[i] = load8<E>((const typename E::raw *)p.x + row * p.ldx + col, row < p.rows ? p.cols - col : 0);
    }
  };
  const int64_t step = (int64_t)gridDim.x * R;
  Row next;
  fetch(next, (int64_t)blockIdx.x * R + group);
  float w[NV][8], b[NV][8];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int col = 8 * (lane + T * i);
    norm_vector8<E>(p.weight, p.weight_type, col, p.cols - col, 1.0f, w[i]);
    norm_vector8<E>(p.bias, p.weight_type, col, p.cols - col, 0.0f, b[i]);
  }
  const float inv_n = 1.0f / (float)p.cols;
  const int cols32 = (p.cols + 31) & ~31;
  for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < p.rows; r0 += step) {
    const int64_t row = r0 + group;
    const bool live = row < p.rows;  // (a dead group of the last round keeps the barriers company)
    float v[NV][8], s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        v[i][e] = E::get(next.x[i], e);
        s[0] += v[i][e];
      }
    fetch(next, row + step);
    group_sum<T, R>(s, words, slot, group);
    const float mean = s[0] * inv_n;
    float q[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int n = p.cols - 8 * (lane + T * i);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float d = e < n ? v[i][e] - mean : 0.0f;
        q[0] = __builtin_fmaf(d, d, q[0]);
      }
    }
    group_sum<T, R>(q, words, slot, group);
    const float rstd = 1.0f / __builtin_sqrtf(q[0] * inv_n + p.eps);
    if (p.codes) {
#pragma unroll
      for (int i = 0; i < NV; i++)
        ckpt_store8(p.codes + row * p.ld_codes, p.scales + row * p.ld_scales, 8 * (lane + T * i), live ? cols32 : 0, v[i]);
    }
    if (!live) continue;  // (T == 64: nothing waits for this wave; else R == 1 and the group is live)
    typename E::raw *y = (typename E::raw *)p.y + row * p.ldy;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int col = 8 * (lane + T * i);
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = __builtin_fmaf((v[i][e] - mean) * rstd, w[i][e], b[i][e]);
      store8<E>(y + col, v[i], p.cols - col);
    }
    if (lane == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
  }
}

// CK: x is a checkpoint.  A row's elements are requested a round ahead, so that they travel while the row before is summed up (16384 x
// 4096 from a checkpoint, with an addend: 146 us without, 92 with; 471 MB).  With two pieces of eight a thread (NV 2: the
// widest rows) there are no registers for that, nor for the weights, which come from the caches again for each row.
template <class E, bool CK, int T, int R, int NV>
__global__ __launch_bounds__(T *R) void norm_backward_kernel(NormGradParams p) {
  __shared__ float words[2][R][T / 64][2];
  __shared__ float fold[R > 1 ? R : 1][R > 1 ? T * 8 : 1];
  const int lane = threadIdx.x % T, group = threadIdx.x / T;
  int slot = 0;
  constexpr bool AHEAD = NV == 1;
  float w[NV][8], dw[NV][8], db[NV][8];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int col = 8 * (lane + T * i);
    if constexpr (AHEAD) norm_vector8<E>(p.weight, p.weight_type, col, p.cols - col, 1.0f, w[i]);
#pragma unroll
    for (int e = 0; e < 8; e++) dw[i][e] = db[i][e] = 0.0f;
  }
  const float inv_n = 1.0f / (float)p.cols;
  const int cols32 = (p.cols + 31) & ~31;
  // a row as it lies in memory; of a row that does not exist: zeros
  struct Row {
    typename std::conditional<CK, Ckpt8, typename E::Raw8>::type x[NV];
    typename E::Raw8 dy[NV], add[NV];
    float mean, rstd;
  };
  auto fetch = [&](Row &q, int64_t row) __attribute__((always_inline)) {
    const bool live = row < p.rows;
    q.mean = live ? p.mean[row] : 0.0f;
    q.rstd = live ? p.rstd[row] : 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int col = 8 * (lane + T * i), n = live ? p.cols - col : 0;
      q.dy[i] = load8<E>((const typename E::raw *)p.dy + row * p.lddy + col, n);
      if constexpr (CK) {
        q.x[i] = Ckpt8{ffn_u2{0, 0}, 127};
        if (live && col < cols32) q.x[i] = ckpt_load8((const uint8_t *)p.x + row * p.ldx, p.scales + row * p.ld_scales, col);
      } else {
        q.x[i] = load8<E>((const typename E::raw *)p.x + row * p.ldx + col, n);
      }
      if (AHEAD && p.add) q.add[i] = load8<E>((const typename E::raw *)p.add + row * p.ldadd + col, p.dx ? n : 0);
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
    float x[NV][8], d[NV][8], s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
      if constexpr (CK) {
        ckpt_get8_finite<ElemF32>(q.x[i], x[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[i][e] = E::get(q.x[i], e);
      }
      if constexpr (!AHEAD) norm_vector8<E>(p.weight, p.weight_type, 8 * (lane + T * i), p.cols - 8 * (lane + T * i), 1.0f, w[i]);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        d[i][e] = E::get(q.dy[i], e);
        x[i][e] = (x[i][e] - q.mean) * q.rstd;
        dw[i][e] = __builtin_fmaf(d[i][e], x[i][e], dw[i][e]);
        db[i][e] += d[i][e];
        d[i][e] *= w[i][e];
        s[0] += d[i][e];
        s[1] = __builtin_fmaf(d[i][e], x[i][e], s[1]);
      }
    }
    if (!p.dx) continue;  // (uniform)
    group_sum<T, R>(s, words, slot, group);
    const float m1 = s[0] * inv_n, m2 = s[1] * inv_n;
    if (row < p.rows) {
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int col = 8 * (lane + T * i);
#pragma unroll
        for (int e = 0; e < 8; e++) d[i][e] = q.rstd * (d[i][e] - m1 - x[i][e] * m2);
        if (p.add) {
          if constexpr (!AHEAD) q.add[i] = load8<E>((const typename E::raw *)p.add + row * p.ldadd + col, p.cols - col);
#pragma unroll
          for (int e = 0; e < 8; e++) d[i][e] += E::get(q.add[i], e);
        }
        store8<E>((typename E::raw *)p.dx + row * p.lddx + col, d[i], p.cols - col);
      }
    }
  }
  if (!p.part && !p.dweight) return;
  float *part_w = p.part + (int64_t)blockIdx.x * p.cols, *part_b = p.part + ((int64_t)gridDim.x + blockIdx.x) * p.cols;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int col = 8 * (lane + T * i);
    if constexpr (R == 1) {
      const int n = p.cols - col;
      if (p.part) {
        store8<ElemF32>(part_w + col, dw[i], n);
        store8<ElemF32>(part_b + col, db[i], n);
      } else if (p.weight_type == CUDA_R_32F) {
        store8<ElemF32>((float *)p.dweight + col, dw[i], n);
        store8<ElemF32>((float *)p.dbias + col, db[i], n);
      } else {
        store8<E>((typename E::raw *)p.dweight + col, dw[i], n);
        store8<E>((typename E::raw *)p.dbias + col, db[i], n);
      }
    } else {
      // the groups' sums meet in LDS, group after group
#pragma unroll
      for (int which = 0; which < 2; which++) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; e++) fold[group][e * T + lane] = which ? db[i][e] : dw[i][e];  // (lane-contiguous: no bank conflicts)
        __syncthreads();
        for (int o = threadIdx.x; o < T * 8; o += T * R) {
          float t = 0.0f;
#pragma unroll
          for (int r = 0; r < R; r++) t += fold[r][o];
          const int c = 8 * (o % T + T * i) + o / T;
          if (c >= p.cols) continue;
          if (p.part) (which ? part_b : part_w)[c] = t;
          else store_elem(which ? p.dbias : p.dweight, p.weight_type, c, t);
        }
      }
    }
  }
}

// dweight (blockIdx.y 0) and dbias (1) from their `shares` partial rows: 16 columns a workgroup, 64 threads a column
struct NormFinishParams {
  const float *part;
  void *dweight, *dbias;
  int32_t shares, cols;
  uint32_t type;
};
template <int COLS, int PH>
__global__ __launch_bounds__(COLS *PH) void norm_finish_kernel(NormFinishParams p) {
  __shared__ float sums[PH][COLS];
  const int c = threadIdx.x % COLS, ph = threadIdx.x / COLS, col = blockIdx.x * COLS + c;
  const float *part = p.part + (int64_t)blockIdx.y * p.shares * p.cols;
  float s = 0.0f;
  if (col < p.cols) {
#pragma unroll 4
    for (int y = ph; y < p.shares; y += PH) s += part[(int64_t)y * p.cols + col];
  }
  sums[ph][c] = s;
  __syncthreads();
#pragma unroll
  for (int half = PH / 2; half; half >>= 1) {
    if (ph < half) sums[ph][c] += sums[ph + half][c];
    __syncthreads();
  }
  if (ph == 0 && col < p.cols) store_elem(blockIdx.y ? p.dbias : p.dweight, p.type, col, sums[0][c]);
}

} // namespace zluda_amd
