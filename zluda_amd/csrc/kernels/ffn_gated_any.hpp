// Gated feed-forward products for operands at any alignment, pitch and size (include/zluda_ffn.h).
//
// A workgroup of four waves takes 64 tokens and 32 features: 64 rows of W, 32 of Wg and the 32 of Wu that belong to them.
// Stages of 32 K elements go through registers, four of them on their way, into LDS (a load of eight elements at any alignment, element by element
// at the end of K), rows padded to 80 bytes so that the 16-byte fragment reads of 16 rows spread over the banks.
//
// Bound by the round trips of its loads where there are few tokens (one at a time 28.7 us for 17 tokens, 1500 x 4000, four 16.3; one token, 4095 x 14336
// 121 and 62, 3.8 TB/s), by its little tiles where there are many (2000, 2047 x 5632 280 us, 329 TFLOP/s).
#pragma once
#include "ffn_gated_store.hpp"

namespace zluda_amd {

template <class E>
__device__ __forceinline__ void ffn_mfma(ffn_u4 a, ffn_u4 b, float __attribute__((ext_vector_type(4))) & c) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __bf16 b8 __attribute__((ext_vector_type(8)));
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  if constexpr (E::type == CUDA_R_16BF) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
#endif
}

template <class E>
__global__ __launch_bounds__(256) void gated_any_kernel(GatedParams p) {
  using raw = typename E::raw;
  typedef float f4 __attribute__((ext_vector_type(4)));
  constexpr int PITCH = 5;  // 16-byte words of a row: four and a pad
  __shared__ ffn_u4 lw[64 * PITCH], lx[64 * PITCH];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, r16 = lane & 15, grp = lane >> 4;
  const int f0 = blockIdx.y * 32, t0 = blockIdx.x * 64;
  // the row and the eight K elements that this thread brings: rows past the end repeat the last one, their results are dropped
  const int row = t >> 2, kc = (t & 3) * 8;
  const int f = min(f0 + (row & 31), p.features - 1) + (row < 32 ? 0 : p.features);
  const raw *w = (const raw *)p.w + (int64_t)f * p.ldw, *x = (const raw *)p.x + (int64_t)min(t0 + row, p.tokens - 1) * p.ldx;
  f4 acc[4];
#pragma unroll
  for (int a = 0; a < 4; a++) acc[a] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  auto stage = [&](const typename E::Raw8 &rw, const typename E::Raw8 &rx) __attribute__((always_inline)) {
    __syncthreads();
    lw[row * PITCH + (t & 3)] = __builtin_bit_cast(ffn_u4, rw);
    lx[row * PITCH + (t & 3)] = __builtin_bit_cast(ffn_u4, rx);
    __syncthreads();
    const ffn_u4 b = lx[(wave * 16 + r16) * PITCH + grp];
#pragma unroll
    for (int a = 0; a < 4; a++) ffn_mfma<E>(lw[(a * 16 + r16) * PITCH + grp], b, acc[a]);
  };
  constexpr int AHEAD = 4;
  const int whole = p.model / 32;  // stages without an end inside
  typename E::Raw8 qw[AHEAD], qx[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; i++)
    if (i < whole) {
      qw[i] = load8<E>(w + 32 * i + kc, 8);
      qx[i] = load8<E>(x + 32 * i + kc, 8);
    }
  int at = 0;
  for (; at + AHEAD <= whole; at += AHEAD) {
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {
      stage(qw[i], qx[i]);
      if (at + AHEAD + i < whole) {
        qw[i] = load8<E>(w + 32 * (at + AHEAD + i) + kc, 8);
        qx[i] = load8<E>(x + 32 * (at + AHEAD + i) + kc, 8);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < AHEAD; i++)
    if (at + i < whole) stage(qw[i], qx[i]);
  if (p.model & 31) {
    const int left = (p.model & 31) - kc;
    stage(load8<E>(w + 32 * whole + kc, left), load8<E>(x + 32 * whole + kc, left));
  }
  float g[2][4], u[2][4];
#pragma unroll
  for (int a = 0; a < 2; a++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int fe = min(f0 + 16 * a + 4 * grp + e, p.features - 1);
      g[a][e] = acc[a][e] + (p.bias ? E::dec(((const raw *)p.bias)[fe]) : 0.0f);
      u[a][e] = acc[a + 2][e] + (p.bias ? E::dec(((const raw *)p.bias)[p.features + fe]) : 0.0f);
    }
  const int token = t0 + wave * 16 + r16;
  gated_with(p, [&](auto kept, auto act) __attribute__((always_inline)) {
    gated_store<E, decltype(kept)::value, decltype(act)::value>(p, f0, token, token < p.tokens, g, u);
  });
}

} // namespace zluda_amd
