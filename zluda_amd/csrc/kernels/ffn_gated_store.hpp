// What the gated feed-forward kernels do with their products G and U: H = act(G) * U, and G and U themselves where they are
// kept.
//
// All of them leave a wave with 16 x 16 tiles in the layout of v_mfma_f32_16x16x32 with the weights as the first operand: lane
// l = 16 grp + c holds, of tile a, features 16 a + 4 grp .. + 3 of token c, and the tile of U for the same features in
// registers of its own.  So H is a product inside the lane.
#pragma once
#include "ffn_common.hpp"

namespace zluda_amd {

struct GatedParams {
  const void *x, *w, *bias;
  void *h, *gate, *up;                // gate, up: elements or codes
  uint8_t *gate_scales, *up_scales;
  int64_t ldx, ldw, ldh, ldg, ldu, ldgs, ldus;
  int32_t tokens, features, model;
  uint32_t activation;
  int32_t kept;                       // 0: nothing, 1: elements, 2: checkpoints
};

// Neighbouring tiles trade halves between the lane groups grp and grp ^ 1, after which a lane of an even group holds eight
// neighbouring features of tile a and a lane of an odd group eight of tile a + 1: from `first` on.
__device__ __forceinline__ int gated_first(int grp) { return (grp & 1) ? 4 * grp + 12 : 4 * grp; }

// a lane's four values of each tile -> 16 bytes a store instruction and lane
template <class E, int TG>
__device__ __forceinline__ void gated_store_rows(typename E::raw *row, int f0, int features, bool live, const float (&v)[TG][4]) {
  static_assert(TG % 2 == 0, "tiles are stored in pairs");
  const int first = gated_first((threadIdx.x & 63) >> 4);
#pragma unroll
  for (int a = 0; a < TG; a += 2) {
    uint32_t lo[2] = {E::pack2(v[a][0], v[a][1]), E::pack2(v[a][2], v[a][3])};
    uint32_t hi[2] = {E::pack2(v[a + 1][0], v[a + 1][1]), E::pack2(v[a + 1][2], v[a + 1][3])};
    ffn_u4 pk = {lo[0], lo[1], hi[0], hi[1]};
#if defined(__HIP_DEVICE_COMPILE__)
    typedef unsigned int u2 __attribute__((ext_vector_type(2)));
    const u2 s0 = __builtin_amdgcn_permlane16_swap(lo[0], hi[0], false, false);
    const u2 s1 = __builtin_amdgcn_permlane16_swap(lo[1], hi[1], false, false);
    pk = ffn_u4{s0[0], s1[0], s0[1], s1[1]};
#endif
    const int f = f0 + 16 * a + first, n = features - f;
    if (live && n >= 8) {
      __builtin_memcpy(row + f, &pk, 16);
    } else if (live && n > 0) {
#pragma unroll
      for (int e = 0; e < 7; e++)
        if (e < n) row[f + e] = (uint16_t)(pk[e >> 1] >> (16 * (e & 1)));
    }
  }
}

// A pair of tiles is a block of 32 features of a checkpoint: its largest magnitude from the four lane groups, then four codes of
// each tile a lane.  Four tiles are transposed between the groups (group grp gets the 16 codes of tile grp), two trade halves, so that a
// lane stores 16 or 8 neighbouring codes.  ODD: there may be values that are not finite.
// 4096 tokens, 4096 x 14336 on the persistent kernel: 666 us with nothing kept, 711 with G and U in 16 bits, 716 in 8 (724 with stores of
// eight codes and of one scale and every value asked whether it is finite; 8192 tokens, 2048 x 8192: 422, 447, 473 and 494).
template <int TG, bool ODD>
__device__ __forceinline__ void gated_store_blocks(uint8_t *codes, uint8_t *scales, int f0, int features32, bool live, const float (&v)[TG][4]) {
  static_assert(TG == 2 || TG == 4, "two or four tiles");
  typedef unsigned int u2 __attribute__((ext_vector_type(2)));
  const int grp = (threadIdx.x & 63) >> 4;
  uint32_t w[TG], byte[TG / 2];
#pragma unroll
  for (int a = 0; a < TG; a += 2) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) m = max(m, ODD ? ckpt_mag(v[a + i][e]) : f2bits(v[a + i][e]) & 0x7fffffffu);
#if defined(__HIP_DEVICE_COMPILE__)
    u2 s = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = max(s[0], s[1]);
    s = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    m = max(s[0], s[1]);
#endif
    byte[a / 2] = ckpt_scale_byte(m);
    const float inv = ckpt_inverse(byte[a / 2]);
#pragma unroll
    for (int i = 0; i < 2; i++) w[a + i] = ckpt_encode4<ODD>(v[a + i][0], v[a + i][1], v[a + i][2], v[a + i][3], inv);
  }
  if constexpr (TG == 4) {
    ffn_u4 out = {w[0], w[1], w[2], w[3]};
#if defined(__HIP_DEVICE_COMPILE__)
    const u2 a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const u2 lo = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), hi = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    out = ffn_u4{lo[0], lo[1], hi[0], hi[1]};
#endif
    if (live && f0 + 16 * grp < features32) *(ffn_u4 *)(codes + f0 + 16 * grp) = out;
    if (live && grp == 0) {
      if (f0 + 32 < features32) {
        const uint16_t both = (uint16_t)(byte[0] | byte[1] << 8);
        __builtin_memcpy(scales + (f0 >> 5), &both, 2);
      } else if (f0 < features32) {
        scales[f0 >> 5] = (uint8_t)byte[0];
      }
    }
  } else {
    u2 s = {w[0], w[1]};
#if defined(__HIP_DEVICE_COMPILE__)
    s = __builtin_amdgcn_permlane16_swap(s[0], s[1], false, false);
#endif
    const int f = f0 + gated_first(grp);
    if (live && f < features32) *(ffn_u2 *)(codes + f) = ffn_u2{s[0], s[1]};
    if (live && grp == 0 && f0 < features32) scales[f0 >> 5] = (uint8_t)byte[0];
  }
}
// G and U of TG tiles of one token a lane (biases added), features f0 .. f0 + 16 TG - 1; f0 a multiple of 32.  Every lane of the
// wave calls; `live`: the lane's token exists.  What is kept and the activation are fixed at compile time and chosen once a wave
// (gated_with): a wave that has its SIMD to itself waits for every branch, and only straight-line code lets the chains of G, U and H
// run in each other's shadow.
template <class E, int KEPT, int ACT, int TG>
__device__ __forceinline__ void gated_store(const GatedParams &p, int f0, int token, bool live, float (&g)[TG][4], float (&u)[TG][4]) {
  using raw = typename E::raw;
  if constexpr (KEPT == 1) {
    gated_store_rows<E, TG>((raw *)p.gate + token * p.ldg, f0, p.features, live, g);
    gated_store_rows<E, TG>((raw *)p.up + token * p.ldu, f0, p.features, live, u);
  } else if constexpr (KEPT == 2) {
    uint8_t *const gc = (uint8_t *)p.gate + token * p.ldg, *const gs = p.gate_scales + token * p.ldgs;
    uint8_t *const uc = (uint8_t *)p.up + token * p.ldu, *const us = p.up_scales + token * p.ldus;
    const int grp = (threadIdx.x & 63) >> 4, features32 = (p.features + 31) & ~31;
    uint32_t m = 0;
#pragma unroll
    for (int a = 0; a < TG; a++)
#pragma unroll
      for (int e = 0; e < 4; e++) m = max(m, max(f2bits(g[a][e]) & 0x7fffffffu, f2bits(u[a][e]) & 0x7fffffffu));
    if (__builtin_expect(f0 + 16 * TG > p.features || __any(m >= kCkptInf), 0)) {
      float x[TG][4], y[TG][4];  // features past the end count as zeros
#pragma unroll
      for (int a = 0; a < TG; a++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const bool in = f0 + 16 * a + 4 * grp + e < p.features;
          x[a][e] = in ? g[a][e] : 0.0f;
          y[a][e] = in ? u[a][e] : 0.0f;
        }
      gated_store_blocks<TG, true>(gc, gs, f0, features32, live, x);
      gated_store_blocks<TG, true>(uc, us, f0, features32, live, y);
    } else {
      gated_store_blocks<TG, false>(gc, gs, f0, features32, live, g);
      gated_store_blocks<TG, false>(uc, us, f0, features32, live, u);
    }
  }
#pragma unroll
  for (int a = 0; a < TG; a++)
#pragma unroll
    for (int e = 0; e < 4; e++) g[a][e] = ffn_act<ACT>(g[a][e]) * u[a][e];
  gated_store_rows<E, TG>((raw *)p.h + token * p.ldh, f0, p.features, live, g);
}

// calls f(integral_constant<int, KEPT>, integral_constant<int, ACT>) for what the problem asks (uniform)
template <class F>
__device__ __forceinline__ void gated_with(const GatedParams &p, F &&f) {
  if (p.kept == 0) ffn_with_act(p.activation, [&](auto act) __attribute__((always_inline)) { f(std::integral_constant<int, 0>{}, act); });
  else if (p.kept == 1) ffn_with_act(p.activation, [&](auto act) __attribute__((always_inline)) { f(std::integral_constant<int, 1>{}, act); });
  else ffn_with_act(p.activation, [&](auto act) __attribute__((always_inline)) { f(std::integral_constant<int, 2>{}, act); });
}

} // namespace zluda_amd
