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

// A pair of tiles is a block of 32 features of a checkpoint: its largest magnitude from the four lane groups, then eight codes
// a lane.  Features past the end count as zeros.
template <int TG>
__device__ __forceinline__ void gated_store_ckpt(uint8_t *codes, uint8_t *scales, int f0, int features, bool live, const float (&v)[TG][4]) {
  const int grp = (threadIdx.x & 63) >> 4, first = gated_first(grp), features32 = (features + 31) & ~31;
#pragma unroll
  for (int a = 0; a < TG; a += 2) {
    float x[2][4];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        x[i][e] = f0 + 16 * (a + i) + 4 * grp + e < features ? v[a + i][e] : 0.0f;
        m = max(m, ckpt_mag(x[i][e]));
      }
    typedef unsigned int u2 __attribute__((ext_vector_type(2)));
    u2 s = {m, m};
#if defined(__HIP_DEVICE_COMPILE__)
    s = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = max(s[0], s[1]);
    s = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    m = max(s[0], s[1]);
#endif
    const uint32_t byte = ckpt_scale_byte(m);
    const float inv = ckpt_inverse(byte);
    s = u2{ckpt_encode4(x[0][0], x[0][1], x[0][2], x[0][3], inv), ckpt_encode4(x[1][0], x[1][1], x[1][2], x[1][3], inv)};
#if defined(__HIP_DEVICE_COMPILE__)
    s = __builtin_amdgcn_permlane16_swap(s[0], s[1], false, false);
#endif
    const int f = f0 + 16 * a;
    if (live && f + first < features32) *(ffn_u2 *)(codes + f + first) = ffn_u2{s[0], s[1]};
    if (live && grp == 0 && f < features32) scales[f >> 5] = (uint8_t)byte;
  }
}

// G and U of TG tiles of one token a lane (biases added), features f0 .. f0 + 16 TG - 1; f0 a multiple of 32.  Every lane of the
// wave calls; `live`: the lane's token exists.
template <class E, int TG>
__device__ __forceinline__ void gated_store(const GatedParams &p, int f0, int token, bool live, float (&g)[TG][4], const float (&u)[TG][4]) {
  using raw = typename E::raw;
  if (p.kept == 1) {
    gated_store_rows<E, TG>((raw *)p.gate + token * p.ldg, f0, p.features, live, g);
    gated_store_rows<E, TG>((raw *)p.up + token * p.ldu, f0, p.features, live, u);
  } else if (p.kept == 2) {
    gated_store_ckpt<TG>((uint8_t *)p.gate + token * p.ldg, p.gate_scales + token * p.ldgs, f0, p.features, live, g);
    gated_store_ckpt<TG>((uint8_t *)p.up + token * p.ldu, p.up_scales + token * p.ldus, f0, p.features, live, u);
  }
  ffn_with_act(p.activation, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < TG; a++)
#pragma unroll
      for (int e = 0; e < 4; e++) g[a][e] = ffn_act<decltype(act)::value>(g[a][e]) * u[a][e];
  });
  gated_store_rows<E, TG>((raw *)p.h + token * p.ldh, f0, p.features, live, g);
}

} // namespace zluda_amd
