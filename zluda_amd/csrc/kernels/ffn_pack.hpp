// Packed matrices (include/zluda_ffn.h): E4M3 codes with a float scale for each 128 neighbours of a row, or each block of 128 x 128.  Packing of
// activations, with the gated activation in front of it, and back.
//
// Memory bound: every value is read once and every code written once.  A thread has eight neighbouring columns, so 16 neighbouring lanes -- a row of
// the DPP network -- hold the 128 that share a scale, and its largest magnitude takes four DPP steps.  Gated activation of 8192 x 14336, bf16: 103 us,
// 5.7 TB/s; back 63 us, 5.6.
#pragma once
#include "ffn_common.hpp"

namespace zluda_amd {

constexpr int kPack = 128;

// the largest of 16 neighbouring lanes, in all of them
__device__ __forceinline__ uint32_t pack_max16(uint32_t m) {
#if defined(__HIP_DEVICE_COMPILE__)
  m = ckpt_quad_max(m);
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xf, 0xf, true));  // row_half_mirror
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x140, 0xf, 0xf, true));  // row_mirror
#endif
  return m;
}
// Magnitude bits of eight values as they count for a scale: what is not finite does not
__device__ __forceinline__ uint32_t pack_mag8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) m = max(m, f2bits(v[e]) & 0x7fffffffu);
  if (__builtin_expect(__any(m >= kCkptInf), 0)) {
    m = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) m = max(m, ckpt_mag(v[e]));
  }
  return m;
}
// (448 = 1.75 * 2^8; the quotient correctly rounded, and no subnormal: its reciprocal is finite)
__device__ __forceinline__ float pack_scale(uint32_t mag) { return __builtin_fmaxf(bits2f(mag) / 448.0f, 0x1p-126f); }

// Four codes.  The quotient by way of the reciprocal (1 ulp) and one correction from its remainder, which leaves it within an ulp of v / s in 32 bits: what
// E4M3 makes of it differs from what the exact quotient gives only within 2^-23 of a border.  The correction makes NaN of infinities.
__device__ __forceinline__ uint32_t pack_encode4(float a, float b, float c, float d, float s, float inv) {
  auto div = [&](float v) __attribute__((always_inline)) {
    const float q = v * inv;
    return __builtin_fmaf(__builtin_fmaf(-q, s, v), inv, q);
  };
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(div(a), div(b), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(div(c), div(d), w, true);
  return (uint32_t)w;
}
__device__ __forceinline__ ffn_u2 pack_encode8(const float (&v)[8], float s) {
  const float inv = __builtin_amdgcn_rcpf(s);
  return ffn_u2{pack_encode4(v[0], v[1], v[2], v[3], s, inv), pack_encode4(v[4], v[5], v[6], v[7], s, inv)};
}
// eight codes of a row, of which the first n exist, at any address
__device__ __forceinline__ void pack_put8(uint8_t *p, ffn_u2 codes, int n) {
  if (n >= 8) {
    __builtin_memcpy(p, &codes, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < n) p[e] = (uint8_t)(codes[e >> 2] >> (8 * (e & 3)));
  }
}

struct ActivateParams {
  const void *gate, *up;  // up or NULL
  void *y;                // or NULL
  uint8_t *codes;         // or NULL
  float *scales;
  int64_t rows, ldg, ldu, ldy, ldc, lds;
  int32_t cols;
  uint32_t activation;    // ZLUDA_FFN_*, 3: a copy
};

// h = act(g) u, or act(g)
__device__ __forceinline__ void activate8(uint32_t act, bool gated, float (&g)[8], const float (&u)[8]) {
  if (act < 3) {
    ffn_with_act(act, [&](auto a) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 8; e++) g[e] = ffn_act<decltype(a)::value>(g[e]);
    });
  }
  if (gated) {
#pragma unroll
    for (int e = 0; e < 8; e++) g[e] *= u[e];
  }
}

// Scales of single rows.  A workgroup has 512 columns and four rows at a time, a wave each.  (Several rows a thread, whose scales lie side by side, gain nothing: two,
// four and eight of 8192 x 14336 102, 103 and 112 us, one 103, of 1024 x 8192 9.3, 10.3 and 12.1, one 8.7.)
template <class E>
__global__ __launch_bounds__(256) void activate_kernel(ActivateParams p) {
  using raw = typename E::raw;
  const int lane = threadIdx.x & 63, col = 8 * (blockIdx.x * 64 + lane), n = p.cols - col;
  for (int64_t row = blockIdx.y * 4 + (threadIdx.x >> 6); row < p.rows; row += (int64_t)gridDim.y * 4) {
    const typename E::Raw8 rg = load8<E>((const raw *)p.gate + row * p.ldg + col, n);
    float h[8], u[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      h[e] = E::get(rg, e);
      u[e] = 1.0f;
    }
    if (p.up) {
      const typename E::Raw8 ru = load8<E>((const raw *)p.up + row * p.ldu + col, n);
#pragma unroll
      for (int e = 0; e < 8; e++) u[e] = E::get(ru, e);
    }
    activate8(p.activation, p.up != nullptr, h, u);
    if (p.y) store8<E>((raw *)p.y + row * p.ldy + col, h, n);
    if (p.codes) {
#pragma unroll
      for (int e = 0; e < 8; e++) h[e] = e < n ? h[e] : 0.0f;  // (act(0) is 0, but a copy of what a row's neighbour holds is not asked for)
      const float s = pack_scale(pack_max16(pack_mag8(h)));
      pack_put8(p.codes + row * p.ldc + col, pack_encode8(h, s), n);
      if ((lane & 15) == 0 && n > 0) p.scales[(int64_t)(col >> 7) * p.lds + row] = s;
    }
  }
}

// Scales of blocks of 128 x 128: a workgroup each, 8 x 8 values a thread, held until the block's largest magnitude is known
template <class E>
__global__ __launch_bounds__(256) void activate_blocks_kernel(ActivateParams p) {
  using raw = typename E::raw;
  __shared__ uint32_t tops[4];
  const int col = blockIdx.x * kPack + 8 * (threadIdx.x & 15), n = p.cols - col;
  for (int64_t blk = blockIdx.y; blk * kPack < p.rows; blk += gridDim.y) {
    const int64_t row0 = blk * kPack + 8 * (threadIdx.x >> 4);
    float h[8][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int live = row0 + i < p.rows ? n : 0;
      const typename E::Raw8 rg = load8<E>((const raw *)p.gate + (row0 + i) * p.ldg + col, live);
      float u[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        h[i][e] = E::get(rg, e);
        u[e] = 1.0f;
      }
      if (p.up) {
        const typename E::Raw8 ru = load8<E>((const raw *)p.up + (row0 + i) * p.ldu + col, live);
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = E::get(ru, e);
      }
      activate8(p.activation, p.up != nullptr, h[i], u);
      if (p.y) store8<E>((raw *)p.y + (row0 + i) * p.ldy + col, h[i], live);
#pragma unroll
      for (int e = 0; e < 8; e++) h[i][e] = e < live ? h[i][e] : 0.0f;
      m = max(m, pack_mag8(h[i]));
    }
    if (!p.codes) continue;
    m = pack_max16(m);
#if defined(__HIP_DEVICE_COMPILE__)
    m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
#endif
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
    __syncthreads();
    const float s = pack_scale(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
    __syncthreads();  // (the next block's maxima)
#pragma unroll
    for (int i = 0; i < 8; i++) pack_put8(p.codes + (row0 + i) * p.ldc + col, pack_encode8(h[i], s), row0 + i < p.rows ? n : 0);
    if (threadIdx.x == 0) p.scales[blk * p.lds + blockIdx.x] = s;
  }
}

struct UnpackParams {
  const uint8_t *codes;
  const float *scales;
  void *y;
  int64_t rows, ldc, lds, ldy;
  int32_t cols;
  int32_t blocks;  // scales of blocks of 128 rows
};
template <class E>
__global__ __launch_bounds__(256) void unpack_kernel(UnpackParams p) {
  const int col = 8 * (blockIdx.x * 64 + (threadIdx.x & 63)), n = p.cols - col;
  if (n <= 0) return;
  const float top = bits2f(E::top);
  for (int64_t row = blockIdx.y * 4 + (threadIdx.x >> 6); row < p.rows; row += (int64_t)gridDim.y * 4) {
    const uint8_t *from = p.codes + row * p.ldc + col;
    ffn_u2 c = {0, 0};
    if (n >= 8) {
      __builtin_memcpy(&c, from, 8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (e < n) c[e >> 2] |= (uint32_t)from[e] << (8 * (e & 3));
    }
    const float s = p.scales[p.blocks ? (row >> 7) * p.lds + (col >> 7) : (int64_t)(col >> 7) * p.lds + row];
    float v[8];
    ckpt_decode4(c[0], s, v);
    ckpt_decode4(c[1], s, v + 4);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = v[e] > top ? top : v[e] < -top ? -top : v[e];
    store8<E>((typename E::raw *)p.y + row * p.ldy + col, v, n);
  }
}

} // namespace zluda_amd
