// Shared pieces of the feed-forward operators' kernels (include/zluda_ffn.h): eight elements of a row at a time at any
// alignment, the activations with their derivatives, the checkpoint format, sums over a wave.
#pragma once
#include "numeric.hpp"

namespace zluda_amd {

typedef uint32_t ffn_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t ffn_u2 __attribute__((ext_vector_type(2)));

// ---- elements -------------------------------------------------------------------------------------------------------------
// Raw8: eight elements as they lie in memory.  top: the bits of the largest finite element, as 32F; top_scale: the scale byte of a checkpoint's block
// from which on a value can lie beyond it.
struct ElemBF16 {
  using raw = uint16_t;
  static constexpr uint32_t type = CUDA_R_16BF;
  static constexpr uint32_t top = 0x7f7f0000u, top_scale = 247;
  struct Raw8 { uint32_t w[4]; };
  static __device__ __forceinline__ float dec(raw v) { return dec_bf16(v); }
  static __device__ __forceinline__ raw enc(float v) { return enc_bf16(v); }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float get(const Raw8 &r, int e) { return (e & 1) ? bits2f(r.w[e >> 1] & 0xffff0000u) : bits2f(r.w[e >> 1] << 16); }
};
struct ElemF16 {
  using raw = uint16_t;
  static constexpr uint32_t type = CUDA_R_16F;
  static constexpr uint32_t top = 0x477fe000u, top_scale = 135;
  struct Raw8 { uint32_t w[4]; };
  static __device__ __forceinline__ float dec(raw v) { return dec_f16(v); }
  static __device__ __forceinline__ raw enc(float v) { return enc_f16(v); }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_f16x2(lo, hi); }
  static __device__ __forceinline__ float get(const Raw8 &r, int e) { return dec_f16((uint16_t)(r.w[e >> 1] >> (16 * (e & 1)))); }
};
struct ElemF32 {
  using raw = float;
  static constexpr uint32_t type = CUDA_R_32F;
  static constexpr uint32_t top = 0x7f7fffffu, top_scale = 247;
  struct Raw8 { uint32_t w[8]; };
  static __device__ __forceinline__ float dec(raw v) { return v; }
  static __device__ __forceinline__ raw enc(float v) { return v; }
  static __device__ __forceinline__ float get(const Raw8 &r, int e) { return bits2f(r.w[e]); }
};

// Eight elements at p, of which the first n exist (n >= 8: all); the others come back as zeros and are not touched.  p is
// aligned to the element only: gfx950 takes 16-byte accesses at any address.
template <class E>
__device__ __forceinline__ typename E::Raw8 load8(const typename E::raw *p, int n) {
  typename E::Raw8 r;
  if (n >= 8) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else {
    typename E::raw t[8];
#pragma unroll
    for (int e = 0; e < 8; e++) t[e] = e < n ? p[e] : typename E::raw(0);
    __builtin_memcpy(&r, t, sizeof(r));
  }
  return r;
}

template <class E>
__device__ __forceinline__ void store8(typename E::raw *p, const float (&v)[8], int n) {
  if (n >= 8) {
    typename E::Raw8 r;
    if constexpr (sizeof(typename E::raw) == 2) {
#pragma unroll
      for (int e = 0; e < 4; e++) r.w[e] = E::pack2(v[2 * e], v[2 * e + 1]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) r.w[e] = f2bits(v[e]);
    }
    __builtin_memcpy(p, &r, sizeof(r));
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < n) p[e] = E::enc(v[e]);
  }
}

// ---- activations ------------------------------------------------------------------------------------------------------------
// act(g) = g s with s = sigmoid(z), z = g (SiLU) or 2 sqrt(2/pi) (g + 0.044715 g^3) (GELU, tanh form), s = [g > 0] (ReLU);
// the derivative is s + g s (1 - s) dz/dg.  v_exp_f32 and v_rcp_f32 are good to 1 ulp, far inside the 16-bit results.
// ACT: ZLUDA_FFN_SILU 0, ZLUDA_FFN_GELU 1, ZLUDA_FFN_RELU 2.
template <int ACT>
__device__ __forceinline__ float ffn_sigma(float g) {
  if constexpr (ACT == 2) return g > 0.0f ? 1.0f : 0.0f;
  else if constexpr (ACT == 0) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g));
  else {
    const float c0 = -2.0f * 0.7978845608028654f * 1.4426950408889634f, c1 = 0.044715f * c0;
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * __builtin_fmaf(g * g, c1, c0)));
  }
}
template <int ACT>
__device__ __forceinline__ float ffn_act(float g) {
  if constexpr (ACT == 2) return g > 0.0f ? g : (g != g ? g : 0.0f);
  else return g * ffn_sigma<ACT>(g);
}
// act(g) and act'(g)
template <int ACT>
__device__ __forceinline__ void ffn_act_grad(float g, float &a, float &da) {
  const float s = ffn_sigma<ACT>(g);
  if constexpr (ACT == 2) {
    a = g > 0.0f ? g : (g != g ? g : 0.0f);
    da = s;
  } else {
    a = g * s;
    if constexpr (ACT == 0) {
      da = __builtin_fmaf(a, 1.0f - s, s);
    } else {
      // (beyond |g| = 64 s is 0 or 1 and the derivative of z multiplies a zero: kept finite there)
      const float gc = __builtin_amdgcn_fmed3f(g, -64.0f, 64.0f);
      const float dz = __builtin_fmaf(gc * gc, 3.0f * 0.044715f * 2.0f * 0.7978845608028654f, 2.0f * 0.7978845608028654f);
      da = __builtin_fmaf(a * (1.0f - s), dz, s);
    }
  }
}

// calls f(integral_constant<int, ACT>) for the activation at hand (uniform)
template <class F>
__device__ __forceinline__ void ffn_with_act(uint32_t act, F &&f) {
  if (act == 0) f(std::integral_constant<int, 0>{});
  else if (act == 1) f(std::integral_constant<int, 1>{});
  else f(std::integral_constant<int, 2>{});
}

// ---- checkpoints ------------------------------------------------------------------------------------------------------------
// Magnitude bits of a value as they count for a block's exponent: an integer order, and nothing that is not finite.
// Almost every block is finite, and a wave finds that out from the plain maximum of the bits: only where one is not (a uniform
// branch) are the values looked at one by one, and only there does the conversion have to turn infinities into NaN.
constexpr uint32_t kCkptInf = 0x7f800000u;
__device__ __forceinline__ uint32_t ckpt_mag(float v) {
  const uint32_t b = f2bits(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// The smallest e >= -126 with |v| <= 448 * 2^e, plus 127, from the largest magnitude's bits: 448 = 1.75 * 2^8, so e is the
// exponent of |v| less 8, one more where the fraction is above .75.
__device__ __forceinline__ uint32_t ckpt_scale_byte(uint32_t mag) {
  const int e = (int)((mag + 0x1fffffu) >> 23) - 135 + 127;
  return (uint32_t)(e < 1 ? 1 : e);
}
__device__ __forceinline__ float ckpt_scale(uint32_t byte) { return bits2f(byte << 23); }
__device__ __forceinline__ float ckpt_inverse(uint32_t byte) { return bits2f((254u - byte) << 23); }  // (byte is 1 .. 247)

// Four values to four codes; `inv` the inverse of the block's scale (a power of two: exact).  ODD: there may be values that are not
// finite; infinities are turned into NaN first (the instruction's own answer to them depends on a mode bit).
template <bool ODD>
__device__ __forceinline__ uint32_t ckpt_encode4(float a, float b, float c, float d, float inv) {
  auto fin = [&](float v) __attribute__((always_inline)) { return ODD ? (v * inv) - (v - v) : v * inv; };  // (v - v: 0, or NaN for what is not finite)
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(fin(a), fin(b), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(fin(c), fin(d), w, true);
  return (uint32_t)w;
}
__device__ __forceinline__ void ckpt_decode4(uint32_t w, float scale, float *v) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  v[0] = lo[0] * scale; v[1] = lo[1] * scale; v[2] = hi[0] * scale; v[3] = hi[1] * scale;
}

// The block of 32 that four neighbouring lanes hold eight values each of: its largest magnitude in all four.
__device__ __forceinline__ uint32_t ckpt_quad_max(uint32_t m) {
#if defined(__HIP_DEVICE_COMPILE__)
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));  // quad_perm [1,0,3,2]
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));  // quad_perm [2,3,0,1]
#endif
  return m;
}
// Eight values of a row (zeros past its end) to their place in a checkpoint.  Four neighbouring lanes hold a block, all four
// of them active; a lane whose eight columns start at or past `cols32` (the row's blocks times 32) stores nothing.
__device__ __forceinline__ void ckpt_store8(uint8_t *codes, uint8_t *scales, int col, int cols32, const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) m = max(m, f2bits(v[e]) & 0x7fffffffu);
  uint32_t byte;
  ffn_u2 out;
  if (__builtin_expect(__any(m >= kCkptInf), 0)) {
    m = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) m = max(m, ckpt_mag(v[e]));
    byte = ckpt_scale_byte(ckpt_quad_max(m));
    const float inv = ckpt_inverse(byte);
    out = ffn_u2{ckpt_encode4<true>(v[0], v[1], v[2], v[3], inv), ckpt_encode4<true>(v[4], v[5], v[6], v[7], inv)};
  } else {
    byte = ckpt_scale_byte(ckpt_quad_max(m));
    const float inv = ckpt_inverse(byte);
    out = ffn_u2{ckpt_encode4<false>(v[0], v[1], v[2], v[3], inv), ckpt_encode4<false>(v[4], v[5], v[6], v[7], inv)};
  }
  if (col < cols32) {
    *(ffn_u2 *)(codes + col) = out;
    if ((col & 31) == 0) scales[col >> 5] = (uint8_t)byte;
  }
}

// Eight values of a row of a plain matrix or of a checkpoint, as they lie there, and their decoding.  E::Raw8 or codes.
struct Ckpt8 { ffn_u2 codes; uint32_t scale; };
__device__ __forceinline__ Ckpt8 ckpt_load8(const uint8_t *codes, const uint8_t *scales, int col) {
  return Ckpt8{*(const ffn_u2 *)(codes + col), scales[col >> 5]};
}
__device__ __forceinline__ void ckpt_get8(const Ckpt8 &c, float (&v)[8]) {
  const float s = ckpt_scale(c.scale);
  ckpt_decode4(c.codes[0], s, v);
  ckpt_decode4(c.codes[1], s, v + 4);
}
// The same for an operand of the type E, with values beyond its largest as that one.  (A block's scale is the smallest under which nothing is above 448, but
// rounding takes what lies in [248, 256) times the scale to 256 times: from the last 1/32 of a type's range to the power of two behind it.  One such
// infinity in X would be a whole column of dW.)  NaN stays.  The blocks that can hold such values are a branch that hardly a wave takes.
template <class E>
__device__ __forceinline__ void ckpt_finite8(float (&v)[8]) {
  const float top = bits2f(E::top);
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = v[e] > top ? top : v[e] < -top ? -top : v[e];
}
template <class E>
__device__ __forceinline__ void ckpt_get8_finite(const Ckpt8 &c, float (&v)[8]) {
  ckpt_get8(c, v);
  if (__builtin_expect(c.scale >= E::top_scale, 0)) ckpt_finite8<E>(v);
}

// ---- sums over lanes --------------------------------------------------------------------------------------------------------
// The sum over a wave's 64 lanes, the same bits in every lane: four DPP steps inside rows of 16, then the rows.
__device__ __forceinline__ float wave_sum(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
  auto step = [&](auto ctrl) __attribute__((always_inline)) {
    v += bits2f((uint32_t)__builtin_amdgcn_mov_dpp((int)f2bits(v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  step(std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  step(std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  step(std::integral_constant<int, 0x141>{});  // row_half_mirror
  step(std::integral_constant<int, 0x140>{});  // row_mirror
  typedef unsigned int u2 __attribute__((ext_vector_type(2)));
  u2 s = __builtin_amdgcn_permlane16_swap(f2bits(v), f2bits(v), false, false);
  v = bits2f(s[0]) + bits2f(s[1]);
  s = __builtin_amdgcn_permlane32_swap(f2bits(v), f2bits(v), false, false);
  v = bits2f(s[0]) + bits2f(s[1]);
#endif
  return v;
}

} // namespace zluda_amd
