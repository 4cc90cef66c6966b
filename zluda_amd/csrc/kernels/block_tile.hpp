// Tiles of P x Q rows over K for the products of 8-bit floats with a scale for each 128 of K, and for 16-bit products grouped by expert.
//
// Stages are 128 bytes of K of the tile's rows: of 8-bit operands exactly one block of scales.  One v_mfma_f32_16x16x128_f8f6f4 multiplies a stage of a
// 16 x 16 tile, starting from zero; what it leaves is added to the accumulators with one multiply-add an element, by the product of the two scales.  (Where
// all P rows of a wave share a scale, that product is one number a lane and column of tiles; otherwise a lane's four rows have their own and it costs one
// multiplication an element more.)  The multiply-adds of a tile run two MFMAs behind it, in the vector unit's share of the matrix unit's time: 16 of its 32 cycles.
//
// Stages travel straight into a ring of LDS slots, rows as eight XOR-swizzled 16-byte chunks, behind them the scales of the tile's rows: a float for
// each row, also where 128 rows share one, so that every mode is read alike.
#pragma once
#include "gemm_mfma_pipe16.hpp"

namespace zluda_amd {

// the 32 codes of a lane's fragment, widened
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
template <int FMT>
__device__ __forceinline__ void block_widen(const v4i (&codes)[2], v8b (&wide)[4]) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
  for (int w = 0; w < 8; w++) {
    v2b lo, hi;
    if constexpr (FMT == 0) {
      lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[w >> 2][w & 3], 1.0f, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[w >> 2][w & 3], 1.0f, true);
    } else {
      lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(codes[w >> 2][w & 3], 1.0f, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(codes[w >> 2][w & 3], 1.0f, true);
    }
    wide[w >> 1][4 * (w & 1)] = lo[0]; wide[w >> 1][4 * (w & 1) + 1] = lo[1];
    wide[w >> 1][4 * (w & 1) + 2] = hi[0]; wide[w >> 1][4 * (w & 1) + 3] = hi[1];
  }
#endif
}

// The chunk swizzle, by the row within a 16-row tile alone: a lane's place in a fragment is then the same in all tiles of its wave, and an immediate
// away.  (The 16 lanes that a ds_read_b128 serves at a time hold rows 0-3 and 12-15 of one lane group, 4-11 of the next, two chunks on: 16 places.)
__device__ __forceinline__ int swz_block(int r) { return (r ^ ((r >> 3) & 1)) & 7; }

// One operand of a tile: rows from the tile's first one on, with their scales
struct TileSide {
  const uint8_t *data;
  int ld, rows;         // bytes between rows; rows there are (at least one)
  const float *scales;  // of the first row in the first block; unused by 16-bit kinds
  int s_row, s_step;    // floats from row to row (per_row) or from 128 rows to the next 128; from a block of K to the next
  bool per_row;
  int s_at;             // the first row's place in its block of 128 (tiles of 96 rows begin anywhere)
};

// 8-bit floats widened to bf16, which holds them exactly, for results in 32 bits.  The 8-bit instruction does not keep 32 bits inside: of each eight
// neighbouring products it drops what lies 2^13 below the largest one (seen with sums of two and three powers of two), which leaves sums of 128 to
// 14336 terms 1.4e-5 off (2-norm; the 16-bit instruction 1e-8).  A 16-bit result hides that in its rounding (1.7e-3, 2.1e-4), a 32-bit one does not.  Four
// v_mfma_f32_16x16x32_bf16 a tile and stage, twice the time, and 16 conversions a fragment.
constexpr int KIND_F8_WIDE = 8;
constexpr bool kind_is_block8(int kind) { return kind == KIND_F8 || kind == KIND_F8_WIDE; }

// MFMAs of a pair of fragments (32 bytes of K a lane), and number ks of them
template <int KIND>
constexpr int kBlockSteps = kind_is_block8(KIND) ? 1 : 2;
template <int KIND, int FP, int FQ>
__device__ __forceinline__ v4f block_mfma(const v4i (&p)[2], const v4i (&q)[2], int ks, v4f c) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (KIND == KIND_F8) {
    const v8i vp = {p[0][0], p[0][1], p[0][2], p[0][3], p[1][0], p[1][1], p[1][2], p[1][3]}, vq = {q[0][0], q[0][1], q[0][2], q[0][3], q[1][0], q[1][1], q[1][2], q[1][3]};
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vp, vq, c, FP, FQ, 0, 0, 0, 0);
  } else if constexpr (KIND == KIND_BF16) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, p[ks]), __builtin_bit_cast(v8b, q[ks]), c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, p[ks]), __builtin_bit_cast(v8h, q[ks]), c, 0, 0, 0);
  }
#endif
  return c;
}

// Tiles of BP x BQ in a ring of NS slots, every fragment of a stage read behind the products of the stage before it (gated_tile_kernel has the same
// loop).  One barrier a stage: behind it stage kt + 1 has landed for every wave and every wave holds its fragments of stage kt, whose slot takes stage
// kt + NS.  The waits count the instructions of the younger stages (mfma_wait_counts.hpp has the rule: rows past the end repeat the last one, so that no
// instruction lacks a round trip to memory; nothing is requested behind the end of K).
// SU: all P rows of a wave share their scales.
template <int KIND, int FP, int FQ, bool SU, int BP, int BQ, int WP, int WQ, int NS>
struct RingTile {
  static constexpr bool F8 = kind_is_block8(KIND), EXACT = KIND == KIND_F8_WIDE;
  static constexpr int NW = WP * WQ, RPP = 8 * NW, LP = BP / RPP, LQ = BQ / RPP;
  static constexpr int SP = (BP + 63) / 64 * 64, SQ = (BQ + 63) / 64 * 64, PIECES = (SP + SQ) / 64, LS = F8 ? (PIECES + NW - 1) / NW : 0;
  static constexpr int NLOAD = LP + LQ + LS;
  static constexpr int TP = BP / WP / 16, TQ = BQ / WQ / 16;
  // 16-byte words: the slots, behind them the scales of one stage more than there are slots (those of P's rows are read while their stage is multiplied, when its
  // slot is already being refilled)
  static constexpr int SLOT = (BP + BQ) * 8, S_SLOT = F8 ? (SP + SQ) / 4 : 0, S_AT = NS * SLOT, WORDS = S_AT + (NS + 1) * S_SLOT;
  static_assert(RPP % 32 == 0 && BP % RPP == 0 && BQ % RPP == 0 && (BP / WP) % 32 == 0 && BQ % (16 * WQ) == 0, "whole passes, whole pairs of tiles");
  static_assert(WORDS * 16 <= 160 * 1024 && (NS - 1) * NLOAD < 64 && NS >= 2, "LDS and vmcnt");

  // stages [first, first + stages) of rows of `kbytes` bytes, walked from `turn` of them on and round
  static __device__ __forceinline__ void run(const TileSide &P, const TileSide &Q, int kbytes, int first, int stages, int turn, v4i *lds, v4f (&acc)[TP][TQ]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave % WP, wq = wave / WP, r16 = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int a = 0; a < TP; a++)
#pragma unroll
      for (int b = 0; b < TQ; b++) acc[a][b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (stages <= 0) return;

    // ---- DMA: lane l -> row l / 8 of the eight an instruction fills, chunk l % 8 -------------------------------------------------
    const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc((void *)P.data, 0, 0x80000000, 0x00020000);
    const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void *)Q.data, 0, 0x80000000, 0x00020000);
    const int drow = wave * 8 + (lane >> 3), dchunk = ((lane & 7) ^ swz_block(drow)) * 16;  // (passes are a multiple of 32 rows apart: same swizzle)
    int op[LP], oq[LQ], os[LS > 0 ? LS : 1];
#pragma unroll
    for (int i = 0; i < LP; i++) op[i] = min(drow + RPP * i, P.rows - 1) * P.ld + dchunk;
#pragma unroll
    for (int i = 0; i < LQ; i++) oq[i] = min(drow + RPP * i, Q.rows - 1) * Q.ld + dchunk;
    // the scales: pieces of 64 rows, P's, then Q's; a wave without one of its own repeats another's
    const __amdgpu_buffer_rsrc_t rsp = __builtin_amdgcn_make_buffer_rsrc((void *)P.scales, 0, 0x80000000, 0x00020000);
    const __amdgpu_buffer_rsrc_t rsq = __builtin_amdgcn_make_buffer_rsrc((void *)Q.scales, 0, 0x80000000, 0x00020000);
#pragma unroll
    for (int i = 0; i < LS; i++) {
      const int piece = (wave + NW * i) % PIECES;
      const TileSide &side = piece < SP / 64 ? P : Q;
      const int row = min((piece < SP / 64 ? piece : piece - SP / 64) * 64 + lane, min(piece < SP / 64 ? BP : BQ, side.rows) - 1);
      os[i] = (side.per_row ? row : (row + side.s_at) >> 7) * side.s_row * 4;
    }
    auto issue = [&](auto i_c, int kt, int slot, int s_slot) __attribute__((always_inline)) {  // instruction i of a stage
      constexpr int i = decltype(i_c)::value;
      const int st = first + (kt + turn < stages ? kt + turn : kt + turn - stages), at = st * 128;
      v4i *base = &lds[slot * SLOT];
      if constexpr (i < LP + LQ) {
        const int oob = at + dchunk < kbytes ? 0 : (int)0x80000000;
        if constexpr (i < LP) lds_dma16(rp, base + wave * 64 + RPP * 8 * i, op[i] | oob, at);
        else lds_dma16(rq, base + BP * 8 + wave * 64 + RPP * 8 * (i - LP), oq[i - LP] | oob, at);
      } else {
        constexpr int j = i - LP - LQ;
        const int piece = (wave + NW * j) % PIECES;
        float *to = (float *)&lds[S_AT + s_slot * S_SLOT] + piece * 64;
        if (piece < SP / 64) lds_dma4(rsp, to, os[j], st * P.s_step * 4);  // (uniform)
        else lds_dma4(rsq, to, os[j], st * Q.s_step * 4);
      }
    };

    // ---- fragments ----------------------------------------------------------------------------------------------------------------
    constexpr int NF = 2 * (TP + TQ), NSC = F8 ? TQ + (SU ? 1 : 0) : 0, NR = NF + NSC, NM = TP * TQ * kBlockSteps<KIND>;  // LDS reads and MFMAs of a stage
    v4i fr[2][TP + TQ][2];                      // [stage parity][P tiles, Q tiles][half of a lane's 32 bytes]
    float sp[2];                                // scales: the one of the wave's P rows
    float sq[2][F8 ? TQ : 1];                   // and of a lane's column of each Q tile
    v4f sr[2];                                  // of its four rows of a P tile, and of the next
    int at_p[2], at_q[2];                       // [half]
#pragma unroll
    for (int h = 0; h < 2; h++) {
      at_p[h] = (wp * (16 * TP) + r16) * 8 + ((2 * grp + h) ^ swz_block(r16));
      at_q[h] = (BP + wq * (16 * TQ) + r16) * 8 + ((2 * grp + h) ^ swz_block(r16));
    }
    auto read = [&](auto r_c, auto cur_c, int slot, int s_slot) __attribute__((always_inline)) {  // LDS read r of a stage
      constexpr int r = decltype(r_c)::value, cur = decltype(cur_c)::value;
      const v4i *base = &lds[slot * SLOT];
      if constexpr (r < NF) {
        constexpr int i = r / 2, h = r % 2, tile = i < TP ? i : i - TP;
        fr[cur][i][h] = base[(i < TP ? at_p : at_q)[h] + tile * 128];
      } else {
        constexpr int j = r - NF;
        const float *s = (const float *)&lds[S_AT + s_slot * S_SLOT];
        if constexpr (j < TQ) sq[cur][j] = s[SP + wq * (16 * TQ) + 16 * j + r16];
        else sp[cur] = s[wp * (16 * TP)];
      }
    };
    // waits until at most `younger` stages of this wave's instructions are outstanding
    auto wait_for = [&](int younger) __attribute__((always_inline)) {
      static_for<NS>([&](auto n_c) {
        constexpr int n = NS - 1 - decltype(n_c)::value;
        if (younger == n || (n == NS - 1 && younger > n) || (n == 0 && younger < 0)) wait_vmcnt_barrier<n * NLOAD>();
      });
    };
    static_for<NS>([&](auto st_c) {
      if (decltype(st_c)::value < stages) static_for<NLOAD>([&](auto i_c) { issue(i_c, decltype(st_c)::value, decltype(st_c)::value, decltype(st_c)::value); });
    });
    wait_for(min(stages, NS) - 1);
    static_for<NR>([&](auto r_c) { read(r_c, std::integral_constant<int, 0>{}, 0, 0); });
    int slot = 0, s_slot = 0;
    auto do_stage = [&](auto cur_c, auto refill_c, int kt) __attribute__((always_inline)) {
      constexpr int cur = decltype(cur_c)::value;
      constexpr bool REFILL = decltype(refill_c)::value != 0;  // stage kt + NS exists
      using Next = std::integral_constant<int, 1 - cur>;
      const int next = slot == NS - 1 ? 0 : slot + 1, s_next = s_slot == NS ? 0 : s_slot + 1, s_last = s_slot == 0 ? NS : s_slot - 1;  // (stage kt + NS's)
      if constexpr (REFILL) wait_vmcnt_barrier<(NS - 2) * NLOAD>();
      else wait_for(min(stages - kt, NS) - 2);
      __builtin_amdgcn_sched_barrier(0);
      float s[F8 ? TQ : 1];
      if constexpr (F8 && SU) {
#pragma unroll
        for (int b = 0; b < TQ; b++) s[b] = sp[cur] * sq[cur][b];
      }
      v8b wide[EXACT ? TP + TQ : 1][4];
      if constexpr (EXACT) {
        static_for<TP + TQ>([&](auto i_c) {
          constexpr int i = decltype(i_c)::value;
          block_widen<i < TP ? FP : FQ>(fr[cur][i], wide[i]);
        });
      }
      const float *const rows = (const float *)&lds[S_AT + s_slot * S_SLOT] + wp * (16 * TP) + 4 * grp;
      if constexpr (F8 && !SU) sr[0] = *(const v4f *)rows;
      v4f t[3];
      auto add = [&](auto x_c) __attribute__((always_inline)) {
        constexpr int x = decltype(x_c)::value, a = x / TQ, b = x % TQ;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if constexpr (SU) acc[a][b][e] = __builtin_fmaf(t[x % 3][e], s[b], acc[a][b][e]);
          else acc[a][b][e] = __builtin_fmaf(t[x % 3][e], sr[a & 1][e] * sq[cur][F8 ? b : 0], acc[a][b][e]);
        }
      };
      static_for<NM>([&](auto x_c) {
        constexpr int x = decltype(x_c)::value, a = x % (TP * TQ) / TQ, b = x % TQ;
        if constexpr (EXACT) {
          t[x % 3] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
          for (int s4 = 0; s4 < 4; s4++) t[x % 3] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wide[a][s4], wide[TP + b][s4], t[x % 3], 0, 0, 0);
#endif
        } else if constexpr (F8) t[x % 3] = block_mfma<KIND, FP, FQ>(fr[cur][a], fr[cur][TP + b], 0, v4f{0.0f, 0.0f, 0.0f, 0.0f});
        else acc[a][b] = block_mfma<KIND, FP, FQ>(fr[cur][a], fr[cur][TP + b], x / (TP * TQ), acc[a][b]);
        constexpr int r0 = NR * x / NM, r1 = NR * (x + 1) / NM;
        static_for<r1 - r0>([&](auto r_c) { read(std::integral_constant<int, r0 + decltype(r_c)::value>{}, Next{}, next, s_next); });
        constexpr int d0 = REFILL ? NLOAD * x / NM : 0, d1 = REFILL ? NLOAD * (x + 1) / NM : 0;
        static_for<d1 - d0>([&](auto i_c) { issue(std::integral_constant<int, d0 + decltype(i_c)::value>{}, kt + NS, slot, s_last); });
        if constexpr (F8 && x >= 2) add(std::integral_constant<int, x - 2>{});
        // (behind the last use of tile a - 2's, whose registers these are)
        if constexpr (F8 && !SU && x >= 2 && (x - 2) % TQ == TQ - 1 && (x - 2) / TQ + 2 < TP) sr[(x - 2) / TQ & 1] = *(const v4f *)(rows + 16 * ((x - 2) / TQ + 2));
        if constexpr (F8 && !SU && x == 0 && TP > 1) sr[1] = *(const v4f *)(rows + 16);
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (F8 && NM >= 2) add(std::integral_constant<int, NM - 2>{});
      if constexpr (F8) add(std::integral_constant<int, NM - 1>{});
      slot = next;
      s_slot = s_next;
    };
    using C0 = std::integral_constant<int, 0>;
    using C1 = std::integral_constant<int, 1>;
    int kt = 0;
    for (; kt + 1 + NS < stages; kt += 2) {
      do_stage(C0{}, C1{}, kt);
      do_stage(C1{}, C1{}, kt + 1);
    }
    if (kt + NS < stages) do_stage(C0{}, C1{}, kt++);
    if (kt & 1) do_stage(C1{}, C0{}, kt++);
    for (; kt + 1 < stages; kt += 2) {
      do_stage(C0{}, C0{}, kt);
      do_stage(C1{}, C0{}, kt + 1);
    }
    if (kt < stages) do_stage(C0{}, C0{}, kt);
  }
};

// Tiles of 256 x 256 on eight waves of 128 x 64, two slots: the sub-steps of gemm_mfma_pipe16_kernel over halves of the wave tile,
//   (P0,QA) reads QB | (P0,QB) reads P1 | barrier | (P1,QB) reads P0 of the next stage | (P1,QA) reads its QB
// with QA the Q half 0 in even stages and 1 in odd ones.  Behind the barrier the slot takes stage kt + 2.  All waits are for everything in flight; rows past
// the end lie outside the buffers' windows and become zeros.
template <int KIND, int FP, int FQ>
struct WideTile {
  static constexpr bool F8 = KIND == KIND_F8;
  static constexpr int BP = 256, BQ = 256, WP = 2, WQ = 4, NW = 8, TP = 8, TQ = 4, RPP = 64, LP = 4, LQ = 4, LS = F8 ? 1 : 0, NLOAD = LP + LQ + LS;
  // LDS in 16-byte words: P's slots, Q's, the scales'.  (So one address a lane and half reaches every tile of an operand in both slots by an immediate.)
  static constexpr int SLOT = 256 * 8, S_SLOT = (BP + BQ) / 4, Q_AT = 2 * SLOT, S_AT = 4 * SLOT, WORDS = S_AT + (F8 ? 2 * S_SLOT : 0);

  static __device__ __forceinline__ void run(const TileSide &P, const TileSide &Q, int kbytes, int first, int stages, v4i *lds, v4f (&acc)[TP][TQ]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave % WP, wq = wave / WP, r16 = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int a = 0; a < TP; a++)
#pragma unroll
      for (int b = 0; b < TQ; b++) acc[a][b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (stages <= 0) return;
    auto window = [&](const TileSide &s) { return (int)min((int64_t)min(s.rows, 256) * s.ld - (s.ld - kbytes), (int64_t)0x7fffffff); };
    const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc((void *)P.data, 0, window(P), 0x00020000);
    const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void *)Q.data, 0, window(Q), 0x00020000);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)(wave < 4 ? P.scales : Q.scales), 0, 0x80000000, 0x00020000);
    const int drow = wave * 8 + (lane >> 3), dchunk = ((lane & 7) ^ swz_block(drow)) * 16;
    const int op = drow * P.ld + dchunk, oq = drow * Q.ld + dchunk;
    int os = 0;
    if constexpr (F8) {
      const TileSide &side = wave < 4 ? P : Q;
      const int row = min((wave & 3) * 64 + lane, side.rows - 1);
      os = (side.per_row ? row * side.s_row : (row >> 7) * side.s_row) * 4;
    }
    const int s_step = (wave < 4 ? P.s_step : Q.s_step) * 4;
    // Instruction i of stage kt into slot `slot`.  What lies past the end of K, or past the last stage, is out of the windows: zeros, no traffic.  (One
    // loop for all stages: with bodies of their own for the last ones the accumulators go to memory and back on the way there.)
    const int end = min(kbytes, (first + stages) * 128);
    auto issue = [&](auto i_c, int kt, int slot) __attribute__((always_inline)) {
      constexpr int i = decltype(i_c)::value;
      const int at = (first + kt) * 128;
      if constexpr (i < LP + LQ) {
        const int oob = at + dchunk < end ? 0 : (int)0x80000000;
        if constexpr (i < LP) lds_dma16(rp, &lds[slot * SLOT + wave * 64 + RPP * 8 * i], op | oob, at + RPP * i * P.ld);
        else lds_dma16(rq, &lds[Q_AT + slot * SLOT + wave * 64 + RPP * 8 * (i - LP)], oq | oob, at + RPP * (i - LP) * Q.ld);
      } else {
        lds_dma4(rs, (float *)&lds[S_AT + slot * S_SLOT] + wave * 64, os | (kt < stages ? 0 : (int)0x80000000), (first + kt) * s_step);
      }
    };
    int at_p[2], at_q[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      at_p[h] = (wp * 128 + r16) * 8 + ((2 * grp + h) ^ swz_block(r16));
      at_q[h] = Q_AT + (wq * 64 + r16) * 8 + ((2 * grp + h) ^ swz_block(r16));
    }
    const float *const s_q = (const float *)&lds[S_AT] + BP + wq * 64 + r16, *const s_p = (const float *)&lds[S_AT] + wp * 128;
    v4i pf[2][4][2], qf[2][2][2];  // [half of the wave tile][tile][half of a lane's 32 bytes]
    float sc[TQ];                  // the stage's factors
    float nq[TQ], np = 0.0f;       // the next one's
    auto read_p = [&](auto h_c, auto r_c, int slot) __attribute__((always_inline)) {
      constexpr int h = decltype(h_c)::value, r = decltype(r_c)::value, tile = h * 4 + r / 2;
      pf[h][r / 2][r % 2] = lds[slot * SLOT + at_p[r % 2] + tile * 128];
    };
    auto read_q = [&](auto h_c, auto r_c, int slot) __attribute__((always_inline)) {
      constexpr int h = decltype(h_c)::value, r = decltype(r_c)::value, tile = h * 2 + r / 2;
      qf[h][r / 2][r % 2] = lds[slot * SLOT + at_q[r % 2] + tile * 128];
    };
    auto read_s = [&](auto r_c, int slot) __attribute__((always_inline)) {
      constexpr int r = decltype(r_c)::value;
      if constexpr (r < TQ) nq[r] = s_q[slot * S_SLOT * 4 + 16 * r];
      else np = s_p[slot * S_SLOT * 4];
    };
    using C0 = std::integral_constant<int, 0>;
    using C1 = std::integral_constant<int, 1>;
    static_for<NLOAD>([&](auto i_c) { issue(i_c, 0, 0); });
    static_for<NLOAD>([&](auto i_c) { issue(i_c, 1, 1); });
    wait_vmcnt_barrier<0>();
    // A wave whose share lies past the end of P or Q brings its part of the stages and meets the others, no more: the waves beside it on its SIMD have the
    // matrix unit to themselves (a tile of at most 128 rows of Q takes little more than half the time).
    if (wp * 128 >= P.rows || wq * 64 >= Q.rows) {
      for (int kt = 0; kt < stages; kt++) {
        wait_vmcnt_barrier<0>();
        static_for<NLOAD>([&](auto i_c) { issue(i_c, kt + 2, kt & 1); });
      }
      __builtin_amdgcn_s_waitcnt(0);
      return;
    }
    static_for<8>([&](auto r_c) { read_p(C0{}, r_c, 0); });
    static_for<4>([&](auto r_c) { read_q(C0{}, r_c, 0); });
    if constexpr (F8) static_for<TQ + 1>([&](auto r_c) { read_s(r_c, 0); });
    v4f t[3];
    auto do_stage = [&](auto odd_c, int kt) __attribute__((always_inline)) {
      constexpr int ODD = decltype(odd_c)::value;
      constexpr int slot = ODD, next = 1 - ODD;
      using QA = std::integral_constant<int, ODD>;
      using QB = std::integral_constant<int, 1 - ODD>;
      if constexpr (F8) {
#pragma unroll
        for (int b = 0; b < TQ; b++) sc[b] = np * nq[b];
      }
      // MFMA g of the stage's 32: sub-step g / 8, tiles (i, j) of its halves
      auto add = [&](auto g_c) __attribute__((always_inline)) {
        constexpr int g = decltype(g_c)::value, sub = g / 8, ph = sub / 2, qh = sub == 0 || sub == 3 ? ODD : 1 - ODD, i = g % 8 / 2, j = g % 2;
        v4f &c = acc[ph * 4 + i][qh * 2 + j];
#pragma unroll
        for (int e = 0; e < 4; e++) c[e] = __builtin_fmaf(t[g % 3][e], sc[qh * 2 + j], c[e]);
      };
      auto substep = [&](auto sub_c, auto &&rd, auto nr_c, auto l0_c, auto l1_c) __attribute__((always_inline)) {
        constexpr int sub = decltype(sub_c)::value, ph = sub / 2, qh = sub == 0 || sub == 3 ? ODD : 1 - ODD;
        constexpr int NR = decltype(nr_c)::value, L0 = decltype(l0_c)::value, L1 = decltype(l1_c)::value;
        constexpr int NM = 8 * kBlockSteps<KIND>;
        static_for<NM>([&](auto x_c) {
          constexpr int x = decltype(x_c)::value, i = x % 8 / 2, j = x % 2, g = sub * 8 + x;
          if constexpr (F8) t[g % 3] = block_mfma<KIND, FP, FQ>(pf[ph][i], qf[qh][j], 0, v4f{0.0f, 0.0f, 0.0f, 0.0f});
          else acc[ph * 4 + i][qh * 2 + j] = block_mfma<KIND, FP, FQ>(pf[ph][i], qf[qh][j], x / 8, acc[ph * 4 + i][qh * 2 + j]);
          constexpr int r0 = NR * x / NM, r1 = NR * (x + 1) / NM;
          static_for<r1 - r0>([&](auto r_c) { rd(std::integral_constant<int, r0 + decltype(r_c)::value>{}); });
          constexpr int d0 = L0 + (L1 - L0) * x / NM, d1 = L0 + (L1 - L0) * (x + 1) / NM;
          static_for<d1 - d0>([&](auto i_c) { issue(std::integral_constant<int, d0 + decltype(i_c)::value>{}, kt + 2, slot); });
          if constexpr (F8 && g >= 2) add(std::integral_constant<int, g - 2>{});
          __builtin_amdgcn_sched_barrier(0);
        });
      };
      using N4 = std::integral_constant<int, 4>;
      using N8 = std::integral_constant<int, 8>;
      using NL = std::integral_constant<int, NLOAD>;
      using NH = std::integral_constant<int, NLOAD / 2>;
      substep(C0{}, [&](auto r_c) { read_q(QB{}, r_c, slot); }, N4{}, C0{}, C0{});
      substep(C1{}, [&](auto r_c) { read_p(C1{}, r_c, slot); }, N8{}, C0{}, C0{});
      wait_vmcnt_barrier<0>();
      __builtin_amdgcn_sched_barrier(0);
      substep(std::integral_constant<int, 2>{}, [&](auto r_c) { read_p(C0{}, r_c, next); }, N8{}, C0{}, NH{});
      substep(std::integral_constant<int, 3>{}, [&](auto r_c) {
        constexpr int r = decltype(r_c)::value;
        if constexpr (r < 4) read_q(QB{}, r_c, next);
        else read_s(std::integral_constant<int, r - 4>{}, next);
      }, std::integral_constant<int, F8 ? 4 + TQ + 1 : 4>{}, NH{}, NL{});
      if constexpr (F8) {
        add(std::integral_constant<int, 30>{});
        add(std::integral_constant<int, 31>{});
      }
    };
    for (int kt = 0; kt < stages; kt += 2) {
      do_stage(C0{}, kt);
      if (kt + 1 < stages) do_stage(C1{}, kt + 1);
    }
    __builtin_amdgcn_s_waitcnt(0);  // (what is in flight past the end writes zeros: not into what comes next)
  }
};

} // namespace zluda_amd
