// Gated feed-forward products in tiles of BF features and BT tokens, one a workgroup, from a single token on up to where the
// persistent kernel has enough tiles.
//
// Few tokens are bound by the read of W: one token, 4096 x 14336, takes 41.0 us (235 MB at 5.7 TB/s; a large copy moves 5.2), 32
// tokens 42.8, 64 tokens (64 x 64 tiles) 44.4.  More are bound by the matrix cores and LDS: 256 tokens (128 x 128) 70 us, 860 TFLOP/s.
//
// Stages of 128 K bytes of the tile's 2 BF rows of W (BF of Wg, BF of Wu) and BT rows of X travel straight into a ring of NS
// slots in LDS; rows are eight 16-byte chunks, XOR-swizzled as in gemm_mfma.hpp.  The fragments of a stage are read from LDS behind
// the products of the stage before it, so a wave waits neither for memory nor for LDS once it runs.  One barrier a stage: behind
// it stage kt + 1 has landed for every wave and every wave holds its fragments of stage kt, whose slot takes stage kt + NS.  The waits
// count the instructions of the younger stages (mfma_wait_counts.hpp has the rule: loads that make a round trip to memory retire in
// order; a K tail holds its row's first chunk).  Nothing is requested behind the end of K, and the last waits count what is left.
//
// LDS rows of W: for each of the WP wave rows its FW gate rows, then its FW up rows.
#pragma once
#include "ffn_gated_any.hpp"
#include "gemm_mfma_pipe.hpp"

namespace zluda_amd {

struct GatedTileParams : MfmaParams {
  GatedParams gated;
};

template <class E, int BF, int BT, int WP, int WQ, int NS>
__global__ __launch_bounds__(64 * WP *WQ) void gated_tile_kernel(GatedTileParams prm) {
  using raw = typename E::raw;
  constexpr int BP = 2 * BF;
  constexpr PipeCounts PC = pipe_counts(false, BP, BT, WP, WQ, 128, NS);
  constexpr int RPP = PC.rpp, LP = PC.lp, LQ = PC.lq, NLOAD = PC.nload;  // rows a DMA pass of the workgroup fills, instructions a stage
  constexpr int FW = BF / WP, TG = FW / 16, TQ = BT / WQ / 16;  // a wave's share
  constexpr int STAGE = (BP + BT) * 8;                // one slot in 16-byte words
  static_assert(RPP % 32 == 0 && BP % RPP == 0 && BT % RPP == 0 && FW % 32 == 0 && BT % (16 * WQ) == 0, "whole passes, whole pairs of tiles");
  static_assert(NS * STAGE * 16 <= 160 * 1024 && (NS - 1) * NLOAD < 64, "LDS and vmcnt");
  __shared__ v4i lds[NS * STAGE];

  const GatedParams &p = prm.gated;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wp = wave % WP, wq = wave / WP, r16 = lane & 15, grp = lane >> 4;
  const WorkItem item = work_item(prm, blockIdx.x);
  const int f0 = item.p * BF, t0 = item.q * BT;

  // ---- DMA: lane l -> row l / 8 of the eight an instruction fills, chunk l % 8 -------------------------------------------------
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void *)p.w, 0, 0x80000000, 0x00020000);
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void *)p.x, 0, 0x80000000, 0x00020000);
  const int drow = wave * 8 + (lane >> 3), dchunk = ((lane & 7) ^ swz(drow)) * 16;  // (passes are a multiple of 32 rows apart: same swizzle)
  int ow[LP], ox[LQ];
#pragma unroll
  for (int i = 0; i < LP; i++) {
    const int r = drow + RPP * i, j = r % (2 * FW);
    const int f = min(f0 + r / (2 * FW) * FW + j % FW, p.features - 1) + (j < FW ? 0 : p.features);
    ow[i] = f * (int)p.ldw * 2 + dchunk;
  }
#pragma unroll
  for (int i = 0; i < LQ; i++) ox[i] = min(t0 + drow + RPP * i, p.tokens - 1) * (int)p.ldx * 2 + dchunk;
  const int kbytes = p.model * 2, stages = (kbytes + 127) / 128;
  // Tiles start their walk along K three stages apart and wrap round.  All starting at K = 0, they would read the same few
  // columns of W at a time, and rows a power of two apart share memory channels (one token, 4096 x 14336: 50.6 -> 42.7 us; rows of
  // 10 KiB do not mind).  Tiles of the same features walk alike and share W in the caches.
  const int turn = item.p * 3 % stages;
  auto issue = [&](auto i_c, int kt, int slot) __attribute__((always_inline)) {  // instruction i of a stage
    constexpr int i = decltype(i_c)::value;
    const int at = (kt + turn < stages ? kt + turn : kt + turn - stages) * 128, oob = at + dchunk < kbytes ? 0 : (int)0x80000000;
    v4i *base = &lds[slot * STAGE + wave * 64];
    if constexpr (i < LP) lds_dma16(rw, base + RPP * 8 * i, ow[i] | oob, at);
    else lds_dma16(rx, base + BP * 8 + RPP * 8 * (i - LP), ox[i - LP] | oob, at);
  };

  v4f acc[2 * TG][TQ];
#pragma unroll
  for (int a = 0; a < 2 * TG; a++)
#pragma unroll
    for (int b = 0; b < TQ; b++) acc[a][b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int NR = 2 * (2 * TG + TQ), NM = 2 * 2 * TG * TQ;  // fragment reads and MFMAs of a stage
  ffn_u4 fr[2][2][2 * TG + TQ];                               // [stage parity][half of the stage][W tiles, X tiles]
  // Word of a fragment inside a slot: tiles are 16 rows apart and the swizzle repeats after 32.  A lane group's two pieces of a stage are
  // neighbours (any K order will do that is the same for W and X): so no part of a ds_read_b128 meets a bank conflict.
  int at_w[2][2], at_x[2][2];  // [half][tile parity]
#pragma unroll
  for (int h = 0; h < 2; h++)
#pragma unroll
    for (int par = 0; par < 2; par++) {
      const int rp = wp * 2 * FW + 16 * par + r16, rq = BP + wq * (16 * TQ) + 16 * par + r16;
      at_w[h][par] = rp * 8 + ((2 * grp + h) ^ swz(rp));
      at_x[h][par] = rq * 8 + ((2 * grp + h) ^ swz(rq));
    }
  auto read = [&](auto r_c, auto cur_c, int slot) __attribute__((always_inline)) {  // fragment read r of a stage
    constexpr int r = decltype(r_c)::value, h = r / (2 * TG + TQ), i = r % (2 * TG + TQ), cur = decltype(cur_c)::value;
    constexpr int tile = i < 2 * TG ? i : i - 2 * TG;
    fr[cur][h][i] = __builtin_bit_cast(ffn_u4, lds[slot * STAGE + (i < 2 * TG ? at_w : at_x)[h][tile & 1] + (tile >> 1) * 256]);
  };
  // waits until at most `younger` stages of this wave's instructions are outstanding
  auto wait_for = [&](int younger) __attribute__((always_inline)) {
    if (younger >= NS - 1) wait_vmcnt_barrier<(NS - 1) * NLOAD>();
    else if (younger == NS - 2) wait_vmcnt_barrier<(NS - 2) * NLOAD>();
    else if (NS > 3 && younger == 1) wait_vmcnt_barrier<NLOAD>();
    else wait_vmcnt_barrier<0>();
  };
  static_assert(PC.wait_prologue == (NS - 1) * NLOAD && PC.wait_stage == (NS - 2) * NLOAD && NS <= 4, "counts");
  static_for<NS>([&](auto st_c) {
    if (decltype(st_c)::value < stages) static_for<NLOAD>([&](auto i_c) { issue(i_c, decltype(st_c)::value, decltype(st_c)::value); });
  });
  wait_for(stages - 1);
  static_for<NR>([&](auto r_c) { read(r_c, std::integral_constant<int, 0>{}, 0); });
  int slot = 0;
  auto do_stage = [&](auto cur_c, auto refill_c, int kt) __attribute__((always_inline)) {
    constexpr int cur = decltype(cur_c)::value;
    constexpr bool REFILL = decltype(refill_c)::value != 0;  // stage kt + NS exists
    using Next = std::integral_constant<int, 1 - cur>;
    const int next = slot == NS - 1 ? 0 : slot + 1;
    if constexpr (REFILL) wait_vmcnt_barrier<PC.wait_stage>();
    else wait_for(min(stages - kt, NS) - 2);
    __builtin_amdgcn_sched_barrier(0);
    // the reads and the DMA spread over all of the MFMAs (reads first, then the DMA: up to 7 % slower, 100 tokens, 2048 x 5632 16.1 against
    // 14.9 us; a stage's requests set out earlier)
    static_for<NM>([&](auto x_c) {
      constexpr int x = decltype(x_c)::value, h = x / (2 * TG * TQ), a = x % (2 * TG * TQ) / TQ, b = x % TQ;
      ffn_mfma<E>(fr[cur][h][a], fr[cur][h][2 * TG + b], acc[a][b]);
      constexpr int r0 = NR * x / NM, r1 = NR * (x + 1) / NM;
      static_for<r1 - r0>([&](auto r_c) { read(std::integral_constant<int, r0 + decltype(r_c)::value>{}, Next{}, next); });
      constexpr int d0 = REFILL ? NLOAD * x / NM : 0, d1 = REFILL ? NLOAD * (x + 1) / NM : 0;
      static_for<d1 - d0>([&](auto i_c) { issue(std::integral_constant<int, d0 + decltype(i_c)::value>{}, kt + NS, slot); });
      __builtin_amdgcn_sched_barrier(0);
    });
    slot = next;
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

  const int fw = f0 + wp * FW;
  float bg[TG][4], bu[TG][4];
#pragma unroll
  for (int a = 0; a < TG; a++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int f = min(fw + 16 * a + 4 * grp + e, p.features - 1);
      bg[a][e] = p.bias ? E::dec(((const raw *)p.bias)[f]) : 0.0f;
      bu[a][e] = p.bias ? E::dec(((const raw *)p.bias)[p.features + f]) : 0.0f;
    }
  gated_with(p, [&](auto kept, auto act) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < TQ; b++) {
      float g[TG][4], u[TG][4];
#pragma unroll
      for (int a = 0; a < TG; a++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          g[a][e] = acc[a][b][e] + bg[a][e];
          u[a][e] = acc[a + TG][b][e] + bu[a][e];
        }
      const int token = t0 + wq * (16 * TQ) + 16 * b + r16;
      gated_store<E, decltype(kept)::value, decltype(act)::value>(p, fw, token, token < p.tokens, g, u);
    }
  });
}

} // namespace zluda_amd
