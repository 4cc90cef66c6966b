// The two matrix products behind the gated layer's backward pass in one launch, in tiles of 128 x 128:
//   dX^T [model][token] = sum over 2 features of W[f][model] dZ[token][f],   dW^T [model][f] = sum over tokens of X[token][model] dZ[token][f].
// Both have 2 x tokens x 2 features x model operations and neither needs the other.  Launched one after the other each leaves a part of the chip idle
// while its last tiles run, and dX, with few tiles of a long K, all the time; together they fill each other's gaps.  (The last sums of the bias gradient ride along.)
//
// One operand (P: W or X) lies along its row index `model`, the other (Q: dZ) along K for dX and along its row index for dW.  Stages of 64 K
// elements travel straight into two slots of LDS; what lies along its row index is transposed by the LDS reads (ds_read_b64_tr_b16).  The layouts
// are those of gemm_mfma_pipe16.hpp: blocks of 1 KiB at a pitch of 1056 bytes, or eight swizzled chunks a row.  A stage is two halves along K; the
// fragments of the one arrive while the products of the other run.  The barrier lies between them: behind it stage kt + 1 has landed and every
// wave has the fragments of stage kt, whose slot takes stage kt + 2.  Two workgroups share a CU, and one computes while the other waits.
//
// Bound by the matrix cores and LDS where there are many tiles (8192 tokens, 2048 x 8192: 1040 us, 1.06 PFLOP/s; that is where tiles of 256 x 256, one
// product after the other, take 810), by the round trips of a stage's requests and the last tiles where there are few (1001 tokens, 1024 x 2816:
// 34 us, MFMAs 42 % of the time).  Tiles of 256 x 256 here, eight waves, have no registers left for the offsets of dZ's rows: 700 tokens, 4096 x 14336 381 us
// at best against 383, 1500, 2048 x 8192 235 against 229.
//
// K rows past the end are requested out of the buffer windows' range and become zeros; every wait is for everything in flight, so that it does not
// matter in which order such requests retire.  (Whole stages past the end requested like that cost 7 % at three stages, 150 tokens.)
#pragma once
#include "../ffn_launchers.hpp"
#include "ffn_gated_any.hpp"
#include "gemm_mfma_pipe16.hpp"

namespace zluda_amd {

constexpr int kGradSlot = 2 * (kGradTile / 8 * (kMcPitch / 16));  // 16-byte words of a stage, the larger form

template <class E, bool QMC>
__device__ __forceinline__ void grad_product_tile(const GradProduct &g, uint32_t id, v4i *lds) {
  constexpr int B = kGradTile, WP = 2, WQ = 2, NW = WP * WQ, TP = B / WP / 16, TQ = B / WQ / 16;
  constexpr int SLOT = kGradSlot, Q_AT = SLOT / 2;  // Q in a slot
  constexpr int PASS = 8 * NW;                      // rows along K that an instruction of all waves fills
  static_assert(B / 2 == 16 * NW && B / PASS == 4, "four instructions an operand and stage");
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wp = wave % WP, wq = wave / WP, r16 = lane & 15, g4 = lane >> 4;
  MfmaParams at;
  at.tiles_p = g.tiles_p; at.tiles_q = g.tiles_q; at.g.batch = 1; at.splits = g.splits; at.group_p = 8;
  const WorkItem item = work_item(at, id);
  const int p0 = item.p * B, q0 = item.q * B;
  const int k0 = item.z * g.split_stages * kGradStage, k_local = min(g.k - k0, g.split_stages * kGradStage);
  const int stages = (k_local + kGradStage - 1) / kGradStage;

  // ---- DMA: a wave instruction fills 1 KiB; wave w the blocks w, w + NW, .. ----------------------------------------------------------
  const v4i rp = {(int)(uintptr_t)g.p, (int)((uintptr_t)g.p >> 32) & 0xffff, (int)0x80000000, 0x00020000};
  const v4i rq = {(int)(uintptr_t)g.q, (int)((uintptr_t)g.q >> 32) & 0xffff, (int)0x80000000, 0x00020000};
  const int mk = mc_block_k(wave) + mc_lane_k(B, lane);  // the lane's K row in the wave's first block
  const int drow = wave * 8 + (lane >> 3), dchunk = ((lane & 7) ^ swz_mixed(drow)) * 16;
  // (a piece of eight past the end of the row index loads the last one: what it becomes is not stored)
  const int op = (mk * g.ldp + min(p0 + 8 * (lane & (B / 8 - 1)), g.np - 8)) * 2;
  int oq[QMC ? 1 : 4];
  if constexpr (QMC) {
    oq[0] = (mk * g.ldq + min(q0 + 8 * (lane & (B / 8 - 1)), g.nq - 8)) * 2;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) oq[i] = min(q0 + drow + PASS * i, g.nq - 1) * g.ldq * 2 + dchunk;
  }
  auto issue = [&](auto i_c, int kt, int slot) __attribute__((always_inline)) {  // instruction i of a stage: four of P, four of Q
    constexpr int i = decltype(i_c)::value & 3;
    constexpr bool of_p = decltype(i_c)::value < 4, rows = of_p || QMC;
    const int left = k_local - kt * kGradStage;  // K rows from the stage's first on
    v4i *base = lds + slot * SLOT + (of_p ? 0 : Q_AT);
    if constexpr (rows) {
      const int ld = of_p ? g.ldp : g.ldq, vo = mk + mc_block_k(NW * i) < left ? (of_p ? op : oq[0]) : (int)0x80000000;
      lds_dma16_uncounted(of_p ? rp : rq, base + (wave + NW * i) * (kMcPitch / 16), vo, (k0 + kt * kGradStage + mc_block_k(NW * i)) * ld * 2);
    } else {
      lds_dma16_uncounted(rq, base + (wave * 8 + PASS * i) * 8, dchunk < left * 2 ? oq[i] : (int)0x80000000, (k0 + kt * kGradStage) * 2);
    }
  };

  // ---- fragments: tiles of 16 rows of either operand, two halves of the stage's K ----------------------------------------------
  const int fp = mc_frag_at(B, g4, r16 >> 2) + 8 * (r16 & 3) + wp * TP * 32;
  const int fq = mc_frag_at(B, g4, r16 >> 2) + 8 * (r16 & 3) + wq * TQ * 32 + Q_AT * 16;
  int fk[2][2];  // dZ along K: [tile parity][half]
  if constexpr (!QMC) {
#pragma unroll
    for (int par = 0; par < 2; par++)
#pragma unroll
      for (int h = 0; h < 2; h++) fk[par][h] = Q_AT + (wq * TQ * 16 + 16 * par + r16) * 8 + ((4 * h + g4) ^ swz_mixed(16 * par + r16));
  }
  ffn_u4 fr[2][TP + TQ];  // [half][P tiles, Q tiles]
  auto read = [&](auto i_c, auto h_c, int slot) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value, tile = i < TP ? i : i - TP, h = decltype(h_c)::value;
    if constexpr (i < TP || QMC) {
      const char *base = (const char *)(lds + slot * SLOT) + (i < TP ? fp : fq) + tile * 32 + h * 512;
      const v2i lo = lds_read_tr16(base), hi = lds_read_tr16(base + 2 * B);
      fr[h][i] = __builtin_bit_cast(ffn_u4, v4i{lo[0], lo[1], hi[0], hi[1]});
    } else {
      fr[h][i] = __builtin_bit_cast(ffn_u4, lds[slot * SLOT + fk[tile & 1][h] + (tile >> 1) * 256]);
    }
  };
  v4f acc[TP][TQ];
#pragma unroll
  for (int a = 0; a < TP; a++)
#pragma unroll
    for (int b = 0; b < TQ; b++) acc[a][b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  static_for<8>([&](auto i_c) { issue(i_c, 0, 0); });
  if (stages > 1) static_for<8>([&](auto i_c) { issue(i_c, 1, 1); });
  wait_vmcnt_barrier<0>();
  using C0 = std::integral_constant<int, 0>;
  using C1 = std::integral_constant<int, 1>;
  static_for<TP + TQ>([&](auto i_c) { read(i_c, C0{}, 0); });
  // the products of half `h`, behind them the fragments of the other half from `slot` and, where `more`, the requests for stage `kt`
  auto half = [&](auto h_c, int slot, auto more_c, int kt) __attribute__((always_inline)) {
    constexpr int h = decltype(h_c)::value;
    static_for<TP * TQ>([&](auto x_c) {
      constexpr int x = decltype(x_c)::value, a = x / TQ, b = x % TQ;
      ffn_mfma<E>(fr[h][a], fr[h][TP + b], acc[a][b]);
      if constexpr (x < TP + TQ) read(x_c, std::integral_constant<int, 1 - h>{}, slot);
      if constexpr (decltype(more_c)::value != 0 && x < 8) issue(x_c, kt, 1 - slot);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // `inside`: stage kt + 2 exists
  auto do_stage = [&](auto slot_c, auto inside_c, int kt) __attribute__((always_inline)) {
    constexpr int slot = decltype(slot_c)::value;
    half(C0{}, slot, C0{}, 0);
    wait_vmcnt_barrier<0>();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (decltype(inside_c)::value == 0) {
      if (kt + 2 < stages) static_for<8>([&](auto i_c) { issue(i_c, kt + 2, slot); });
    }
    half(C1{}, 1 - slot, inside_c, kt + 2);
  };
  int kt = 0;
  for (; kt + 4 <= stages; kt += 2) {
    do_stage(C0{}, C1{}, kt);
    do_stage(C1{}, C1{}, kt + 1);
  }
  // one to three are left (what is read behind the last one is not used)
  if (kt < stages) {
    do_stage(C0{}, C0{}, kt);
    if (kt + 1 < stages) {
      do_stage(C1{}, C0{}, kt + 1);
      if (kt + 2 < stages) do_stage(C0{}, C0{}, kt + 2);
    }
  }

  // ---- D: a lane has P rows 4 g4 .. + 3 of a tile, column r16 ----------------------------------------------------------------------------
  const int pc = p0 + wp * TP * 16, qc = q0 + wq * TQ * 16;
  if (g.splits > 1) {
    const int64_t pitch = (int64_t)g.tiles_p * B, plane = pitch * g.tiles_q * B;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)(g.part + item.z * plane + qc * pitch + pc), 0, 0xFFFFFFFF, 0x00020000);
    const int vo = (r16 * (int)pitch + 4 * g4) * 4;
#pragma unroll
    for (int a = 0; a < TP; a++)
#pragma unroll
      for (int b = 0; b < TQ; b++) buffer_store_b128_guarded(__builtin_bit_cast(v4i, acc[a][b]), rs, vo, (b * 16 * (int)pitch + a * 16) * 4);
    return;
  }
  const int64_t corner = qc * g.ldd + pc;
  const __amdgpu_buffer_rsrc_t rs =
      __builtin_amdgcn_make_buffer_rsrc((void *)((typename E::raw *)g.d + corner), 0, tile_window_bytes(g.ldd, g.np, g.nq, corner, 2), 0x00020000);
  const int first = (g4 & 1) ? 4 * g4 + 12 : 4 * g4;  // pairs of tiles trade halves: eight rows, 16 bytes a lane
  const int vo = (r16 * (int)g.ldd + first) * 2;
#pragma unroll
  for (int a = 0; a < TP; a += 2)
#pragma unroll
    for (int b = 0; b < TQ; b++) {
      const v4f lo = acc[a][b], hi = acc[a + 1][b];
      const uint32_t l0 = E::pack2(lo[0], lo[1]), l1 = E::pack2(lo[2], lo[3]), h0 = E::pack2(hi[0], hi[1]), h1 = E::pack2(hi[2], hi[3]);
      v4i out = {(int)l0, (int)l1, (int)h0, (int)h1};
#if defined(__HIP_DEVICE_COMPILE__)
      const v2u s0 = __builtin_amdgcn_permlane16_swap(l0, h0, false, false), s1 = __builtin_amdgcn_permlane16_swap(l1, h1, false, false);
      out = v4i{(int)s0[0], (int)s1[0], (int)s0[1], (int)s1[1]};
#endif
      buffer_store_b128_guarded(out, rs, pc + a * 16 + first < g.np ? vo : kStoreNowhere, (b * 16 * (int)g.ldd + a * 16) * 2);
    }
}

// 64 columns of the bias gradient: every fourth row to a wave, then the four sums in order.  (A launch of its own for it takes 4 us.)
template <class E>
__device__ __forceinline__ void grad_bias_sums(const GradProductsParams &p, int strip, float *lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = strip * 64 + lane, cols = p.dw.nq;
  float sum = 0.0f;
  if (col < cols) {
    const float *from = p.sums + col;
#pragma unroll 8
    for (int z = wave; z < p.shares; z += 4) sum += from[(int64_t)z * cols];
  }
  lds[threadIdx.x] = sum;
  __syncthreads();
  if (wave == 0 && col < cols) ((typename E::raw *)p.dbias)[col] = E::enc(((lds[lane] + lds[lane + 64]) + lds[lane + 128]) + lds[lane + 192]);
}

template <class E>
__global__ __launch_bounds__(256, 2) void grad_products_kernel(GradProductsParams prm) {
  __shared__ v4i lds[2 * kGradSlot];
  const uint32_t dw_groups = (uint32_t)(prm.dw.tiles_p * prm.dw.tiles_q), id = blockIdx.x - prm.dx_groups;
  if (blockIdx.x < prm.dx_groups) grad_product_tile<E, false>(prm.dx, blockIdx.x, lds);
  else if (id < dw_groups) grad_product_tile<E, true>(prm.dw, id, lds);
  else grad_bias_sums<E>(prm, (int)(id - dw_groups), (float *)lds);
}

} // namespace zluda_amd
