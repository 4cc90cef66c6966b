// The gradients of products grouped by expert, both in one launch:
//   dX^T [model][row] = sum over features of W_e[feature][model] dY[row][feature],   dW_e^T [model][feature] = sum over the expert's rows of X[row][model] dY[row][feature].
// One operand (P: W_e or X) lies along its row index, the other (Q: dY) along K for dX and along its row index for dW, as in ffn_grad_products.hpp, whose 128 x 128
// tiles and LDS layouts these are; and tiles of 256 x 256 on eight waves of 128 x 64, with the sub-steps of WideTile (block_tile.hpp).
#pragma once
#include "ffn_elementwise.hpp"
#include "ffn_grouped_tile.hpp"

namespace zluda_amd {

struct GroupedGradParams {
  const int32_t *offsets;
  const void *dy, *x, *w;
  void *dx, *dw;                 // or NULL
  int64_t lddx, lddw;
  int32_t lddy, ldx, ldw;
  int32_t rows, experts, features, model;
  uint32_t dx_groups;            // workgroups of dx, the first ones
  // tiles of 128 x 128 may share out dx's K: share z of a row leaves its sums in part[z][row], whole tiles of model wide
  float *part;
  int32_t dx_splits, dx_split_stages;
};

// The 256 x 256 tile whose first row and column are p0 and q0.  LDS: P's two slots, Q's two, in blocks of 1 KiB at a pitch of 1056 bytes or (Q along K) eight swizzled
// chunks a row.  All waits are for everything in flight; K rows, and rows of Q along K, past the end are out of the windows' range and become zeros.
template <class E, bool QMC>
__device__ __forceinline__ void grouped_grad_wide(const GradProduct &g, int p0, int q0, v4i *lds) {
  constexpr int B = 256, WP = 2, NW = 8, TP = 8, TQ = 4, SLOT = B / 8 * (kMcPitch / 16), Q_AT = 2 * SLOT, QSLOT = QMC ? SLOT : B * 8;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wp = wave % WP, wq = wave / WP, r16 = lane & 15, g4 = lane >> 4;
  const int stages = (g.k + kGradStage - 1) / kGradStage;
  const char *const qrows = (const char *)g.q + (QMC ? 0 : (int64_t)q0 * g.ldq * 2);
  const int qbytes = QMC ? (int)0x80000000 : (int)min((int64_t)(min(g.nq - q0, B) - 1) * g.ldq * 2 + g.k * 2, (int64_t)0x7fffffff);
  const v4i rp = {(int)(uintptr_t)g.p, (int)((uintptr_t)g.p >> 32) & 0xffff, (int)0x80000000, 0x00020000};
  const v4i rq = {(int)(uintptr_t)qrows, (int)((uintptr_t)qrows >> 32) & 0xffff, qbytes, 0x00020000};
  const int mk = mc_block_k(wave) + mc_lane_k(B, lane);  // the lane's K row in the wave's first block
  const int drow = wave * 8 + (lane >> 3), dchunk = ((lane & 7) ^ swz_mixed(drow)) * 16;
  // (a piece of eight past the end of the row index loads the last one: what it becomes is not stored)
  const int op = (mk * g.ldp + min(p0 + 8 * (lane & 31), g.np - 8)) * 2;
  const int oq = QMC ? (mk * g.ldq + min(q0 + 8 * (lane & 31), g.nq - 8)) * 2 : drow * g.ldq * 2 + dchunk;
  auto issue = [&](auto i_c, int kt, int slot) __attribute__((always_inline)) {  // instruction i of a stage: four of P, four of Q
    constexpr int i = decltype(i_c)::value & 3;
    constexpr bool of_p = decltype(i_c)::value < 4;
    const int left = g.k - kt * kGradStage;  // K rows from the stage's first on
    if constexpr (of_p || QMC) {
      const int ld = of_p ? g.ldp : g.ldq, vo = mk + mc_block_k(NW * i) < left ? (of_p ? op : oq) : (int)0x80000000;
      lds_dma16_uncounted(of_p ? rp : rq, lds + (of_p ? slot * SLOT : Q_AT + slot * QSLOT) + (wave + NW * i) * (kMcPitch / 16), vo, (kt * kGradStage + mc_block_k(NW * i)) * ld * 2);
    } else {
      lds_dma16_uncounted(rq, lds + Q_AT + slot * QSLOT + (wave * 8 + 64 * i) * 8, dchunk < left * 2 ? oq : (int)0x80000000, kt * kGradStage * 2 + 64 * i * g.ldq * 2);
    }
  };
  v4f acc[TP][TQ];
#pragma unroll
  for (int a = 0; a < TP; a++)
#pragma unroll
    for (int b = 0; b < TQ; b++) acc[a][b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  static_for<8>([&](auto i_c) { issue(i_c, 0, 0); });
  static_for<8>([&](auto i_c) { issue(i_c, 1, 1); });
  wait_vmcnt_barrier<0>();
  if (wp * 128 >= g.np - p0 || wq * 64 >= g.nq - q0) {  // nothing of the wave's own: as in WideTile
    for (int kt = 0; kt < stages; kt++) {
      wait_vmcnt_barrier<0>();
      static_for<8>([&](auto i_c) { issue(i_c, kt + 2, kt & 1); });
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    return;
  }
  // ---- fragments: [half of the wave tile][tile][half of the stage's K] ----------------------------------------------------------------
  const char *const fp = (const char *)lds + mc_frag_at(B, g4, r16 >> 2) + 8 * (r16 & 3) + wp * 256;
  const char *const fq = (const char *)(lds + Q_AT) + mc_frag_at(B, g4, r16 >> 2) + 8 * (r16 & 3) + wq * 128;
  int fk[2];
#pragma unroll
  for (int h = 0; h < 2; h++) fk[h] = Q_AT + (wq * 64 + r16) * 8 + ((4 * h + g4) ^ swz_mixed(r16));
  v4i pf[2][4][2], qf[2][2][2];
  auto mc_read = [&](const char *from) __attribute__((always_inline)) {
    const v2i lo = lds_read_tr16(from), hi = lds_read_tr16(from + 2 * B);
    return v4i{lo[0], lo[1], hi[0], hi[1]};
  };
  auto read_p = [&](auto h_c, auto r_c, int slot) __attribute__((always_inline)) {
    constexpr int h = decltype(h_c)::value, r = decltype(r_c)::value, tile = h * 4 + r % 4, ks = r / 4;
    pf[h][r % 4][ks] = mc_read(fp + slot * SLOT * 16 + tile * 32 + ks * 16 * kMcPitch);
  };
  auto read_q = [&](auto h_c, auto r_c, int slot) __attribute__((always_inline)) {
    constexpr int h = decltype(h_c)::value, r = decltype(r_c)::value, tile = h * 2 + r % 2, ks = r / 2;
    if constexpr (QMC) qf[h][r % 2][ks] = mc_read(fq + slot * QSLOT * 16 + tile * 32 + ks * 16 * kMcPitch);
    else qf[h][r % 2][ks] = lds[slot * QSLOT + fk[ks] + tile * 128];
  };
  using C0 = std::integral_constant<int, 0>;
  using C1 = std::integral_constant<int, 1>;
  static_for<8>([&](auto r_c) { read_p(C0{}, r_c, 0); });
  static_for<4>([&](auto r_c) { read_q(C0{}, r_c, 0); });
  auto do_stage = [&](auto odd_c, int kt) __attribute__((always_inline)) {
    constexpr int ODD = decltype(odd_c)::value, slot = ODD, next = 1 - ODD;
    using QB = std::integral_constant<int, 1 - ODD>;
    auto substep = [&](auto sub_c, auto &&rd, auto nr_c, auto l0_c, auto l1_c) __attribute__((always_inline)) {
      constexpr int sub = decltype(sub_c)::value, ph = sub / 2, qh = sub == 0 || sub == 3 ? ODD : 1 - ODD, NM = 16;
      constexpr int NR = decltype(nr_c)::value, L0 = decltype(l0_c)::value, L1 = decltype(l1_c)::value;
      static_for<NM>([&](auto x_c) {
        constexpr int x = decltype(x_c)::value, i = x % 8 / 2, j = x % 2, ks = x / 8;
        v4f &c = acc[ph * 4 + i][qh * 2 + j];
        ffn_mfma<E>(__builtin_bit_cast(ffn_u4, pf[ph][i][ks]), __builtin_bit_cast(ffn_u4, qf[qh][j][ks]), c);
        constexpr int r0 = NR * x / NM, r1 = NR * (x + 1) / NM;
        static_for<r1 - r0>([&](auto r_c) { rd(std::integral_constant<int, r0 + decltype(r_c)::value>{}); });
        constexpr int d0 = L0 + (L1 - L0) * x / NM, d1 = L0 + (L1 - L0) * (x + 1) / NM;
        static_for<d1 - d0>([&](auto i_c) { issue(std::integral_constant<int, d0 + decltype(i_c)::value>{}, kt + 2, slot); });
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    using N4 = std::integral_constant<int, 4>;
    using N8 = std::integral_constant<int, 8>;
    substep(C0{}, [&](auto r_c) { read_q(QB{}, r_c, slot); }, N4{}, C0{}, C0{});
    substep(C1{}, [&](auto r_c) { read_p(C1{}, r_c, slot); }, N8{}, C0{}, C0{});
    wait_vmcnt_barrier<0>();
    __builtin_amdgcn_sched_barrier(0);
    substep(std::integral_constant<int, 2>{}, [&](auto r_c) { read_p(C0{}, r_c, next); }, N8{}, C0{}, N4{});
    substep(std::integral_constant<int, 3>{}, [&](auto r_c) { read_q(QB{}, r_c, next); }, N4{}, N4{}, N8{});
  };
  for (int kt = 0; kt < stages; kt += 2) {
    do_stage(C0{}, kt);
    if (kt + 1 < stages) do_stage(C1{}, kt + 1);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // ---- D: a lane has P rows 4 g4 .. + 3 of a tile, column r16; pairs of tiles trade halves: eight rows, 16 bytes a lane ------------------------
  const int pc = p0 + wp * 128, qc = q0 + wq * 64;
  const int64_t corner = qc * g.ldd + pc;
  const __amdgpu_buffer_rsrc_t rs =
      __builtin_amdgcn_make_buffer_rsrc((void *)((typename E::raw *)g.d + corner), 0, tile_window_bytes(g.ldd, g.np, g.nq, corner, 2), 0x00020000);
  const int first = (g4 & 1) ? 4 * g4 + 12 : 4 * g4;
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

// B: 128 or 256, rows and columns of a tile
template <class E, int B>
__global__ __launch_bounds__(B == 256 ? 512 : 256, 2) void grouped_grad_kernel(GroupedGradParams p) {
  using raw = typename E::raw;
  __shared__ v4i lds[B == 256 ? 4 * (256 / 8) * (kMcPitch / 16) : 2 * kGradSlot];
  const int tiles_m = (p.model + B - 1) / B;
  GradProduct g;
  g.part = nullptr; g.splits = 1; g.np = p.model; g.tiles_p = tiles_m;
  if (blockIdx.x < p.dx_groups) {
    GroupedParams q;
    q.offsets = p.offsets; q.experts = p.experts; q.rows = p.rows;
    const uint32_t tiles = B == 256 ? p.dx_groups : p.dx_groups / (uint32_t)p.dx_splits, z = B == 256 ? 0 : blockIdx.x / tiles;
    const GroupedItem it = grouped_item(q, tiles_m, B, blockIdx.x - z * tiles, tiles);
    if (it.rows.e < 0) return;
    g.p = (const raw *)p.w + (int64_t)it.rows.e * p.features * p.ldw; g.ldp = p.ldw;
    g.q = (const raw *)p.dy + (int64_t)it.rows.first * p.lddy; g.ldq = p.lddy;
    g.d = (raw *)p.dx + it.rows.first * p.lddx; g.ldd = p.lddx;
    g.nq = it.rows.n; g.k = p.features; g.split_stages = (g.k + kGradStage - 1) / kGradStage;
    if constexpr (B == 256) {
      grouped_grad_wide<E, false>(g, it.p * B, it.rows.at, lds);
    } else {
      const int64_t pitch = (int64_t)tiles_m * B;
      g.splits = p.dx_splits; g.split_stages = p.dx_split_stages;
      g.part = p.part + it.rows.first * pitch; g.part_plane = p.rows * pitch; g.part_rows = g.nq;
      grad_product_at<E, false>(g, it.p * B, it.rows.at, (int)z, lds);
    }
    return;
  }
  MfmaParams at;
  at.tiles_p = tiles_m; at.tiles_q = (p.features + B - 1) / B; at.g.batch = p.experts; at.splits = 1; at.group_p = 8;
  const WorkItem item = work_item(at, blockIdx.x - p.dx_groups);
  int first;
  const int n = expert_rows(p.offsets, p.experts, p.rows, item.bt, first);
  g.p = (const raw *)p.x + (int64_t)first * p.ldx; g.ldp = p.ldx;
  g.q = (const raw *)p.dy + (int64_t)first * p.lddy; g.ldq = p.lddy;
  g.d = (raw *)p.dw + (int64_t)item.bt * p.features * p.lddw; g.ldd = p.lddw;
  g.nq = p.features; g.k = n; g.split_stages = (n + kGradStage - 1) / kGradStage;
  if constexpr (B == 256) grouped_grad_wide<E, true>(g, item.p * B, item.q * B, lds);
  else grad_product_at<E, true>(g, item.p * B, item.q * B, 0, lds);
}

// the shares of dx, of the rows that experts have
template <class E>
__global__ __launch_bounds__(256) void grouped_round_kernel(RoundParams p, const int32_t *offsets, int32_t experts) {
  round_rows<E>(p, min(max(offsets[0], 0), (int)p.rows), min(max(offsets[experts], 0), (int)p.rows));
}

} // namespace zluda_amd
