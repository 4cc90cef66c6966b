// The products of block_gemm.hpp for a few tokens and matrices whose reading takes no longer than a launch: one kernel, where tiles that share K out over
// workgroups need a second one.
//
// Eight waves share K out, 128 of it at a time, over 16 rows of P, and join their sums in LDS in a fixed order.  A lane loads its fragments straight into registers,
// four blocks ahead: with no ring to fill and no barrier before the end, a short K is a single round trip to memory, which is what bounds it.  2048 x 2048, one
// token: 5.3 us in a graph (an empty launch takes 3.5), 6.3 on 64 x 32 tiles and their second kernel.  Long K and large matrices are left to those: such loads
// reach 3.3 TB/s (14336 x 4096, 17.5 us), tiles through LDS 5.2.
#pragma once
#include "block_gemm.hpp"

namespace zluda_amd {

template <int FP, int FQ, bool SU, bool EXACT>
__global__ __launch_bounds__(512, 4) void block_decode_kernel(MfmaParams prm) {
  constexpr int NW = 8, AHEAD = EXACT ? 3 : 4;
  __shared__ float sums[NW][64][4];
  fetch_args(prm);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, grp = lane >> 4;
  const WorkItem item = work_item(prm);
  const int p0 = item.p * 16, q0 = item.q * 16;
  TileSide P, Q;
  block_sides(prm, p0, q0, item.bt, P, Q);
  const int K = prm.g.K, blocks = (K + 127) / 128;
  const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc((void *)P.data, 0, 0x80000000, 0x00020000);
  const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void *)Q.data, 0, 0x80000000, 0x00020000);
  const __amdgpu_buffer_rsrc_t rsp = __builtin_amdgcn_make_buffer_rsrc((void *)P.scales, 0, 0x80000000, 0x00020000);
  const __amdgpu_buffer_rsrc_t rsq = __builtin_amdgcn_make_buffer_rsrc((void *)Q.scales, 0, 0x80000000, 0x00020000);
  // (rows past the end are out of the windows too.  Which of a block's 128 a lane has matters only in that it is the same of P and of Q: 16 and 16 that its
  // neighbours carry on, so that an instruction reads 64 bytes of each row)
  constexpr int kOut = (int)0x80000000;
  const int op = r16 < P.rows ? r16 * P.ld + 16 * grp : kOut, oq = r16 < Q.rows ? r16 * Q.ld + 16 * grp : kOut;
  const int osq = r16 >= Q.rows ? kOut : Q.per_row ? r16 * Q.s_row * 4 : 0;  // (16 rows lie in one block of 128)
  int osp[SU ? 1 : 4];
#pragma unroll
  for (int e = 0; e < (SU ? 1 : 4); e++) osp[e] = 4 * grp + e >= P.rows ? kOut : P.per_row ? (4 * grp + e) * P.s_row * 4 : 0;

  v4i pf[AHEAD][2], qf[AHEAD][2];
  float sp[AHEAD][SU ? 1 : 4], sq[AHEAD];
  // the wave's block i, what lies past the end of K or past the last block as zeros: out of the windows, no traffic
  auto load = [&](auto j_c, int i) __attribute__((always_inline)) {
    constexpr int j = decltype(j_c)::value;
    const int blk = wave + NW * i, at = blk * 128, none = blk < blocks ? 0 : kOut, s_blk = min(blk, blocks - 1);  // (uniform offsets stay within the windows)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int oob = at + 16 * grp + 64 * h < K ? 0 : kOut;
      pf[j][h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rp, (op + 64 * h) | oob, at, 0));
      qf[j][h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rq, (oq + 64 * h) | oob, at, 0));
    }
#pragma unroll
    for (int e = 0; e < (SU ? 1 : 4); e++) sp[j][e] = bits2f(__builtin_amdgcn_raw_buffer_load_b32(rsp, osp[e] | none, s_blk * P.s_step * 4, 0));
    sq[j] = bits2f(__builtin_amdgcn_raw_buffer_load_b32(rsq, osq | none, s_blk * Q.s_step * 4, 0));
  };
  v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
  static_for<AHEAD>([&](auto j_c) { load(j_c, decltype(j_c)::value); });
  for (int i0 = 0; wave + NW * i0 < blocks; i0 += AHEAD) {
    static_for<AHEAD>([&](auto j_c) {
      constexpr int j = decltype(j_c)::value;
      v4f t = {0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (EXACT) {
        v8b wp[4], wq[4];
        block_widen<FP>(pf[j], wp);
        block_widen<FQ>(qf[j], wq);
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int s4 = 0; s4 < 4; s4++) t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wp[s4], wq[s4], t, 0, 0, 0);
#endif
      } else {
        t = block_mfma<KIND_F8, FP, FQ>(pf[j], qf[j], 0, t);
      }
#pragma unroll
      for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(t[e], sp[j][SU ? 0 : e] * sq[j], acc[e]);
      __builtin_amdgcn_sched_barrier(0);
      load(j_c, i0 + AHEAD + j);
      __builtin_amdgcn_sched_barrier(0);
    });
  }
  *(v4f *)sums[wave][lane] = acc;
  __syncthreads();
  const int row = threadIdx.x & 15, col = threadIdx.x >> 4;
  if (col >= 16 || row >= P.rows || col >= Q.rows) return;
  float v = 0.0f;
#pragma unroll
  for (int w = 0; w < NW; w++) v += sums[w][(row >> 2) * 16 + col][row & 3];
  Epilogue ep(prm.g, item.bt);
  ep.store_f(prm.swapped ? q0 + col : p0 + row, prm.swapped ? p0 + row : q0 + col, v);
}

} // namespace zluda_amd
