// Products grouped by expert (include/zluda_ffn.h): which rows a workgroup has, and the kernel for operands at any alignment, pitch and size.
//
// The rows of an expert are known on the device only.  Tiles of rows are counted expert after expert, and a grid has room for the most there can be:
// one for each whole tile and one for each expert.  A workgroup finds its tile with a scan over the experts' counts, 64 of them at a time.
#pragma once
#include "ffn_common.hpp"

namespace zluda_amd {

// the rows of an expert, clamped to the matrices whatever `offsets` holds
__device__ __forceinline__ int expert_rows(const int32_t *offsets, int experts, int rows, int e, int &first) {
  first = 0;
  if (e >= experts) return 0;
  first = min(max(offsets[e], 0), rows);
  return max(min(max(offsets[e + 1], 0), rows) - first, 0);
}

struct RowTile {
  int e;          // -1: there is no such tile
  int first, n;   // the expert's rows
  int at;         // the tile's first one among them
};
// Sums of tile counts stop here: what `offsets` should not hold overflows nothing.  (A grid has fewer tiles.)
constexpr int kMostTiles = 1 << 30;
// Tile `slot` of `side` rows; every wave finds it for itself (all lanes active)
__device__ __forceinline__ RowTile find_row_tile(const int32_t *offsets, int experts, int rows, int side, int slot) {
  RowTile r{-1, 0, 0, 0};
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base < experts; base += 64) {
    int first;
    const int n = expert_rows(offsets, experts, rows, base + lane, first), tiles = (int)(((uint32_t)n + side - 1) / (uint32_t)side);
    int up_to = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int t = __shfl_up(up_to, d, 64);
      if (lane >= d) up_to = min(up_to + t, kMostTiles);
    }
    const uint64_t past = __ballot(before + up_to > slot);
    if (past) {
      const int l = __builtin_ctzll(past);
      r.e = base + l;
      r.first = __builtin_amdgcn_readlane(first, l);
      r.n = __builtin_amdgcn_readlane(n, l);
      r.at = (slot - before - (__builtin_amdgcn_readlane(up_to, l) - __builtin_amdgcn_readlane(tiles, l))) * side;
      return r;
    }
    before = min(before + __builtin_amdgcn_readlane(up_to, 63), kMostTiles);
  }
  return r;
}

// How many tiles of `side` rows there are, up to `most` of them
__device__ __forceinline__ int count_row_tiles(const int32_t *offsets, int experts, int rows, int side, int most) {
  int all = 0;
  for (int base = 0; base < experts; base += 64) {
    int first;
    all = min(all + (int)(((uint32_t)expert_rows(offsets, experts, rows, base + (threadIdx.x & 63), first) + side - 1) / (uint32_t)side), most);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) all = min(all + __shfl_xor(all, d, 64), most);
  return __builtin_amdgcn_readfirstlane(all);
}

struct GroupedParams {
  const int32_t *offsets;
  const void *a, *b;          // forward: x, w; dx: dy, w; dw: dy, x
  void *d;
  const float *a_scales, *b_scales;  // of packed operands
  int64_t lda, ldb, ldd, lda_scales, ldb_scales;
  int32_t rows, experts, features, model;
  uint32_t type, d_type;      // of the operands, of d
};

// Any alignment, pitch and size: 64 x 64 tiles of D, 4 x 4 values a thread, 16 of K at a time.  MODE 0: y, 1: dx, 2: dw.
// Bound by the arithmetic of its vector units.
template <int MODE>
__global__ __launch_bounds__(256) void grouped_any_kernel(GroupedParams p) {
  constexpr int S = 64, K = 16;
  __shared__ float as[K][S + 1], bs[K][S + 1];
  const int t = threadIdx.x, ti = (t & 15) * 4, tj = (t >> 4) * 4;
  const bool packed = MODE == 0 && p.type == CUDA_R_8F_E4M3;
  const int j0 = blockIdx.x * S, cols = MODE == 0 ? p.features : p.model;
  const int slots = MODE == 2 ? 1 : (int)((p.rows + S - 1) / S + min(p.experts, p.rows));
  for (int slot = MODE == 2 ? 0 : (int)blockIdx.y; slot < slots; slot += MODE == 2 ? 1 : (int)gridDim.y) {
    RowTile g{0, 0, 0, 0};
    if constexpr (MODE == 2) {
      g.e = blockIdx.z;
      g.n = expert_rows(p.offsets, p.experts, p.rows, g.e, g.first);
    } else {
      g = find_row_tile(p.offsets, p.experts, p.rows, S, slot);
      if (g.e < 0) return;
    }
    const int i0 = MODE == 2 ? blockIdx.y * S : g.at, d_rows = MODE == 2 ? p.features : g.n, kn = MODE == 0 ? p.model : MODE == 1 ? p.features : g.n;
    const int64_t w0 = (int64_t)g.e * p.features;
    auto a_at = [&](int i, int k) -> float {
      if constexpr (MODE == 2) return load_elem(p.a, p.type, (int64_t)(g.first + k) * p.lda + i);
      else {
        const float v = load_elem(p.a, p.type, (int64_t)(g.first + i) * p.lda + k);
        return packed ? v * p.a_scales[(int64_t)(k >> 7) * p.lda_scales + g.first + i] : v;
      }
    };
    auto b_at = [&](int k, int j) -> float {
      if constexpr (MODE == 0) {
        const float v = load_elem(p.b, p.type, (w0 + j) * p.ldb + k);
        return packed ? v * p.b_scales[((int64_t)g.e * ((p.features + 127) >> 7) + (j >> 7)) * p.ldb_scales + (k >> 7)] : v;
      } else if constexpr (MODE == 1) {
        return load_elem(p.b, p.type, (w0 + k) * p.ldb + j);
      } else {
        return load_elem(p.b, p.type, (int64_t)(g.first + k) * p.ldb + j);
      }
    };
    float acc[4][4];
#pragma unroll
    for (int a = 0; a < 4; a++)
#pragma unroll
      for (int b = 0; b < 4; b++) acc[a][b] = 0.0f;
    for (int k0 = 0; k0 < kn; k0 += K) {
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int e = t + 256 * r;
        const int ka = MODE == 2 ? e >> 6 : e & 15, ia = MODE == 2 ? e & 63 : e >> 4;  // neighbouring threads along the unit stride
        as[ka][ia] = i0 + ia < d_rows && k0 + ka < kn ? a_at(i0 + ia, k0 + ka) : 0.0f;
        const int kb = MODE != 0 ? e >> 6 : e & 15, jb = MODE != 0 ? e & 63 : e >> 4;
        bs[kb][jb] = j0 + jb < cols && k0 + kb < kn ? b_at(k0 + kb, j0 + jb) : 0.0f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; k++) {
        float av[4], bv[4];
#pragma unroll
        for (int a = 0; a < 4; a++) av[a] = as[k][tj + a];
#pragma unroll
        for (int b = 0; b < 4; b++) bv[b] = bs[k][ti + b];
#pragma unroll
        for (int a = 0; a < 4; a++)
#pragma unroll
          for (int b = 0; b < 4; b++) acc[a][b] = __builtin_fmaf(av[a], bv[b], acc[a][b]);
      }
      __syncthreads();
    }
#pragma unroll
    for (int a = 0; a < 4; a++)
#pragma unroll
      for (int b = 0; b < 4; b++) {
        const int i = i0 + tj + a, j = j0 + ti + b;
        if (i < d_rows && j < cols) store_elem(p.d, p.d_type, (MODE == 2 ? w0 + i : (int64_t)g.first + i) * p.ldd + j, acc[a][b]);
      }
  }
}

} // namespace zluda_amd
