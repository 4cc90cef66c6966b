// The entry points of include/zluda_ffn.h: argument checks, kernel choice and launches.  The products of the gated layer's
// backward pass are matmuls of the launch layer (include/zluda_gemm_launch.h).
#include "../../include/zluda_ffn.h"

#include <algorithm>
#include <cstring>

#include "../../include/zluda_gemm_launch.h"
#include "ffn_launchers.hpp"
#include "kernels/ffn_elementwise.hpp"
#include "kernels/ffn_norm.hpp"
#include "planner.hpp"

using namespace zluda_amd;

namespace {

// Split-K partial tiles of the matmuls that make dX and dW one after the other, or one of them alone.  With twice as much the planner splits further than pays
// here, with half as much not far enough.  Whole backward passes, us, with 16, 32 and 8 MiB: dX alone, 1001 tokens, 1024 x 2816 30.8, 33.9, 34.9; 500, 4096 x
// 11008 108, 115, 164; dW alone, 8192, 1024 x 512 37.0, 40.5, 45.5; both, 8192, 1024 x 512 61.9, 64.3, 67.3; 1500, 1023 x 4000 98, 96, 122; 3000, 512 x 512 32.2, 32.2, 29.0.
constexpr uint64_t kGemmWorkspace = 16ull << 20;
constexpr int kGridY = 65535;

inline bool is_h16(uint32_t type) { return type == CUDA_R_16F || type == CUDA_R_16BF; }
inline uint64_t elem_size(uint32_t type) { return type == CUDA_R_32F ? 4 : type == CUDA_R_8F_E4M3 ? 1 : 2; }
inline uint64_t aligned256(uint64_t n) { return (n + 255) & ~255ull; }
inline int cus() {
  const int n = (int)zluda_gemm_device_cu_count();
  return n ? n : 256;
}

// a matrix that has to be there: rows x cols of `type`, or a checkpoint where `ckpt` allows one
uint32_t check_matrix(const zluda_ffn_matrix &m, uint64_t rows, uint64_t cols, uint32_t type, bool ckpt) {
  if (!m.data && rows) return CUBLAS_STATUS_INVALID_VALUE;
  if (m.type == CUDA_R_8F_E4M3) {
    if (!ckpt) return CUBLAS_STATUS_NOT_SUPPORTED;
    if ((!m.scales && rows) || m.ld < (int64_t)cols || m.ld % 32 || m.ld_scales < (int64_t)((cols + 31) / 32) || ((uintptr_t)m.data & 15))
      return CUBLAS_STATUS_INVALID_VALUE;
    return CUBLAS_STATUS_SUCCESS;
  }
  if (m.type != type) return CUBLAS_STATUS_NOT_SUPPORTED;
  if (m.ld < (int64_t)cols || ((uintptr_t)m.data & (elem_size(type) - 1))) return CUBLAS_STATUS_INVALID_VALUE;
  return CUBLAS_STATUS_SUCCESS;
}
#define FFN_CHECK(expr)                            \
  do {                                             \
    const uint32_t st_ = (expr);                   \
    if (st_ != CUBLAS_STATUS_SUCCESS) return st_;  \
  } while (0)

inline uint32_t check_vector(const void *v, uint32_t type) { return ((uintptr_t)v & (elem_size(type) - 1)) ? CUBLAS_STATUS_INVALID_VALUE : CUBLAS_STATUS_SUCCESS; }

// sizes of a gated layer; tokens may be 0
uint32_t check_sizes(uint32_t activation, uint64_t tokens, uint64_t features, uint64_t model) {
  if (activation > ZLUDA_FFN_RELU || !features || !model) return CUBLAS_STATUS_INVALID_VALUE;
  return tokens > kMaxSide || features > kMaxFeatures || model > kMaxSide ? CUBLAS_STATUS_NOT_SUPPORTED : CUBLAS_STATUS_SUCCESS;
}

uint32_t check_forward(const zluda_ffn_gated *p) {
  if (!p) return CUBLAS_STATUS_INVALID_VALUE;
  FFN_CHECK(check_sizes(p->activation, p->tokens, p->features, p->model));
  if (!is_h16(p->x.type)) return CUBLAS_STATUS_NOT_SUPPORTED;
  FFN_CHECK(check_matrix(p->x, p->tokens, p->model, p->x.type, false));
  FFN_CHECK(check_matrix(p->w, 2 * p->features, p->model, p->x.type, false));
  FFN_CHECK(check_matrix(p->h, p->tokens, p->features, p->x.type, false));
  FFN_CHECK(check_vector(p->bias, p->x.type));
  if (!p->gate.data != !p->up.data) return CUBLAS_STATUS_INVALID_VALUE;
  if (p->gate.data) {
    if (p->gate.type != p->up.type) return CUBLAS_STATUS_NOT_SUPPORTED;
    FFN_CHECK(check_matrix(p->gate, p->tokens, p->features, p->x.type, true));
    FFN_CHECK(check_matrix(p->up, p->tokens, p->features, p->x.type, true));
  }
  return CUBLAS_STATUS_SUCCESS;
}

// where the parts of the backward pass's workspace lie
struct GradPlan {
  uint64_t dz, x, sums, gemm, acc, total;  // offsets
  uint64_t dx_rows, dw_rows;               // tokens of a matmul
  int64_t lddz;
  uint32_t shares;                         // partial rows of dbias
  GradTogether together;
};

// Workgroups of gated_grad_kernel along the rows.  Without sums a row of its own for every thread (8192 x 8192: 112 us, 130 with eight
// workgroups a CU that walk the rows); with them at least four rows a thread and at most eight workgroups a CU, because each
// leaves a row of partial sums (1001 x 2816: 10.9 us, 15.4 with one row a thread).
uint32_t grad_shares(uint64_t tokens, uint64_t features, bool sums) {
  const uint64_t strips = column_strips(features), each = sums ? 16 : 4, most = std::max<uint64_t>(1, (tokens + each - 1) / each);
  const uint64_t want = sums ? std::max<uint64_t>(1, ((uint64_t)cus() * 8 + strips - 1) / strips) : most;
  return (uint32_t)std::min<uint64_t>({want, most, kGridY});
}

// Rows of the workspace's matrices start on cache lines (128 bytes): elsewhere each piece of a row that the matmuls fetch touches two
// (forward products, 603 tokens, 8608 features: model 3520 87 us, 3496 109).
int64_t aligned_pitch(uint64_t cols) { return (int64_t)((cols + 63) & ~63ull); }

GradPlan grad_plan(const zluda_ffn_gated_grad *p) {
  GradPlan g;
  memset(&g, 0, sizeof(g));
  uint64_t at = 0;
  g.lddz = p->dz.data ? p->dz.ld : aligned_pitch(2 * p->features);
  g.shares = grad_shares(p->tokens, p->features, p->dbias != nullptr);
  g.together = grad_together(p, cus());
  g.dz = at;
  if (!p->dz.data) at += aligned256(p->tokens * (uint64_t)g.lddz * 2);
  g.x = at;
  if (p->dw.data && p->x.type == CUDA_R_8F_E4M3) at += aligned256(p->tokens * (uint64_t)aligned_pitch(p->model) * 2);
  g.sums = at;
  if (p->dbias) at += aligned256((uint64_t)g.shares * 2 * p->features * 4);
  g.gemm = at;
  if (p->dx.data || p->dw.data) at += std::max<uint64_t>(kGemmWorkspace, g.together.part);
  // dW over several parts is summed in 32 bits and rounded once
  g.acc = at;
  g.dx_rows = rows_in_window(p->tokens, g.lddz);
  g.dw_rows = rows_in_window(p->tokens, std::max(g.lddz, p->x.type == CUDA_R_8F_E4M3 ? aligned_pitch(p->model) : p->x.ld));
  if (p->dw.data && g.dw_rows < p->tokens) at += aligned256(2 * p->features * (uint64_t)aligned_pitch(p->model) * 4);
  g.total = at;
  return g;
}

uint32_t check_backward(const zluda_ffn_gated_grad *p) {
  if (!p) return CUBLAS_STATUS_INVALID_VALUE;
  FFN_CHECK(check_sizes(p->activation, p->tokens, p->features, p->model));
  const uint32_t type = p->dh.type;
  if (!is_h16(type)) return CUBLAS_STATUS_NOT_SUPPORTED;
  FFN_CHECK(check_matrix(p->dh, p->tokens, p->features, type, false));
  if (p->gate.type != p->up.type) return CUBLAS_STATUS_NOT_SUPPORTED;
  FFN_CHECK(check_matrix(p->gate, p->tokens, p->features, type, true));
  FFN_CHECK(check_matrix(p->up, p->tokens, p->features, type, true));
  if (p->dx.data) {
    FFN_CHECK(check_matrix(p->dx, p->tokens, p->model, type, false));
    FFN_CHECK(check_matrix(p->w, 2 * p->features, p->model, type, false));
  }
  if (p->dw.data) {
    FFN_CHECK(check_matrix(p->dw, 2 * p->features, p->model, type, false));
    FFN_CHECK(check_matrix(p->x, p->tokens, p->model, type, true));
  }
  if (p->h.data) FFN_CHECK(check_matrix(p->h, p->tokens, p->features, type, false));
  if (p->dz.data) FFN_CHECK(check_matrix(p->dz, p->tokens, 2 * p->features, type, false));
  return check_vector(p->dbias, type);
}

template <class E>
uint32_t launch_checkpoint(bool store, const CheckpointParams &p, hipStream_t s) {
  const dim3 grid(column_strips(p.cols), (uint32_t)std::min<int64_t>((p.rows + 3) / 4, kGridY));
  return store ? launch_kernel(checkpoint_store_kernel<E>, grid, dim3(256), s, p) : launch_kernel(checkpoint_load_kernel<E>, grid, dim3(256), s, p);
}

uint32_t run_checkpoint(bool store, uint64_t rows, uint64_t cols, const zluda_ffn_matrix &x, const zluda_ffn_matrix &c, hipStream_t s) {
  CheckpointParams p{x.data, (uint8_t *)c.data, (uint8_t *)c.scales, (int64_t)rows, x.ld, c.ld, c.ld_scales, (int32_t)cols};
  switch (x.type) {
  case CUDA_R_16BF: return launch_checkpoint<ElemBF16>(store, p, s);
  case CUDA_R_16F: return launch_checkpoint<ElemF16>(store, p, s);
  default: return launch_checkpoint<ElemF32>(store, p, s);
  }
}

uint32_t checkpoint_call(bool store, uint64_t rows, uint64_t cols, const zluda_ffn_matrix *x, const zluda_ffn_matrix *c, void *stream) {
  if (!x || !c || !cols) return CUBLAS_STATUS_INVALID_VALUE;
  if (cols > kMaxSide || rows > (uint64_t)INT64_MAX / 2 || (!is_h16(x->type) && x->type != CUDA_R_32F) || c->type != CUDA_R_8F_E4M3) return CUBLAS_STATUS_NOT_SUPPORTED;
  FFN_CHECK(check_matrix(*x, rows, cols, x->type, false));
  FFN_CHECK(check_matrix(*c, rows, cols, x->type, true));
  if (!rows) return CUBLAS_STATUS_SUCCESS;
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  return run_checkpoint(store, rows, cols, *x, *c, (hipStream_t)stream);
}

template <class E, bool CK>
uint32_t launch_gated_grad(const GatedGradParams &g, uint32_t shares, hipStream_t s) {
  const dim3 grid(column_strips(g.features) + (g.load.x ? column_strips(g.load.cols) : 0), shares);
  switch (g.activation) {
  case ZLUDA_FFN_SILU: return launch_kernel(gated_grad_kernel<E, CK, 0>, grid, dim3(256), s, g);
  case ZLUDA_FFN_GELU: return launch_kernel(gated_grad_kernel<E, CK, 1>, grid, dim3(256), s, g);
  default: return launch_kernel(gated_grad_kernel<E, CK, 2>, grid, dim3(256), s, g);
  }
}

// D = op(A) op(B) + beta D of column-major matrices on the framework's matmul kernels: 16-bit A and B, D of `d_type`
uint32_t run_matmul(uint32_t type, uint32_t transa, uint32_t transb, uint64_t m, uint64_t n, uint64_t k, const void *A, int64_t lda, const void *B, int64_t ldb,
                    uint32_t d_type, float beta, void *D, int64_t ldd, void *ws, uint64_t ws_size, hipStream_t s) {
  const float one = 1.0f;
  zluda_gemm_problem q;
  memset(&q, 0, sizeof(q));
  q.op.compute_type = CUBLAS_COMPUTE_32F;
  q.op.scale_type = CUDA_R_32F;
  q.op.pointer_mode = CUBLASLT_POINTER_MODE_HOST;
  q.op.transa = transa; q.op.transb = transb;
  q.op.epilogue = CUBLASLT_EPILOGUE_DEFAULT;
  q.op.bias_type = -1;
  q.op.epilogue_aux_type = -1;
  q.a = {type, CUBLASLT_ORDER_COL, transa ? k : m, transa ? m : k, lda, 1, 0};
  q.b = {type, CUBLASLT_ORDER_COL, transb ? n : k, transb ? k : n, ldb, 1, 0};
  q.c = {d_type, CUBLASLT_ORDER_COL, m, n, ldd, 1, 0};
  q.d = q.c;
  q.alpha = &one; q.beta = &beta;
  q.A = A; q.B = B; q.C = D; q.D = D;
  q.workspace = ws; q.workspace_size = ws_size;
  zluda_gemm_plan plan;
  static_assert(kTrVariants[3].bp == 256 && kTrVariants[3].bq == 256, "the largest tile");
  const uint32_t cu = zluda_gemm_device_cu_count();
  uint32_t st = CUBLAS_STATUS_NOT_SUPPORTED;
  if (grad_largest_tiles(m, n, cu)) st = zluda_gemm_plan_problem(&q, ZLUDA_KERNEL_MFMA_TR16, 3, cu, &plan);
  if (st != CUBLAS_STATUS_SUCCESS) st = zluda_gemm_plan_problem(&q, ZLUDA_KERNEL_AUTO, -1, cu, &plan);
  if (st == CUBLAS_STATUS_SUCCESS) st = zluda_gemm_launch(&q, &plan, s);
  return st;
}

uint32_t zero_rows(void *p, uint64_t rows, uint64_t row_bytes, int64_t pitch_bytes, hipStream_t s) {
  const ZeroParams z{p, (int64_t)rows, (int64_t)row_bytes, pitch_bytes};
  return launch_kernel(zero_rows_kernel, dim3((uint32_t)std::min<uint64_t>(2048, (rows * row_bytes / 2 + 255) / 256)), dim3(256), s, z);
}

uint32_t round_rows(uint32_t type, const RoundParams &r, hipStream_t s) {
  const dim3 grid(column_strips(r.cols), (uint32_t)std::min<int64_t>((r.rows + 3) / 4, kGridY));
  return type == CUDA_R_16BF ? launch_kernel(round_rows_kernel<ElemBF16>, grid, dim3(256), s, r) : launch_kernel(round_rows_kernel<ElemF16>, grid, dim3(256), s, r);
}

// the two products and the bias gradient in one launch, then the sums of dX's shares
uint32_t run_together(uint32_t type, const zluda_ffn_gated_grad *p, const zluda_ffn_matrix &x, const GradPlan &plan, const GatedGradParams &g, float *part, hipStream_t s) {
  const GradTogether &t = plan.together;
  const int model = (int)p->model, tokens = (int)p->tokens, f2 = (int)(2 * p->features);
  auto tiles = [](int n) { return (n + kGradTile - 1) / kGradTile; };
  GradProductsParams m;
  m.dx = {p->w.data, g.dz, p->dx.data, part, p->dx.ld, (int32_t)p->w.ld, (int32_t)plan.lddz, model, tokens, f2, tiles(model), tiles(tokens), (int32_t)t.splits, (int32_t)t.split_stages};
  m.dw = {x.data, g.dz, p->dw.data, nullptr, p->dw.ld, (int32_t)x.ld, (int32_t)plan.lddz, model, f2, tokens, tiles(model), tiles(f2), 1, (tokens + kGradStage - 1) / kGradStage};
  m.dx_groups = (uint32_t)(m.dx.tiles_p * m.dx.tiles_q) * t.splits;
  m.sums = g.part; m.dbias = p->dbias; m.shares = (int32_t)plan.shares;
  FFN_CHECK(launch_grad_products(type, m, s));
  if (t.splits == 1) return CUBLAS_STATUS_SUCCESS;
  const int64_t pitch = (int64_t)m.dx.tiles_p * kGradTile;
  return round_rows(type, {part, p->dx.data, tokens, pitch, p->dx.ld, pitch * m.dx.tiles_q * kGradTile, model, (int32_t)t.splits}, s);
}

// ---- layer norm ---------------------------------------------------------------------------------------------------------------
uint32_t check_norm(uint64_t rows, uint64_t cols, const zluda_ffn_matrix &x, uint32_t type, bool x_ckpt, uint32_t weight_type) {
  if (!cols) return CUBLAS_STATUS_INVALID_VALUE;
  if (cols > ZLUDA_FFN_NORM_MAX_COLS || rows > (uint64_t)INT64_MAX / 2 || (!is_h16(type) && type != CUDA_R_32F) || (weight_type != type && weight_type != CUDA_R_32F))
    return CUBLAS_STATUS_NOT_SUPPORTED;
  return check_matrix(x, rows, cols, type, x_ckpt);
}

template <class E>
uint32_t launch_norm(const NormParams &p, hipStream_t s) {
  auto groups = [&](int rows_each, int per_cu) { return dim3((uint32_t)std::min<uint64_t>((p.rows + rows_each - 1) / rows_each, (uint64_t)cus() * per_cu)); };
  if (p.cols <= 512) return launch_kernel(norm_forward_kernel<E, 64, 4, 1>, groups(4, 8), dim3(256), s, p);
  if (p.cols <= 1024) return launch_kernel(norm_forward_kernel<E, 64, 4, 2>, groups(4, 8), dim3(256), s, p);
  if (p.cols <= 2048) return launch_kernel(norm_forward_kernel<E, 256, 1, 1>, groups(1, 8), dim3(256), s, p);
  if (p.cols <= 4096) return launch_kernel(norm_forward_kernel<E, 256, 1, 2>, groups(1, 8), dim3(256), s, p);
  if (p.cols <= 8192) return launch_kernel(norm_forward_kernel<E, 512, 1, 2>, groups(1, 4), dim3(512), s, p);
  return launch_kernel(norm_forward_kernel<E, 1024, 1, 2>, groups(1, 2), dim3(1024), s, p);
}

// Rows a workgroup of the gradient kernel takes at a time, and workgroups: two a CU (one of 1024 threads), each with at least two
// rounds of rows where there are more than 64 rounds, because every workgroup's partial sums are written and read again (us with at
// least 1, 2, 4 rounds: 300 x 4096 bf16 12.2, 10.6, 11.1; 777 x 1001 f16 10.1, 10.0, 11.5; 400 x 16384 32.6, 29.1, 30.8; 62 x 9353 13.7,
// 16.1, 21.8; 3 x 10216 11.1, 13.3, 15.8)
int norm_grad_rows_each(uint64_t cols) { return cols <= 512 ? 8 : cols <= 1024 ? 4 : cols <= 2048 ? 2 : 1; }
uint32_t norm_grad_groups(uint64_t rows, uint64_t cols) {
  const int each = norm_grad_rows_each(cols), least = rows <= 64ull * each ? each : 2 * each;
  if (rows <= 3ull * each) return 1;  // (the sums are its own: no second launch; 2 x 3000 5.2 us, 7.1 by way of partial sums, 4 x 3000 7.8 and 6.9)
  return (uint32_t)std::min<uint64_t>((rows + least - 1) / least, (uint64_t)cus() * (cols <= 4096 ? 2 : 1));
}

template <class E, bool CK>
uint32_t launch_norm_grad(const NormGradParams &p, uint32_t groups, hipStream_t s) {
  if (p.cols <= 512) return launch_kernel(norm_backward_kernel<E, CK, 64, 8, 1>, dim3(groups), dim3(512), s, p);
  if (p.cols <= 1024) return launch_kernel(norm_backward_kernel<E, CK, 128, 4, 1>, dim3(groups), dim3(512), s, p);
  if (p.cols <= 2048) return launch_kernel(norm_backward_kernel<E, CK, 256, 2, 1>, dim3(groups), dim3(512), s, p);
  if (p.cols <= 4096) return launch_kernel(norm_backward_kernel<E, CK, 512, 1, 1>, dim3(groups), dim3(512), s, p);
  if (p.cols <= 8192) return launch_kernel(norm_backward_kernel<E, CK, 1024, 1, 1>, dim3(groups), dim3(1024), s, p);
  return launch_kernel(norm_backward_kernel<E, CK, 1024, 1, 2>, dim3(groups), dim3(1024), s, p);
}
template <class E>
uint32_t launch_norm_grad(const NormGradParams &p, bool ck, uint32_t groups, hipStream_t s) {
  return ck ? launch_norm_grad<E, true>(p, groups, s) : launch_norm_grad<E, false>(p, groups, s);
}

uint32_t check_norm_backward(const zluda_ffn_norm_grad *p) {
  if (!p) return CUBLAS_STATUS_INVALID_VALUE;
  const uint32_t type = p->dy.type;
  FFN_CHECK(check_norm(p->rows, p->cols, p->x, type, true, p->weight_type));
  FFN_CHECK(check_matrix(p->dy, p->rows, p->cols, type, false));
  if (p->add.data) FFN_CHECK(check_matrix(p->add, p->rows, p->cols, type, false));
  if (p->dx.data) FFN_CHECK(check_matrix(p->dx, p->rows, p->cols, type, false));
  if (!p->dweight != !p->dbias || (!p->dx.data && !p->dweight && p->rows) || ((!p->mean || !p->rstd) && p->rows)) return CUBLAS_STATUS_INVALID_VALUE;
  FFN_CHECK(check_vector(p->weight, p->weight_type));
  FFN_CHECK(check_vector(p->dweight, p->weight_type));
  FFN_CHECK(check_vector(p->dbias, p->weight_type));
  FFN_CHECK(check_vector(p->mean, CUDA_R_32F));
  return check_vector(p->rstd, CUDA_R_32F);
}

} // namespace

// ---- gated feed-forward ---------------------------------------------------------------------------------------------------------
extern "C" uint32_t zluda_ffn_gated_forward_workspace(const zluda_ffn_gated *p, size_t *bytes) {
  if (!p || !bytes) return CUBLAS_STATUS_INVALID_VALUE;
  FFN_CHECK(check_sizes(p->activation, p->tokens, p->features, p->model));
  *bytes = 0;
  return CUBLAS_STATUS_SUCCESS;
}

extern "C" uint32_t zluda_ffn_gated_forward(const zluda_ffn_gated *p, void *workspace, size_t workspace_size, void *stream) {
  FFN_CHECK(check_forward(p));
  if (!p->tokens) return CUBLAS_STATUS_SUCCESS;
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  GatedParams g;
  memset(&g, 0, sizeof(g));
  g.x = p->x.data; g.w = p->w.data; g.bias = p->bias;
  g.h = p->h.data; g.gate = p->gate.data; g.up = p->up.data;
  g.gate_scales = (uint8_t *)p->gate.scales; g.up_scales = (uint8_t *)p->up.scales;
  g.ldx = p->x.ld; g.ldw = p->w.ld; g.ldh = p->h.ld; g.ldg = p->gate.ld; g.ldu = p->up.ld;
  g.ldgs = p->gate.ld_scales; g.ldus = p->up.ld_scales;
  g.tokens = (int32_t)p->tokens; g.features = (int32_t)p->features; g.model = (int32_t)p->model;
  g.activation = p->activation;
  g.kept = !p->gate.data ? 0 : p->gate.type == CUDA_R_8F_E4M3 ? 2 : 1;
  const uint64_t part = rows_in_window(p->tokens, p->x.ld);
  for (uint64_t t = 0; t < p->tokens; t += part) {
    g.tokens = (int32_t)std::min(part, p->tokens - t);
    FFN_CHECK(p->x.type == CUDA_R_16BF ? launch_gated_bf16(g, (hipStream_t)stream) : launch_gated_f16(g, (hipStream_t)stream));
    const int64_t kept = g.kept == 2 ? 1 : 2;
    g.x = (const char *)g.x + part * g.ldx * 2;
    g.h = (char *)g.h + part * g.ldh * 2;
    if (g.kept) {
      g.gate = (char *)g.gate + part * g.ldg * kept;
      g.up = (char *)g.up + part * g.ldu * kept;
    }
    if (g.kept == 2) {
      g.gate_scales += part * g.ldgs;
      g.up_scales += part * g.ldus;
    }
  }
  return CUBLAS_STATUS_SUCCESS;
}

extern "C" uint32_t zluda_ffn_gated_backward_workspace(const zluda_ffn_gated_grad *p, size_t *bytes) {
  if (!p || !bytes) return CUBLAS_STATUS_INVALID_VALUE;
  FFN_CHECK(check_sizes(p->activation, p->tokens, p->features, p->model));
  *bytes = (size_t)grad_plan(p).total;
  return CUBLAS_STATUS_SUCCESS;
}

extern "C" uint32_t zluda_ffn_gated_backward(const zluda_ffn_gated_grad *p, void *workspace, size_t workspace_size, void *stream) {
  FFN_CHECK(check_backward(p));
  const hipStream_t s = (hipStream_t)stream;
  const uint32_t type = p->dh.type;
  const GradPlan plan = grad_plan(p);
  if (plan.total > workspace_size || (plan.total && !workspace)) return CUBLAS_STATUS_ALLOC_FAILED;
  if ((uintptr_t)workspace & 15) return CUBLAS_STATUS_INVALID_VALUE;
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (!p->tokens) {  // sums of no terms
    if (p->dw.data) FFN_CHECK(zero_rows(p->dw.data, 2 * p->features, p->model * 2, p->dw.ld * 2, s));
    if (p->dbias) FFN_CHECK(zero_rows(p->dbias, 1, p->features * 4, 0, s));
    return CUBLAS_STATUS_SUCCESS;
  }
  char *ws = (char *)workspace;
  GatedGradParams g;
  memset(&g, 0, sizeof(g));
  g.dh = p->dh.data; g.gate = p->gate.data; g.up = p->up.data;
  g.gate_scales = (const uint8_t *)p->gate.scales; g.up_scales = (const uint8_t *)p->up.scales;
  g.dz = p->dz.data ? p->dz.data : ws + plan.dz;
  g.h = p->h.data;
  g.part = p->dbias ? (float *)(ws + plan.sums) : nullptr;
  g.tokens = (int64_t)p->tokens;
  g.lddh = p->dh.ld; g.ldg = p->gate.ld; g.ldu = p->up.ld; g.ldgs = p->gate.ld_scales; g.ldus = p->up.ld_scales;
  g.lddz = plan.lddz; g.ldh = p->h.ld;
  g.features = (int32_t)p->features;
  g.activation = p->activation;
  const bool ck = p->gate.type == CUDA_R_8F_E4M3;
  // a checkpoint of x is decoded for the product by the same launch
  zluda_ffn_matrix x = p->x;
  if (p->dw.data && p->x.type == CUDA_R_8F_E4M3) {
    x = {ws + plan.x, nullptr, aligned_pitch(p->model), 0, type};
    g.load = CheckpointParams{x.data, (uint8_t *)p->x.data, (uint8_t *)p->x.scales, (int64_t)p->tokens, x.ld, p->x.ld, p->x.ld_scales, (int32_t)p->model};
  }
  FFN_CHECK(type == CUDA_R_16BF ? (ck ? launch_gated_grad<ElemBF16, true>(g, plan.shares, s) : launch_gated_grad<ElemBF16, false>(g, plan.shares, s))
                                : (ck ? launch_gated_grad<ElemF16, true>(g, plan.shares, s) : launch_gated_grad<ElemF16, false>(g, plan.shares, s)));
  void *gemm_ws = ws + plan.gemm;
  if (plan.together.splits && grad_together_operands(p, x, plan.lddz, g.dz)) return run_together(type, p, x, plan, g, (float *)gemm_ws, s);
  if (p->dbias) {
    NormFinishParams f{g.part, p->dbias, nullptr, (int32_t)plan.shares, (int32_t)(2 * p->features), type};
    FFN_CHECK(launch_kernel(norm_finish_kernel<16, 64>, dim3((uint32_t)((2 * p->features + 15) / 16), 1), dim3(1024), s, f));
  }
  const uint64_t f2 = 2 * p->features;
  // row-major matrices are column-major ones transposed: dx^T = W^T dz^T, dw^T = x^T dz
  auto rows_of = [](const void *m, int64_t ld, uint64_t row) { return (char *)m + row * ld * 2; };
  if (p->dx.data)
    for (uint64_t t = 0; t < p->tokens; t += plan.dx_rows)
      FFN_CHECK(run_matmul(type, CUBLAS_OP_N, CUBLAS_OP_N, p->model, std::min(plan.dx_rows, p->tokens - t), f2, p->w.data, p->w.ld, rows_of(g.dz, plan.lddz, t), plan.lddz,
                           type, 0.0f, rows_of(p->dx.data, p->dx.ld, t), p->dx.ld, gemm_ws, kGemmWorkspace, s));
  if (p->dw.data) {
    const bool parts = plan.dw_rows < p->tokens;
    void *sum = parts ? ws + plan.acc : p->dw.data;
    const int64_t ld_sum = parts ? aligned_pitch(p->model) : p->dw.ld;
    for (uint64_t t = 0; t < p->tokens; t += plan.dw_rows)
      FFN_CHECK(run_matmul(type, CUBLAS_OP_N, CUBLAS_OP_T, p->model, f2, std::min(plan.dw_rows, p->tokens - t), rows_of(x.data, x.ld, t), x.ld, rows_of(g.dz, plan.lddz, t),
                           plan.lddz, parts ? CUDA_R_32F : type, t ? 1.0f : 0.0f, sum, ld_sum, gemm_ws, kGemmWorkspace, s));
    if (parts) FFN_CHECK(round_rows(type, {(const float *)sum, p->dw.data, (int64_t)f2, ld_sum, p->dw.ld, 0, (int32_t)p->model, 1}, s));
  }
  return CUBLAS_STATUS_SUCCESS;
}

// ---- layer norm -----------------------------------------------------------------------------------------------------------------
extern "C" uint32_t zluda_ffn_norm_forward(const zluda_ffn_norm *p, void *stream) {
  if (!p) return CUBLAS_STATUS_INVALID_VALUE;
  FFN_CHECK(check_norm(p->rows, p->cols, p->x, p->x.type, false, p->weight_type));
  FFN_CHECK(check_matrix(p->y, p->rows, p->cols, p->x.type, false));
  if (p->kept.data) {
    if (p->kept.type != CUDA_R_8F_E4M3) return CUBLAS_STATUS_NOT_SUPPORTED;
    FFN_CHECK(check_matrix(p->kept, p->rows, p->cols, p->x.type, true));
  }
  FFN_CHECK(check_vector(p->weight, p->weight_type));
  FFN_CHECK(check_vector(p->bias, p->weight_type));
  FFN_CHECK(check_vector(p->mean, CUDA_R_32F));
  FFN_CHECK(check_vector(p->rstd, CUDA_R_32F));
  if (!p->rows) return CUBLAS_STATUS_SUCCESS;
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  NormParams n{p->x.data, p->y.data, (uint8_t *)p->kept.data, (uint8_t *)p->kept.scales, p->weight, p->bias, p->mean, p->rstd, (int64_t)p->rows, p->x.ld,
               p->y.ld, p->kept.ld, p->kept.ld_scales, p->eps, (int32_t)p->cols, p->weight_type};
  switch (p->x.type) {
  case CUDA_R_16BF: return launch_norm<ElemBF16>(n, (hipStream_t)stream);
  case CUDA_R_16F: return launch_norm<ElemF16>(n, (hipStream_t)stream);
  default: return launch_norm<ElemF32>(n, (hipStream_t)stream);
  }
}

extern "C" uint32_t zluda_ffn_norm_backward_workspace(const zluda_ffn_norm_grad *p, size_t *bytes) {
  if (!p || !bytes || !p->cols) return CUBLAS_STATUS_INVALID_VALUE;
  if (p->cols > ZLUDA_FFN_NORM_MAX_COLS) return CUBLAS_STATUS_NOT_SUPPORTED;
  const uint32_t groups = p->rows ? norm_grad_groups(p->rows, p->cols) : 1;
  *bytes = p->dweight && groups > 1 ? (size_t)groups * 2 * p->cols * 4 : 0;  // (a single workgroup has the sums themselves)
  return CUBLAS_STATUS_SUCCESS;
}

extern "C" uint32_t zluda_ffn_norm_backward(const zluda_ffn_norm_grad *p, void *workspace, size_t workspace_size, void *stream) {
  FFN_CHECK(check_norm_backward(p));
  size_t need = 0;
  FFN_CHECK(zluda_ffn_norm_backward_workspace(p, &need));
  if (need > workspace_size || (need && !workspace)) return CUBLAS_STATUS_ALLOC_FAILED;
  if ((uintptr_t)workspace & 15) return CUBLAS_STATUS_INVALID_VALUE;
  if (!zluda_gemm_device_cu_count()) return CUBLAS_STATUS_NOT_INITIALIZED;
  const hipStream_t s = (hipStream_t)stream;
  if (!p->rows) {  // sums of no terms
    if (p->dweight) {
      FFN_CHECK(zero_rows(p->dweight, 1, p->cols * elem_size(p->weight_type), 0, s));
      FFN_CHECK(zero_rows(p->dbias, 1, p->cols * elem_size(p->weight_type), 0, s));
    }
    return CUBLAS_STATUS_SUCCESS;
  }
  const uint32_t groups = norm_grad_groups(p->rows, p->cols);
  NormGradParams n{p->x.data, p->dy.data, p->add.data, (const uint8_t *)p->x.scales, p->dx.data, p->weight, p->mean, p->rstd, p->dweight && groups > 1 ? (float *)workspace : nullptr,
                   groups > 1 ? nullptr : p->dweight, groups > 1 ? nullptr : p->dbias, (int64_t)p->rows, p->x.ld, p->x.ld_scales, p->dy.ld, p->add.ld, p->dx.ld, (int32_t)p->cols, p->weight_type};
  const bool ck = p->x.type == CUDA_R_8F_E4M3;
  FFN_CHECK(p->dy.type == CUDA_R_16BF  ? launch_norm_grad<ElemBF16>(n, ck, groups, s)
            : p->dy.type == CUDA_R_16F ? launch_norm_grad<ElemF16>(n, ck, groups, s)
                                       : launch_norm_grad<ElemF32>(n, ck, groups, s));
  if (!p->dweight || groups == 1) return CUBLAS_STATUS_SUCCESS;
  NormFinishParams f{n.part, p->dweight, p->dbias, (int32_t)groups, (int32_t)p->cols, p->weight_type};
  return launch_kernel(norm_finish_kernel<16, 64>, dim3((uint32_t)((p->cols + 15) / 16), 2), dim3(1024), s, f);
}

// ---- checkpoints ----------------------------------------------------------------------------------------------------------------
extern "C" uint32_t zluda_ffn_checkpoint_store(uint64_t rows, uint64_t cols, const zluda_ffn_matrix *x, const zluda_ffn_matrix *checkpoint, void *stream) {
  return checkpoint_call(true, rows, cols, x, checkpoint, stream);
}
extern "C" uint32_t zluda_ffn_checkpoint_load(uint64_t rows, uint64_t cols, const zluda_ffn_matrix *checkpoint, const zluda_ffn_matrix *x, void *stream) {
  return checkpoint_call(false, rows, cols, x, checkpoint, stream);
}
