"""Which kernel, tile and shares of K the products with a scale for each 128 of K take, and which workspace gradients by expert ask for, without a GPU: what the launchers and the
kernels rely on, over sizes around every rule."""
import ctypes as C

import pytest

from zluda_amd import abi as K, ffn

VEC, BLK = K.CUBLASLT_MATMUL_MATRIX_SCALE_VEC128_32F, K.CUBLASLT_MATMUL_MATRIX_SCALE_BLK128x128_32F
TILES = [(256, 256, 512), (128, 128, 256), (64, 64, 256), (64, 32, 256), (128, 64, 256), (128, 128, 256), (128, 96, 256), (16, 16, 512)]      # rows of P, of Q, threads
CUS = 256


def plan(api, m, n, k, out=K.CUDA_R_16BF, modes=(BLK, VEC), row_major=False, batch=1, workspace=32 << 20, variant=-1, kernel=0):
    p = K.zluda_gemm_problem()

    def lay(x, typ, rows, cols, ld, order=K.CUBLASLT_ORDER_COL):
        x.type, x.order, x.rows, x.cols, x.ld, x.batch_count, x.batch_stride = typ, order, rows, cols, ld, batch, ld * (rows if order else cols)
    k16 = -(-k // 16) * 16
    order = K.CUBLASLT_ORDER_ROW if row_major else K.CUBLASLT_ORDER_COL
    lay(p.a, K.CUDA_R_8F_E4M3, k, m, k16)
    lay(p.b, K.CUDA_R_8F_E4M3, k, n, k16)
    for x in (p.c, p.d):
        lay(x, out, m, n, n if row_major else m, order)
    o = p.op
    o.compute_type, o.scale_type, o.transa, o.epilogue, o.bias_type, o.epilogue_aux_type = K.CUBLAS_COMPUTE_32F, K.CUDA_R_32F, K.CUBLAS_OP_T, K.CUBLASLT_EPILOGUE_DEFAULT, -1, -1
    o.a_scale_mode, o.b_scale_mode, o.a_scale, o.b_scale = *modes, 4096, 8192
    one, zero = C.c_float(1), C.c_float(0)
    p.alpha, p.beta, p.A, p.B, p.C, p.D = C.addressof(one), C.addressof(zero), 1 << 20, 1 << 21, 1 << 22, 1 << 22
    p.workspace_size = workspace
    got = K.zluda_gemm_plan()
    st = api.zluda_gemm_plan_problem(C.byref(p), kernel, variant, CUS, C.byref(got))
    return (st, got)


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (256, 1, 1024), (2048, 1, 2048), (2048, 16, 2048), (4096, 16, 2048), (4112, 1, 2048), (2048, 17, 2048), (2048, 1, 2064), (4096, 1, 14336),
                                   (14336, 4, 4096), (333, 5632, 2000), (5632, 333, 2000), (8192, 8192, 8192), (3264, 2559, 320), (100, 100, 100000), (128, 128, 512)])
def test_plans(api, m, n, k):
    for out in (K.CUDA_R_16BF, K.CUDA_R_32F):
        for modes in ((BLK, VEC), (VEC, VEC), (VEC, BLK)):
            for row_major in (False, True):
                for batch, workspace in ((1, 32 << 20), (1, 0), (3, 1 << 20)):
                    st, p = plan(api, m, n, k, out, modes, row_major, batch, workspace)
                    assert st == 0 and p.kernel == K.ZLUDA_KERNEL_MFMA_BLK8
                    swapped = row_major and n > 1                  # (a single column of pitch 1 is either)
                    np, nq = (n, m) if swapped else (m, n)
                    bp, bq, threads = TILES[p.variant]
                    tiles, blocks = -(-np // bp) * -(-nq // bq), -(-k // 128)
                    assert p.swapped == swapped and (p.grid_x, p.grid_y, p.block) == (tiles, batch, threads)
                    assert 1 <= p.grid_z <= max(1, blocks // 4) and p.workspace <= workspace
                    assert p.workspace == (p.grid_z * batch * tiles * bp * bq * 4 if p.grid_z > 1 else 0)
                    # shares of K inside the workgroup: few tokens, two blocks of K a wave, one round of workgroups
                    assert (p.variant == 7) == (nq <= 16 and k <= 2048 and -(-np // 16) * batch <= CUS)
                    if out == K.CUDA_R_32F:
                        assert p.variant in (2, 3, 4, 7)
                    if modes[1 if swapped else 0] == VEC:
                        assert p.variant != 0


def test_forced_variants(api):
    for v in range(8):
        st, p = plan(api, 512, 300, 1024, variant=v, kernel=K.ZLUDA_KERNEL_MFMA_BLK8)
        assert st == 0 and p.variant == v
        assert plan(api, 512, 300, 1024, modes=(VEC, VEC), variant=v, kernel=K.ZLUDA_KERNEL_MFMA_BLK8)[0] == (0 if v else K.CUBLAS_STATUS_NOT_SUPPORTED)
        assert plan(api, 512, 300, 1024, out=K.CUDA_R_32F, variant=v, kernel=K.ZLUDA_KERNEL_MFMA_BLK8)[0] == (0 if v in (2, 3, 4, 7) else K.CUBLAS_STATUS_NOT_SUPPORTED)
    assert plan(api, 512, 300, 1024, variant=8, kernel=K.ZLUDA_KERNEL_MFMA_BLK8)[0] == K.CUBLAS_STATUS_INVALID_VALUE
    assert api.zluda_gemm_variant_count(K.ZLUDA_KERNEL_MFMA_BLK8) == 8


def grad_workspace(rows, experts, features, model, dx=True, dw=True, **ld):
    return ffn.GroupedBackward(dict(type=K.CUDA_R_16BF, rows=rows, experts=experts, features=features, model=model, dx=dx, dw=dw, **ld)).workspace


def test_workspace_of_gradients_by_expert():
    # few tiles of dx with a long K: whole shares of rows x (model, whole tiles of 128) in 32 bits
    for rows, experts, features, model in ((64, 8, 5632, 2048), (692, 2, 4744, 2688), (64, 1, 4096, 4096), (300, 8, 2816, 1000)):
        ws, share = grad_workspace(rows, experts, features, model), rows * -(-model // 128) * 128 * 4
        assert ws and ws % share == 0 and 2 <= ws // share <= 16
        assert grad_workspace(rows, experts, features, model, dx=False) == 0
        assert grad_workspace(rows, experts, features, model, ldw=model + 1) == 0          # (the kernel for any alignment)
    for rows, experts, features, model in ((16384, 8, 5632, 2048), (0, 8, 5632, 2048), (2000, 2, 1024, 1024), (64, 8, 64, 4096)):
        assert grad_workspace(rows, experts, features, model) == 0
    p, n = ffn.zluda_ffn_grouped_grad(10, 0, 200, 300), C.c_size_t()
    assert ffn.load().zluda_ffn_grouped_backward_workspace(C.byref(p), C.byref(n)) == K.CUBLAS_STATUS_INVALID_VALUE
    p = ffn.zluda_ffn_grouped_grad(10, 5000, 200, 300)
    assert ffn.load().zluda_ffn_grouped_backward_workspace(C.byref(p), C.byref(n)) == K.CUBLAS_STATUS_NOT_SUPPORTED
    # pitches that are not set yet, or make no sense
    p = ffn.zluda_ffn_grouped_grad(64, 8, 5632, 2048)
    for name in ("dx", "dw"):
        getattr(p, name).data = 16
    for ld in (0, -8, -(1 << 62)):
        for name in ("dy", "x", "w", "dx", "dw"):
            for other in ("dy", "x", "w", "dx", "dw"):
                getattr(p, other).ld = ld if other == name else 5632
            assert ffn.load().zluda_ffn_grouped_backward_workspace(C.byref(p), C.byref(n)) == 0 and n.value == 0
