"""cublasLtMatmul with a scale for each 128 of K where its result goes on: GELU with its input kept, GELU's gradient, alpha per row; and plans that name a kernel
without shares of K with some."""
import ctypes as C

import pytest
import torch

import ffn_oracle as O
import packed_oracle as P
from test_gpu_ffn import DEV, TYPES, randn, stream
from test_gpu_scaled_matmul import BLK, F8, VEC, Operand
from zluda_amd import abi as K, cublaslt

pytestmark = pytest.mark.gpu
SIZES = [(64, 1, 256), (264, 9, 1040), (520, 300, 400), (1024, 1024, 512)]


def setup(api, m, n, k, out, **over):
    A, B = Operand(m, k, "e4m3", BLK, 1), Operand(n, k, "e4m3", VEC, 2)
    spec = dict(m=m, n=n, k=k, a_type=F8["e4m3"][1], b_type=F8["e4m3"][1], d_type=TYPES[out][1], compute_type=K.CUBLAS_COMPUTE_32F, scale_type=K.CUDA_R_32F, transa=K.CUBLAS_OP_T,
                lda=A.ld, ldb=B.ld, a_scale_mode=BLK, b_scale_mode=VEC, **over)
    return A, B, cublaslt.MatmulCall(api, spec, max_workspace=8 << 20), P.scaled_product(B.codes[0], A.codes[0], B.spread[0], A.spread[0], out == "f32")


def call_it(call, A, B, D, alpha=None, **pointers):
    call.set_pointers(a_scale=A.scales.data_ptr(), b_scale=B.scales.data_ptr(), **pointers)
    ws = torch.empty(8 << 20, dtype=torch.uint8, device=DEV)
    assert call.run(C.c_float(1) if alpha is None else alpha, A.ptr, B.ptr, C.c_float(0), D.data_ptr(), D.data_ptr(), ws.data_ptr(), ws.numel(), stream()) == 0
    torch.cuda.synchronize()
    call.close()


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gelu_with_its_input_kept(gpu_api, m, n, k, out):
    dt = TYPES[out][0]
    A, B, call, (v, e) = setup(gpu_api, m, n, k, out, epilogue=K.CUBLASLT_EPILOGUE_GELU_AUX_BIAS, aux_ld=m)
    D, aux, bias = torch.empty((n, m), dtype=dt, device=DEV), torch.empty((n, m), dtype=dt, device=DEV), randn(5, m).to(dt)
    call_it(call, A, B, D, bias=bias.data_ptr(), aux=aux.data_ptr())
    v = v + bias.double()
    O.check(aux, (v, e + 2 * O.E32 * (v.abs() + bias.double().abs())), "aux")
    g, _, z, _ = O.act("gelu", aux.double())                    # (of what is kept)
    O.check(D, (g, (z + 16) * 4 * O.E32 * g.abs() + aux.double().abs() * 2.0 ** -126), "D")


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gelu_s_gradient(gpu_api, m, n, k, out):
    dt = TYPES[out][0]
    A, B, call, (v, e) = setup(gpu_api, m, n, k, out, epilogue=K.CUBLASLT_EPILOGUE_DGELU, aux_ld=m)
    D, aux = torch.empty((n, m), dtype=dt, device=DEV), randn(5, n, m).to(dt)
    call_it(call, A, B, D, aux=aux.data_ptr())
    _, dg, z, terms = O.act("gelu", aux.double())
    e = e + O.UNIT[dt] * (v.abs() + e) * 1.001 + O.TINY[dt]        # the product is rounded to D's type in front of the gradient's pass
    # the gradient's pass has the tanh t, 1 - 2 / (1 + exp), at the size of 1, where the reciprocal, the product and the difference leave it 4 * 2^-24 off, and makes
    # (1 + t) / 2 + x / 2 (1 - t^2) u' of it, whose derivative in t is 1 / 2 - x t u': for x << 0 that is far above the gradient itself
    x = aux.double()
    du = O.K2 / 2 * (1 + 3 * 0.044715 * x * x)
    off = (z + 16) * 4 * O.E32 * terms + 4 * O.E32 * (1 + x.abs() * du)
    O.check(D, (v * dg, e * (dg.abs() + off) + v.abs() * off), "D")


@pytest.mark.parametrize("m,n,k", SIZES)
def test_alpha_for_each_row(gpu_api, m, n, k):
    A, B, call, (v, e) = setup(gpu_api, m, n, k, "bf16", pointer_mode=K.CUBLASLT_POINTER_MODE_ALPHA_DEVICE_VECTOR_BETA_ZERO)
    alpha, D = randn(7, m), torch.empty((n, m), dtype=torch.bfloat16, device=DEV)
    call_it(call, A, B, D, alpha=alpha.data_ptr())
    a = alpha.double()
    O.check(D, (v * a, e * a.abs() + 2 * O.E32 * (v * a).abs()), "D")


def test_a_plan_with_shares_for_a_kernel_without(gpu_api):
    A, B = Operand(256, 1024, "e4m3", BLK, 1), Operand(4, 1024, "e4m3", VEC, 2)
    D, ws = torch.full((4, 256), 5.0, dtype=torch.bfloat16, device=DEV), torch.empty(8 << 20, dtype=torch.uint8, device=DEV)
    from oracle.cases import Case  # (its problem() lays out a zluda_gemm_problem)
    case = Case(dict(m=256, n=4, k=1024, a_type=K.CUDA_R_8F_E4M3, b_type=K.CUDA_R_8F_E4M3, c_type=K.CUDA_R_16BF, d_type=K.CUDA_R_16BF, compute_type=K.CUBLAS_COMPUTE_32F,
                     scale_type=K.CUDA_R_32F, transa=1), 1)
    one, zero = C.c_float(1), C.c_float(0)
    p = case.problem(dict(A=A.ptr, B=B.ptr, C=D.data_ptr(), D=D.data_ptr(), alpha=C.addressof(one), beta=C.addressof(zero)))
    p.op.a_scale_mode, p.op.b_scale_mode, p.op.a_scale, p.op.b_scale = BLK, VEC, A.scales.data_ptr(), B.scales.data_ptr()
    p.workspace, p.workspace_size = ws.data_ptr(), ws.numel()
    plan = K.zluda_gemm_plan()
    assert gpu_api.zluda_gemm_plan_problem(C.byref(p), K.ZLUDA_KERNEL_MFMA_BLK8, 7, gpu_api.zluda_gemm_device_cu_count(), C.byref(plan)) == 0
    assert plan.grid_z == 1 and plan.workspace == 0
    plan.grid_z, plan.workspace = 2, 1 << 20
    assert gpu_api.zluda_gemm_launch(C.byref(p), C.byref(plan), stream()) == K.CUBLAS_STATUS_INVALID_VALUE
    torch.cuda.synchronize()
    assert (D == 5).all()
