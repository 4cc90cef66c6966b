"""A row-major D of one column and pitch 1: unit strides both ways."""
import ctypes as C

import pytest
import torch

from zluda_amd import abi as K, cublaslt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", ["i8", "f8", "bf16", "f32"])
@pytest.mark.parametrize("m", [2, 16, 40, 200, 300])
@pytest.mark.parametrize("trans", [(1, 0), (0, 0)])
def test_row_major_column(gpu_api, typ, m, trans):
    k = 64
    torch.manual_seed(m)
    a, b = torch.randint(-8, 9, (m, k)), torch.randint(-8, 9, (1, k))
    dt, code, out, ocode, compute, scale = {
        "i8": (torch.int8, K.CUDA_R_8I, torch.int32, K.CUDA_R_32I, K.CUBLAS_COMPUTE_32I, K.CUDA_R_32I),
        "f8": (torch.float8_e4m3fn, K.CUDA_R_8F_E4M3, torch.float32, K.CUDA_R_32F, K.CUBLAS_COMPUTE_32F, K.CUDA_R_32F),
        "bf16": (torch.bfloat16, K.CUDA_R_16BF, torch.float32, K.CUDA_R_32F, K.CUBLAS_COMPUTE_32F, K.CUDA_R_32F),
        "f32": (torch.float32, K.CUDA_R_32F, torch.float32, K.CUDA_R_32F, K.CUBLAS_COMPUTE_32F, K.CUDA_R_32F)}[typ]
    A = (a if trans[0] else a.t().contiguous()).float().to(dt).cuda()
    B, D = b.float().to(dt).cuda(), torch.full((m + 64,), 77, dtype=out, device="cuda")
    call = cublaslt.MatmulCall(gpu_api, dict(m=m, n=1, k=k, a_type=code, b_type=code, d_type=ocode, compute_type=compute, scale_type=scale, transa=trans[0], transb=trans[1],
                                             order_c=K.CUBLASLT_ORDER_ROW, order_d=K.CUBLASLT_ORDER_ROW))
    one, zero = (C.c_int32(1), C.c_int32(0)) if typ == "i8" else (C.c_float(1), C.c_float(0))
    assert call.run(one, A.data_ptr(), B.data_ptr(), zero, D.data_ptr(), D.data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(D[:m].cpu().long(), (a @ b.t())[:, 0]) and (D[m:] == 77).all(), call.kernel
    call.close()
