"""cublasLtMatmul of 8-bit floats with a float scale for each 128 of K (VEC128_32F, BLK128x128_32F) on the GPU against 64 bits: every pair of modes, type,
layout and epilogue, sizes around the edges of the tiles, with guard bytes around D."""
import ctypes as C

import pytest
import torch

import ffn_oracle as O
import packed_oracle as P
from test_gpu_ffn import DEV, Mat, TYPES, randn, stream
from zluda_amd import abi as K, cublaslt

pytestmark = pytest.mark.gpu
VEC, BLK = K.CUBLASLT_MATMUL_MATRIX_SCALE_VEC128_32F, K.CUBLASLT_MATMUL_MATRIX_SCALE_BLK128x128_32F
F8 = {"e4m3": (torch.float8_e4m3fn, K.CUDA_R_8F_E4M3), "e5m2": (torch.float8_e5m2, K.CUDA_R_8F_E5M2)}
EPI = {("none", 0): K.CUBLASLT_EPILOGUE_DEFAULT, ("none", 1): K.CUBLASLT_EPILOGUE_BIAS, ("relu", 0): K.CUBLASLT_EPILOGUE_RELU, ("relu", 1): K.CUBLASLT_EPILOGUE_RELU_BIAS,
       ("gelu", 0): K.CUBLASLT_EPILOGUE_GELU, ("gelu", 1): K.CUBLASLT_EPILOGUE_GELU_BIAS}


class Operand:
    """rows x k codes (row: one index of D), k- or row-contiguous, in `batch` copies, with their scales and what they stand for"""

    def __init__(self, rows, k, typ, mode, seed, kc=True, pad=0, skip=0, batch=1):
        self.rows, self.k, self.kc = rows, k, kc
        gen = torch.Generator(device=DEV)
        gen.manual_seed(seed)
        v = torch.randn((batch, rows, k), device=DEV, generator=gen).to(F8[typ][0])
        lead = k if kc else rows
        self.ld = lead + pad
        self.stride = (rows if kc else k) * self.ld + (16 if batch > 1 else 0)
        self.raw = torch.full((256 + skip + batch * self.stride,), 0x7F, dtype=torch.uint8, device=DEV)     # (NaN around the operand)
        for b in range(batch):
            at = 256 + skip + b * self.stride
            m = self.raw[at:at + (rows if kc else k) * self.ld].view(rows if kc else k, self.ld)[:, :lead]
            m.copy_((v[b] if kc else v[b].t()).contiguous().view(torch.uint8))
        self.ptr = self.raw.data_ptr() + 256 + skip
        kb = P.blocks(k)
        shape = (batch, kb, rows) if mode == VEC else (batch, P.blocks(rows), -(-kb // 4) * 4)
        self.scales = torch.exp2(torch.rand(shape, device=DEV, generator=gen) * 8 - 4)
        s = self.scales.double()
        if mode == VEC:
            s = s.transpose(1, 2).repeat_interleave(128, 2)
        else:
            s = s[:, :, :kb].repeat_interleave(128, 1)[:, :rows].repeat_interleave(128, 2)
        self.codes, self.spread = v.double(), s[:, :, :k]


def run(api, m, n, k, a_mode=BLK, b_mode=VEC, a="e4m3", b="e4m3", out="bf16", act="none", bias=0, akc=True, bkc=True, row_major=False, pad=0, skip=0, batch=1, beta=0.0, alpha=1.0,
        workspace=32 << 20, kernel=None, variant=-1, d_scale=None, bias_type=None, seed=0):
    A, B = Operand(m, k, a, a_mode, seed + 1, akc, pad, skip, batch), Operand(n, k, b, b_mode, seed + 2, bkc, pad, skip, batch)
    dt, dcode = TYPES[out]
    # D as the rows of its unit stride
    q, p = (m, n) if row_major else (n, m)
    D = Mat(batch * q, p, dt, p + pad, skip, randn(seed + 3, batch * q, p) if beta else None)
    spec = dict(m=m, n=n, k=k, batch=batch, a_type=F8[a][1], b_type=F8[b][1], d_type=dcode, compute_type=K.CUBLAS_COMPUTE_32F, scale_type=K.CUDA_R_32F,
                transa=K.CUBLAS_OP_T if akc else K.CUBLAS_OP_N, transb=K.CUBLAS_OP_N if bkc else K.CUBLAS_OP_T, lda=A.ld, ldb=B.ld, ldc=D.ld, ldd=D.ld,
                a_scale_mode=a_mode, b_scale_mode=b_mode, epilogue=EPI[(act, bias)])
    if batch > 1:
        spec.update(stride_a=A.stride, stride_b=B.stride, stride_c=q * D.ld, stride_d=q * D.ld)
    if row_major:
        spec.update(order_c=K.CUBLASLT_ORDER_ROW, order_d=K.CUBLASLT_ORDER_ROW)
    bt = torch.float32 if bias_type else dt
    vec = randn(seed + 4, m).to(bt) if bias else None
    if bias_type:
        spec["bias_type"] = K.CUDA_R_32F
    call = cublaslt.MatmulCall(api, spec, forced_kernel=kernel, forced_variant=variant, max_workspace=workspace)
    sd = torch.tensor([d_scale], device=DEV) if d_scale is not None else None
    call.set_pointers(bias=vec.data_ptr() if bias else None, a_scale=A.scales.data_ptr(), b_scale=B.scales.data_ptr(), d_scale=sd.data_ptr() if sd is not None else None)
    ws = torch.empty(max(16, workspace), dtype=torch.uint8, device=DEV)
    old = D.view.double().clone() if beta else None
    st = call.run(C.c_float(alpha), A.ptr, B.ptr, C.c_float(beta), D.ptr, D.ptr, ws.data_ptr(), workspace, stream())
    torch.cuda.synchronize()
    got_kernel, got_variant = call.kernel, call.variant
    call.close()
    assert st == 0, "status %d" % st
    what = "%dx%dx%d kernel %d/%d" % (m, n, k, got_kernel, got_variant)
    assert D.guards(), what
    for i in range(batch):
        v, e = P.scaled_product(B.codes[i], A.codes[i], B.spread[i], A.spread[i], out == "f32")      # n x m
        v, e = v * alpha, e * abs(alpha) + 2 * O.E32 * abs(alpha) * v.abs()
        if row_major:
            v, e = v.t(), e.t()
        if beta:
            c = old[i * q:(i + 1) * q] * beta
            v, e = v + c, e + 2 * O.E32 * (v.abs() + c.abs())
        if bias:
            t = vec.double()[:, None] if row_major else vec.double()
            v, e = v + t, e + 2 * O.E32 * (v.abs() + t.abs())
        if act == "relu":
            v = v.clamp(min=0)
        elif act == "gelu":
            a_, _, za, _ = O.act("gelu", v)
            # (the sigmoid comes out of v_rcp_f32, whose results below 2^-126, the smallest normal number, are zeros: up to |v| 2^-126)
            v, e = a_, 1.13 * e + (za + 16) * 4 * O.E32 * a_.abs() + (v.abs() + e) * 2.0 ** -126
        if d_scale is not None:
            v, e = v * d_scale, e * abs(d_scale) + O.E32 * (v * d_scale).abs()
        O.check(D.view[i * q:(i + 1) * q], (v, e), what)
    return got_kernel, got_variant


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (16, 1, 128), (64, 64, 128), (65, 3, 144), (128, 17, 256), (256, 33, 400), (200, 100, 1040), (384, 300, 2000), (1000, 64, 512),
                                   (72, 513, 640), (520, 260, 4096), (4096, 1, 2048), (2048, 5, 14336), (256, 256, 128), (257, 511, 384)])
def test_sizes(gpu_api, m, n, k):
    for a_mode, b_mode in ((BLK, VEC), (VEC, VEC), (VEC, BLK), (BLK, BLK)):
        run(gpu_api, m, n, k, a_mode, b_mode)
    run(gpu_api, m, n, k, workspace=0)
    run(gpu_api, m, n, k, VEC, BLK, row_major=True)


@pytest.mark.parametrize("variant", [0, 1, 2, 3, 4, 5])
@pytest.mark.parametrize("k", [16, 128, 256, 272, 384, 512, 640, 784, 1040, 1152, 2048])
def test_every_tile_at_every_length(gpu_api, variant, k):
    """counts of stages around those of the rings, whole tiles and ragged ones, shared out along K and not"""
    for m, n in ((256, 256), (130, 40), (300, 290), (520, 1)):
        for modes in ((BLK, VEC), (BLK, BLK), (VEC, VEC), (VEC, BLK)):
            if variant == 0 and modes[0] == VEC:
                continue
            assert run(gpu_api, m, n, k, *modes, kernel=K.ZLUDA_KERNEL_MFMA_BLK8, variant=variant) == (K.ZLUDA_KERNEL_MFMA_BLK8, variant)
            if variant in (2, 3, 4):
                assert run(gpu_api, m, n, k, *modes, out="f32", kernel=K.ZLUDA_KERNEL_MFMA_BLK8, variant=variant) == (K.ZLUDA_KERNEL_MFMA_BLK8, variant)
        run(gpu_api, m, n, k, BLK, VEC, kernel=K.ZLUDA_KERNEL_MFMA_BLK8, variant=variant, workspace=0, act="gelu", bias=1, pad=16)


@pytest.mark.parametrize("a,b", [("e4m3", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
def test_types(gpu_api, a, b, out):
    for m, n, k in ((136, 1, 272), (264, 70, 528), (512, 300, 1024)):
        run(gpu_api, m, n, k, a=a, b=b, out=out)
        run(gpu_api, m, n, k, VEC, VEC, a=a, b=b, out=out)


@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
@pytest.mark.parametrize("bias", [0, 1])
def test_epilogues(gpu_api, act, bias):
    for m, n, k in ((136, 2, 272), (300, 70, 528), (512, 300, 1024)):
        for kw in (dict(), dict(out="f16", alpha=0.5), dict(row_major=True), dict(beta=0.5), dict(out="f32", d_scale=3.0), dict(bias_type=1, a_mode=VEC)):
            run(gpu_api, m, n, k, act=act, bias=bias, **kw)


@pytest.mark.parametrize("akc,bkc", [(True, False), (False, True), (False, False)])
def test_other_layouts(gpu_api, akc, bkc):
    run(gpu_api, 100, 37, 300, akc=akc, bkc=bkc)
    run(gpu_api, 256, 128, 256, VEC, VEC, akc=akc, bkc=bkc, row_major=True)


@pytest.mark.parametrize("pad,skip,k", [(16, 16, 512), (4, 0, 512), (1, 3, 512), (0, 0, 509), (0, 0, 520)])
def test_any_alignment(gpu_api, pad, skip, k):
    run(gpu_api, 200, 70, k, pad=pad, skip=skip)
    run(gpu_api, 200, 1, k, VEC, VEC, pad=pad, skip=skip)


def test_batches(gpu_api):
    for m, n, k in ((200, 3, 400), (264, 140, 272), (512, 512, 256)):
        for modes in ((BLK, VEC), (VEC, VEC), (VEC, BLK)):
            run(gpu_api, m, n, k, *modes, batch=3)


def test_rows_of_nan_scales_stay_where_they_are(gpu_api):
    """a NaN or an infinity in one row's scales, or one code, is no other row's business"""
    m, n, k = 264, 70, 400
    A, B = Operand(m, k, "e4m3", VEC, 1), Operand(n, k, "e4m3", VEC, 2)
    B.scales[0, 1, 5] = float("nan")
    A.scales[0, 2, 7] = float("inf")
    B.raw[256 + 9 * k + 3] = 0x7F
    D = torch.zeros((n, m), dtype=torch.bfloat16, device=DEV)
    call = cublaslt.MatmulCall(gpu_api, dict(m=m, n=n, k=k, a_type=F8["e4m3"][1], b_type=F8["e4m3"][1], d_type=K.CUDA_R_16BF, compute_type=K.CUBLAS_COMPUTE_32F, scale_type=K.CUDA_R_32F,
                                             transa=K.CUBLAS_OP_T, a_scale_mode=VEC, b_scale_mode=VEC))
    call.set_pointers(a_scale=A.scales.data_ptr(), b_scale=B.scales.data_ptr())
    assert call.run(C.c_float(1), A.ptr, B.ptr, C.c_float(0), D.data_ptr(), D.data_ptr(), None, 0, stream()) == 0
    torch.cuda.synchronize()
    call.close()
    v, e = P.scaled_product(B.codes[0], A.codes[0], B.spread[0], A.spread[0])
    assert torch.isnan(D[5]).all() and torch.isnan(D[9]).all() and not torch.isfinite(D[:, 7]).any()
    keep_q, keep_p = [i for i in range(n) if i not in (5, 9)], [i for i in range(m) if i != 7]
    O.check(D[keep_q][:, keep_p], (v[keep_q][:, keep_p], e[keep_q][:, keep_p]))


def test_refusals(gpu_api):
    """one operand alone, integers, 16-bit types, other matrices' modes, a scale pointer that is missing or misaligned"""
    base = dict(m=64, n=64, k=128, a_type=K.CUDA_R_8F_E4M3, b_type=K.CUDA_R_8F_E4M3, d_type=K.CUDA_R_16BF, compute_type=K.CUBLAS_COMPUTE_32F, scale_type=K.CUDA_R_32F,
                transa=K.CUBLAS_OP_T)
    for over in (dict(a_scale_mode=VEC), dict(b_scale_mode=BLK), dict(a_scale_mode=VEC, b_scale_mode=K.CUBLASLT_MATMUL_MATRIX_SCALE_OUTER_VEC_32F),
                 dict(a_scale_mode=VEC, b_scale_mode=VEC, a_type=K.CUDA_R_16BF, b_type=K.CUDA_R_16BF),
                 dict(a_scale_mode=VEC, b_scale_mode=VEC, a_type=K.CUDA_R_8I, b_type=K.CUDA_R_8I, compute_type=K.CUBLAS_COMPUTE_32I),
                 dict(a_scale_mode=VEC, b_scale_mode=VEC, epilogue=K.CUBLASLT_EPILOGUE_BGRADA)):
        with pytest.raises(cublaslt.CublasLtError):
            cublaslt.MatmulCall(gpu_api, dict(base, **over))
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device=DEV)
    call = cublaslt.MatmulCall(gpu_api, dict(base, a_scale_mode=VEC, b_scale_mode=VEC))
    args = (C.c_float(1), buf.data_ptr(), buf.data_ptr(), C.c_float(0), buf.data_ptr(), buf.data_ptr(), None, 0, stream())
    call.set_pointers(a_scale=buf.data_ptr())
    assert call.run(*args) == K.CUBLAS_STATUS_INVALID_VALUE
    call.set_pointers(b_scale=buf.data_ptr() + 2)
    assert call.run(*args) == K.CUBLAS_STATUS_INVALID_VALUE
    call.close()
