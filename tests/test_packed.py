"""RMS norm, packing and products grouped by expert without a GPU: structures, what is refused before anything is launched, workspaces; and the scale
modes for 128 of K in cublasLtMatmul's descriptors and planning."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

from zluda_amd import abi as K, cublaslt, ffn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
IV, NS, NOMEM, NOINIT = (K.CUBLAS_STATUS_INVALID_VALUE, K.CUBLAS_STATUS_NOT_SUPPORTED, K.CUBLAS_STATUS_ALLOC_FAILED, K.CUBLAS_STATUS_NOT_INITIALIZED)
BF, F16, F32, E4, E5 = K.CUDA_R_16BF, K.CUDA_R_16F, K.CUDA_R_32F, K.CUDA_R_8F_E4M3, K.CUDA_R_8F_E5M2
M = ffn.zluda_ffn_matrix


def test_structures_have_the_header_s_sizes():
    """the ctypes mirror against a C compiler"""
    structs = {n: getattr(ffn, n) for n in ("zluda_ffn_rms", "zluda_ffn_rms_grad", "zluda_ffn_activation", "zluda_ffn_grouped", "zluda_ffn_grouped_grad")}
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = os.path.join(tmp, "s.c"), os.path.join(tmp, "s")
        with open(src, "w") as f:
            f.write('#include "zluda_ffn.h"\n#include <stdio.h>\nint main(void) {\n')
            for n, s in structs.items():
                f.write('printf("%%zu\\n", sizeof(%s));\n' % n + "".join('printf("%%zu\\n", offsetof(%s, %s));\n' % (n, m[0]) for m in s._fields_))
            f.write("return 0; }\n")
        subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [v for s in structs.values() for v in [C.sizeof(s)] + [getattr(s, m[0]).offset for m in s._fields_]]


def _with(p, over):
    for path, v in over.items():
        at = p
        *inner, last = path.split("__")
        for name in inner:
            at = getattr(at, name)
        setattr(at, last, v)
    return p


def rms(**over):
    p = ffn.zluda_ffn_rms(4, 64, 1e-5, BF)
    p.x, p.residual, p.sum, p.y, p.packed = M(256, None, 64, 0, BF), M(1024, None, 64, 0, BF), M(2048, None, 64, 0, BF), M(4096, None, 64, 0, BF), M(8192, 8448, 64, 4, E4)
    return _with(p, over)


def rms_grad(**over):
    p = ffn.zluda_ffn_rms_grad(4, 64, BF)
    p.h, p.dy, p.dx = M(256, None, 64, 0, BF), M(1024, None, 64, 0, BF), M(2048, None, 64, 0, BF)
    p.rstd, p.dweight = 4096, 8192
    return _with(p, over)


def activation(**over):
    p = ffn.zluda_ffn_activation(ffn.SILU, 1, 4, 200)
    p.gate, p.up, p.y, p.packed = M(256, None, 400, 0, BF), M(656, None, 400, 0, BF), M(8192, None, 200, 0, BF), M(16384, 32768, 200, 4, E4)
    return _with(p, over)


def grouped(**over):
    p = ffn.zluda_ffn_grouped(10, 3, 200, 300, 64)
    p.x, p.w, p.y = M(256, None, 300, 0, BF), M(8192, None, 300, 0, BF), M(1 << 20, None, 200, 0, BF)
    return _with(p, over)


def grouped8(**over):
    p = grouped()
    p.x, p.w = M(256, 1 << 16, 300, 10, E4), M(8192, 1 << 17, 300, 3, E4)
    return _with(p, over)


def grouped_grad(**over):
    p = ffn.zluda_ffn_grouped_grad(10, 3, 200, 300, 64)
    p.dy, p.x, p.w, p.dx, p.dw = M(256, None, 200, 0, BF), M(8192, None, 300, 0, BF), M(1 << 16, None, 300, 0, BF), M(1 << 20, None, 300, 0, BF), M(1 << 21, None, 300, 0, BF)
    return _with(p, over)


REFUSED = [
    ("rms_forward", rms, dict(cols=0), IV), ("rms_forward", rms, dict(cols=16385), NS), ("rms_forward", rms, dict(x__type=E4), NS), ("rms_forward", rms, dict(weight_type=F16), NS),
    ("rms_forward", rms, dict(x__data=None), IV), ("rms_forward", rms, dict(x__data=257), IV), ("rms_forward", rms, dict(x__ld=63), IV), ("rms_forward", rms, dict(residual__type=F16), NS),
    ("rms_forward", rms, dict(residual__ld=63), IV), ("rms_forward", rms, dict(sum__ld=63), IV), ("rms_forward", rms, dict(y__type=F32), NS), ("rms_forward", rms, dict(packed__type=E5), NS),
    ("rms_forward", rms, dict(packed__scales=None), IV), ("rms_forward", rms, dict(packed__scales=8449), IV), ("rms_forward", rms, dict(packed__ld=63), IV),
    ("rms_forward", rms, dict(packed__ld_scales=3), IV), ("rms_forward", rms, dict(sum__data=None, y__data=None, packed__data=None), IV), ("rms_forward", rms, dict(sum__data=4096), IV),
    ("rms_forward", rms, dict(weight=1), IV), ("rms_forward", rms, dict(rstd=2), IV),
    ("rms_backward", rms_grad, dict(cols=0), IV), ("rms_backward", rms_grad, dict(cols=20000), NS), ("rms_backward", rms_grad, dict(h__data=None), IV), ("rms_backward", rms_grad, dict(h__type=E4), NS),
    ("rms_backward", rms_grad, dict(dy__type=F16), NS), ("rms_backward", rms_grad, dict(rstd=None), IV), ("rms_backward", rms_grad, dict(rstd=6), IV),
    ("rms_backward", rms_grad, dict(dx__data=None, dweight=None), IV), ("rms_backward", rms_grad, dict(add__data=64, add__type=BF, add__ld=63), IV), ("rms_backward", rms_grad, dict(dweight=1), IV),
    ("activate", activation, dict(activation=4), IV), ("activate", activation, dict(activation=ffn.COPY), IV), ("activate", activation, dict(block_rows=0), IV),
    ("activate", activation, dict(block_rows=64), IV), ("activate", activation, dict(cols=0), IV), ("activate", activation, dict(gate__type=E4), NS), ("activate", activation, dict(up__type=F16), NS),
    ("activate", activation, dict(gate__data=None), IV), ("activate", activation, dict(gate__ld=199), IV), ("activate", activation, dict(up__ld=199), IV), ("activate", activation, dict(y__ld=199), IV),
    ("activate", activation, dict(y__data=None, packed__data=None), IV), ("activate", activation, dict(packed__ld_scales=3), IV), ("activate", activation, dict(packed__ld=199), IV),
    ("activate", activation, dict(block_rows=128, packed__ld_scales=1), IV), ("activate", activation, dict(rows=1 << 63), NS), ("activate", activation, dict(cols=1 << 31), NS),
    ("grouped_forward", grouped, dict(offsets=None), IV), ("grouped_forward", grouped, dict(offsets=66), IV), ("grouped_forward", grouped, dict(experts=0), IV),
    ("grouped_forward", grouped, dict(experts=4097), NS), ("grouped_forward", grouped, dict(features=0), IV), ("grouped_forward", grouped, dict(model=0), IV),
    ("grouped_forward", grouped, dict(features=(1 << 20) + 1), NS), ("grouped_forward", grouped, dict(rows=1 << 31), NS), ("grouped_forward", grouped, dict(x__type=F32), NS),
    ("grouped_forward", grouped, dict(w__type=F16), NS), ("grouped_forward", grouped, dict(y__type=F32), NS), ("grouped_forward", grouped, dict(x__ld=299), IV), ("grouped_forward", grouped, dict(w__ld=299), IV),
    ("grouped_forward", grouped, dict(y__ld=199), IV), ("grouped_forward", grouped, dict(x__data=None), IV), ("grouped_forward", grouped, dict(w__data=None), IV),
    ("grouped_forward", grouped, dict(y__data=None), IV), ("grouped_forward", grouped, dict(y__data=257), IV),
    ("grouped_forward", grouped8, dict(x__scales=None), IV), ("grouped_forward", grouped8, dict(x__ld_scales=9), IV), ("grouped_forward", grouped8, dict(w__scales=None), IV),
    ("grouped_forward", grouped8, dict(w__ld_scales=2), IV), ("grouped_forward", grouped8, dict(w__type=BF), NS), ("grouped_forward", grouped8, dict(y__type=E4), NS),
    ("grouped_forward", grouped8, dict(w__scales=66), IV),
    ("grouped_backward", grouped_grad, dict(offsets=None), IV), ("grouped_backward", grouped_grad, dict(dy__type=E4), NS), ("grouped_backward", grouped_grad, dict(x__type=F16), NS),
    ("grouped_backward", grouped_grad, dict(w__data=None), IV), ("grouped_backward", grouped_grad, dict(x__data=None), IV), ("grouped_backward", grouped_grad, dict(dx__ld=299), IV),
    ("grouped_backward", grouped_grad, dict(dw__ld=299), IV), ("grouped_backward", grouped_grad, dict(dx__data=None, dw__data=None), IV), ("grouped_backward", grouped_grad, dict(dw__type=F32), NS),
]


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_refusals(i):
    name, make, over, want = REFUSED[i]
    p = make(**over)
    args = (C.byref(p), None) if name in ("rms_forward", "activate") else (C.byref(p), 1 << 20, 1 << 40, None)
    assert getattr(ffn.load(), "zluda_ffn_" + name)(*args) == want, REFUSED[i]


def test_null_structures_and_small_workspaces():
    lib, n = ffn.load(), C.c_size_t()
    assert lib.zluda_ffn_rms_forward(None, None) == IV and lib.zluda_ffn_rms_backward(None, None, 0, None) == IV and lib.zluda_ffn_activate(None, None) == IV
    assert lib.zluda_ffn_grouped_forward(None, None, 0, None) == IV and lib.zluda_ffn_grouped_backward(None, None, 0, None) == IV
    for fn, make in (("rms_backward", rms_grad), ("grouped_forward", grouped), ("grouped_backward", grouped_grad)):
        query = getattr(lib, "zluda_ffn_" + fn + "_workspace")
        assert query(None, C.byref(n)) == IV and query(C.byref(make()), None) == IV
    q = rms_grad(rows=1)
    assert lib.zluda_ffn_rms_backward_workspace(C.byref(q), C.byref(n)) == 0 and n.value == 0      # one workgroup: no partial sums
    q = rms_grad(rows=4000)
    assert lib.zluda_ffn_rms_backward_workspace(C.byref(q), C.byref(n)) == 0 and n.value >= 64 * 4
    assert lib.zluda_ffn_rms_backward(C.byref(q), 1 << 20, n.value - 1, None) == NOMEM and lib.zluda_ffn_rms_backward(C.byref(q), None, n.value, None) == NOMEM
    assert lib.zluda_ffn_rms_backward(C.byref(q), (1 << 20) + 8, n.value, None) == IV
    x, c = M(256, None, 64, 0, BF), M(512, 1024, 64, 4, E4)
    un = lib.zluda_ffn_unpack
    assert un(4, 64, 1, None, C.byref(x), None) == IV and un(4, 0, 1, C.byref(c), C.byref(x), None) == IV and un(4, 64, 2, C.byref(c), C.byref(x), None) == IV
    assert un(4, 64, 1, C.byref(x), C.byref(x), None) == IV and un(4, 65, 1, C.byref(c), C.byref(x), None) == IV and un(5, 64, 1, C.byref(c), C.byref(x), None) == IV
    assert un(0, 64, 1, C.byref(c), C.byref(x), None) == 0


def test_calls_without_a_device_say_so(api):
    if torch.cuda.is_available():
        pytest.skip("there is a device")
    lib = ffn.load()
    assert lib.zluda_ffn_rms_forward(C.byref(rms()), None) == NOINIT and lib.zluda_ffn_activate(C.byref(activation()), None) == NOINIT
    for make, fn in ((rms_grad, "rms_backward"), (grouped, "grouped_forward"), (grouped8, "grouped_forward"), (grouped_grad, "grouped_backward")):
        assert getattr(lib, "zluda_ffn_" + fn)(C.byref(make()), 1 << 20, 1 << 40, None) == NOINIT


def test_calls_of_no_rows_do_nothing(api):
    lib = ffn.load()
    assert lib.zluda_ffn_rms_forward(C.byref(rms(rows=0)), None) == 0 and lib.zluda_ffn_activate(C.byref(activation(rows=0)), None) == 0
    assert lib.zluda_ffn_grouped_forward(C.byref(grouped(rows=0)), None, 0, None) == 0


def test_pitches_are_those_of_the_matmul():
    assert ffn.packed_pitches(5, 300) == (304, 5) and ffn.packed_pitches(5, 300, 128) == (304, 4) and ffn.packed_pitches(300, 129, 128) == (144, 4)
    codes, scales = ffn.packed_buffers(300, 600, "cpu", 128)
    assert codes.shape == (300, 608) and scales.shape == (3, 8)
    codes, scales = ffn.packed_buffers(300, 600, "cpu")
    assert scales.shape == (5, 300)


VEC, BLK = K.CUBLASLT_MATMUL_MATRIX_SCALE_VEC128_32F, K.CUBLASLT_MATMUL_MATRIX_SCALE_BLK128x128_32F
BASE = dict(m=256, n=64, k=512, a_type=E4, b_type=E4, d_type=BF, compute_type=K.CUBLAS_COMPUTE_32F, scale_type=F32, transa=1)


def test_scale_modes_of_the_descriptor(api):
    desc, got, n = C.c_void_p(), C.c_int32(), C.c_size_t()
    assert api.cublasLtMatmulDescCreate(C.byref(desc), K.CUBLAS_COMPUTE_32F, F32) == 0
    for mode in (VEC, BLK):
        for attr in (K.CUBLASLT_MATMUL_DESC_A_SCALE_MODE, K.CUBLASLT_MATMUL_DESC_B_SCALE_MODE):
            assert api.desc_set(desc, attr, C.c_int32, mode) == 0
            assert api.cublasLtMatmulDescGetAttribute(desc, attr, C.byref(got), 4, C.byref(n)) == 0 and got.value == mode
        assert api.desc_set(desc, K.CUBLASLT_MATMUL_DESC_D_SCALE_MODE, C.c_int32, mode) == NS
    api.cublasLtMatmulDescDestroy(desc)


@pytest.mark.parametrize("over,ok", [(dict(), True), (dict(a_scale_mode=BLK), True), (dict(b_scale_mode=BLK), True), (dict(a_scale_mode=BLK, b_scale_mode=BLK), True), (dict(b_type=E5), True),
                                     (dict(k=500), True), (dict(transa=0), True), (dict(a_scale_mode=0), False),
                                     (dict(b_scale_mode=K.CUBLASLT_MATMUL_MATRIX_SCALE_VEC32_UE8M0), False), (dict(a_type=BF, b_type=BF), False),
                                     (dict(a_type=K.CUDA_R_8I, b_type=K.CUDA_R_8I, compute_type=K.CUBLAS_COMPUTE_32I), False),
                                     (dict(epilogue=K.CUBLASLT_EPILOGUE_BGRADB), False)])
def test_scale_modes_in_planning(api, over, ok):
    spec = dict(BASE, a_scale_mode=VEC, b_scale_mode=VEC)
    spec.update(over)
    if ok:
        cublaslt.MatmulCall(api, spec).close()
    else:
        with pytest.raises(cublaslt.CublasLtError):
            cublaslt.MatmulCall(api, spec)
