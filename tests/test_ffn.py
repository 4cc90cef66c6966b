"""The feed-forward operators without a GPU: exports, structures, what is refused before anything is launched, workspace sizes, and
the 64-bit definitions that the GPU tests compare with."""
import ctypes as C
import os
import re
import subprocess
import tempfile

import pytest
import torch

import ffn_oracle as O
from zluda_amd import abi, cublaslt, ffn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
IV, NS, NOMEM, NOINIT = (abi.CUBLAS_STATUS_INVALID_VALUE, abi.CUBLAS_STATUS_NOT_SUPPORTED, abi.CUBLAS_STATUS_ALLOC_FAILED, abi.CUBLAS_STATUS_NOT_INITIALIZED)
BF, F16, F32, E4 = abi.CUDA_R_16BF, abi.CUDA_R_16F, abi.CUDA_R_32F, abi.CUDA_R_8F_E4M3


def test_every_declared_symbol_is_exported(api):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "zluda_ffn.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(zluda_ffn_\w+)\s*\(", text))
    assert names == set(ffn.SIGNATURES)
    for n in names:
        assert hasattr(api.lib, n), n


def test_structures_have_the_header_s_sizes():
    """the ctypes mirror against a C compiler"""
    structs = {n: getattr(ffn, n) for n in ("zluda_ffn_matrix", "zluda_ffn_gated", "zluda_ffn_gated_grad", "zluda_ffn_norm", "zluda_ffn_norm_grad")}
    with tempfile.TemporaryDirectory() as tmp:
        src = os.path.join(tmp, "s.c")
        lines = ["%s %s" % (n, f[0]) for n, s in structs.items() for f in s._fields_]
        with open(src, "w") as f:
            f.write('#include "zluda_ffn.h"\n#include <stdio.h>\nint main(void) {\n' + "".join(
                'printf("%%zu\\n", sizeof(%s));\n' % n for n in structs) + "".join('printf("%%zu\\n", offsetof(%s, %s));\n' % tuple(x.split()) for x in lines) + "return 0; }\n")
        exe = os.path.join(tmp, "s")
        subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    want = [C.sizeof(s) for s in structs.values()] + [getattr(s, f[0]).offset for s in structs.values() for f in s._fields_]
    assert got == want


def forward(**over):
    p = ffn.zluda_ffn_gated(0, 4, 64, 32)
    M = ffn.zluda_ffn_matrix
    p.x, p.w, p.h = M(256, None, 32, 0, BF), M(512, None, 32, 0, BF), M(1024, None, 64, 0, BF)
    return _with(p, over)


def backward(**over):
    p = ffn.zluda_ffn_gated_grad(0, 4, 64, 32)
    M = ffn.zluda_ffn_matrix
    p.dh, p.gate, p.up, p.x, p.w = (M(256 * (i + 1), None, n, 0, BF) for i, n in enumerate((64, 64, 64, 32, 32)))
    p.dx, p.dw = M(8192, None, 32, 0, BF), M(16384, None, 32, 0, BF)
    return _with(p, over)


def norm(**over):
    p = ffn.zluda_ffn_norm(4, 64, 1e-5, BF)
    p.x, p.y = ffn.zluda_ffn_matrix(256, None, 64, 0, BF), ffn.zluda_ffn_matrix(512, None, 64, 0, BF)
    return _with(p, over)


def norm_grad(**over):
    p = ffn.zluda_ffn_norm_grad(4, 64, BF)
    M = ffn.zluda_ffn_matrix
    p.x, p.dy, p.dx = M(256, None, 64, 0, BF), M(512, None, 64, 0, BF), M(1024, None, 64, 0, BF)
    p.mean, p.rstd, p.dweight, p.dbias = 4096, 8192, 16384, 32768
    return _with(p, over)


def _with(p, over):
    for path, v in over.items():
        at = p
        *inner, last = path.split("__")
        for name in inner:
            at = getattr(at, name)
        setattr(at, last, v)
    return p


REFUSED = [
    ("gated_forward", forward, dict(activation=3), IV), ("gated_forward", forward, dict(features=0), IV), ("gated_forward", forward, dict(model=0), IV),
    ("gated_forward", forward, dict(x__type=F32), NS), ("gated_forward", forward, dict(x__type=E4), NS), ("gated_forward", forward, dict(w__type=F16), NS),
    ("gated_forward", forward, dict(x__data=None), IV), ("gated_forward", forward, dict(w__data=None), IV), ("gated_forward", forward, dict(h__data=None), IV),
    ("gated_forward", forward, dict(x__ld=31), IV), ("gated_forward", forward, dict(w__ld=31), IV), ("gated_forward", forward, dict(h__ld=63), IV),
    ("gated_forward", forward, dict(x__data=257), IV), ("gated_forward", forward, dict(bias=3), IV), ("gated_forward", forward, dict(gate__data=64), IV),
    ("gated_forward", forward, dict(tokens=1 << 31), NS), ("gated_forward", forward, dict(features=1 << 31), NS), ("gated_forward", forward, dict(features=(1 << 20) + 1), NS),
    ("gated_forward", forward, dict(gate__data=64, gate__type=BF, gate__ld=64, up__data=64, up__type=E4, up__ld=64, up__scales=64, up__ld_scales=2), NS),
    ("gated_forward", forward, dict(gate__data=64, gate__type=F32, gate__ld=64, up__data=64, up__type=F32, up__ld=64), NS),
    ("gated_forward", forward, dict(gate__data=64, gate__type=E4, gate__ld=64, gate__scales=1, gate__ld_scales=2, up__data=64, up__type=E4, up__ld=64, up__ld_scales=2), IV),
    ("gated_forward", forward, dict(gate__data=64, gate__type=E4, gate__ld=80, gate__scales=1, gate__ld_scales=2, up__data=64, up__type=E4, up__ld=64, up__scales=1, up__ld_scales=2), IV),
    ("gated_forward", forward, dict(gate__data=64, gate__type=E4, gate__ld=64, gate__scales=1, gate__ld_scales=1, up__data=64, up__type=E4, up__ld=64, up__scales=1, up__ld_scales=2), IV),
    ("gated_forward", forward, dict(gate__data=72, gate__type=E4, gate__ld=64, gate__scales=1, gate__ld_scales=2, up__data=64, up__type=E4, up__ld=64, up__scales=1, up__ld_scales=2), IV),
    ("gated_backward", backward, dict(activation=7), IV), ("gated_backward", backward, dict(dh__data=None), IV), ("gated_backward", backward, dict(gate__data=None), IV),
    ("gated_backward", backward, dict(up__type=F16), NS), ("gated_backward", backward, dict(dh__type=F32), NS), ("gated_backward", backward, dict(w__data=None), IV),
    ("gated_backward", backward, dict(x__data=None), IV), ("gated_backward", backward, dict(dx__ld=31), IV), ("gated_backward", backward, dict(dw__ld=31), IV),
    ("gated_backward", backward, dict(dw__type=F32), NS), ("gated_backward", backward, dict(x__type=E4, x__ld=32), IV), ("gated_backward", backward, dict(dbias=1), IV),
    ("gated_backward", backward, dict(dz__data=64, dz__type=BF, dz__ld=127), IV), ("gated_backward", backward, dict(h__data=64, h__type=BF, h__ld=63), IV),
    ("norm_forward", norm, dict(cols=0), IV), ("norm_forward", norm, dict(cols=16385, x__ld=16385, y__ld=16385), NS), ("norm_forward", norm, dict(x__type=E4), NS),
    ("norm_forward", norm, dict(weight_type=F16), NS), ("norm_forward", norm, dict(x__data=None), IV), ("norm_forward", norm, dict(y__data=None), IV),
    ("norm_forward", norm, dict(y__type=F32), NS), ("norm_forward", norm, dict(x__ld=63), IV), ("norm_forward", norm, dict(mean=2), IV), ("norm_forward", norm, dict(weight=1), IV),
    ("norm_forward", norm, dict(kept__data=64, kept__type=BF, kept__ld=64), NS), ("norm_forward", norm, dict(kept__data=64, kept__type=E4, kept__ld=64, kept__ld_scales=2), IV),
    ("norm_backward", norm_grad, dict(cols=0), IV), ("norm_backward", norm_grad, dict(cols=20000), NS), ("norm_backward", norm_grad, dict(mean=None), IV),
    ("norm_backward", norm_grad, dict(dbias=None), IV), ("norm_backward", norm_grad, dict(dx__data=None, dweight=None, dbias=None), IV),
    ("norm_backward", norm_grad, dict(add__data=64, add__type=BF, add__ld=63), IV), ("norm_backward", norm_grad, dict(dy__type=F16), NS), ("norm_backward", norm_grad, dict(weight_type=F16), NS),
]


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_refusals(i):
    name, make, over, want = REFUSED[i]
    lib = ffn.load()
    p = make(**over)
    args = (C.byref(p), None) if name == "norm_forward" else (C.byref(p), 1 << 20, 1 << 40, None)
    assert getattr(lib, "zluda_ffn_" + name)(*args) == want, REFUSED[i]


def test_null_structures_and_small_workspaces():
    lib = ffn.load()
    n = C.c_size_t()
    assert lib.zluda_ffn_gated_forward(None, None, 0, None) == IV and lib.zluda_ffn_gated_backward(None, None, 0, None) == IV
    assert lib.zluda_ffn_norm_forward(None, None) == IV and lib.zluda_ffn_norm_backward(None, None, 0, None) == IV
    assert lib.zluda_ffn_gated_backward_workspace(None, C.byref(n)) == IV and lib.zluda_ffn_gated_forward_workspace(C.byref(forward()), None) == IV
    p = backward()
    assert lib.zluda_ffn_gated_backward_workspace(C.byref(p), C.byref(n)) == 0 and n.value > 4 * 128 * 2
    assert lib.zluda_ffn_gated_backward(C.byref(p), 1 << 20, n.value - 1, None) == NOMEM
    assert lib.zluda_ffn_gated_backward(C.byref(p), None, n.value, None) == NOMEM
    assert lib.zluda_ffn_gated_backward(C.byref(p), (1 << 20) + 8, n.value, None) == IV
    q = norm_grad(rows=1)
    assert lib.zluda_ffn_norm_backward_workspace(C.byref(q), C.byref(n)) == 0 and n.value == 0      # one workgroup: no partial sums
    q = norm_grad(rows=4000)
    assert lib.zluda_ffn_norm_backward_workspace(C.byref(q), C.byref(n)) == 0 and n.value >= 2 * 64 * 4
    assert lib.zluda_ffn_norm_backward(C.byref(q), 1 << 20, n.value - 1, None) == NOMEM
    M = ffn.zluda_ffn_matrix
    x, c = M(256, None, 64, 0, BF), M(512, 1024, 64, 2, E4)
    store = lib.zluda_ffn_checkpoint_store
    assert store(4, 64, None, C.byref(c), None) == IV and store(4, 0, C.byref(x), C.byref(c), None) == IV
    assert store(4, 64, C.byref(c), C.byref(x), None) == NS and store(4, 65, C.byref(x), C.byref(c), None) == IV
    assert store(0, 64, C.byref(x), C.byref(c), None) == 0


def test_calls_without_a_device_say_so(api):
    if torch.cuda.is_available():
        pytest.skip("there is a device")
    lib = ffn.load()
    assert lib.zluda_ffn_gated_forward(C.byref(forward()), None, 0, None) == NOINIT
    assert lib.zluda_ffn_gated_backward(C.byref(backward()), 1 << 20, 1 << 40, None) == NOINIT
    assert lib.zluda_ffn_norm_forward(C.byref(norm()), None) == NOINIT
    assert lib.zluda_ffn_norm_backward(C.byref(norm_grad()), 1 << 20, 1 << 40, None) == NOINIT
    with pytest.raises(cublaslt.CublasLtError):
        ffn.Checkpoint(dict(type=BF, rows=4, cols=64)).store(x=256, codes=512, scales=1024)


@pytest.mark.parametrize("act", O.ACTS)
def test_the_oracle_s_gated_gradient_against_autograd(act):
    torch.manual_seed(1)
    x, w, dh = torch.randn(5, 7, dtype=torch.float64), torch.randn(12, 7, dtype=torch.float64), torch.randn(5, 6, dtype=torch.float64)
    x.requires_grad_(), w.requires_grad_()
    z = x @ w.t()
    g = z[:, :6]
    a = {"silu": torch.nn.functional.silu(g), "gelu": torch.nn.functional.gelu(g, approximate="tanh"), "relu": g.relu()}[act]
    h = a * z[:, 6:]
    torch.autograd.backward(h, dh)
    assert torch.allclose(O.act(act, g.detach())[0], a.detach(), rtol=1e-12)
    with torch.no_grad():
        unit = dict(O.UNIT), dict(O.TINY)
        O.UNIT[torch.float64], O.TINY[torch.float64] = 0.0, 0.0
        try:
            out = O.gated_backward(act, dh, z[:, :6], z[:, 6:], x, w)
        finally:
            O.UNIT, O.TINY = unit
    assert torch.allclose(out["dx"][0], x.grad, rtol=1e-10) and torch.allclose(out["dw"][0], w.grad, rtol=1e-10)


def test_the_oracle_s_norm_gradient_against_autograd():
    torch.manual_seed(2)
    x, w, b = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((6, 50), (50,), (50,)))
    dy, add = torch.randn(6, 50, dtype=torch.float64), torch.randn(6, 50, dtype=torch.float64)
    y = torch.nn.functional.layer_norm(x, (50,), w, b, 1e-5)
    torch.autograd.backward(y, dy)
    with torch.no_grad():
        f = O.norm_forward(x, w, b, 1e-5)
        assert torch.allclose(f["y"][0], y, rtol=1e-10)
        o = O.norm_backward(x, dy, w, f["mean"][0], f["rstd"][0], add)
    assert torch.allclose(o["dx"][0], x.grad + add, rtol=1e-9) and torch.allclose(o["dweight"][0], w.grad, rtol=1e-9) and torch.allclose(o["dbias"][0], b.grad, rtol=1e-9)


def test_the_oracle_s_checkpoint_against_the_formats():
    """codes decode to the values, each the nearest of all 256 codes, ties to the even code; scales are minimal"""
    torch.manual_seed(3)
    x = torch.randn(40, 96) * torch.exp(3 * torch.randn(40, 1))
    x[0] = 0
    x[1, :32] = torch.arange(32) * 0.0625 + 1
    values, codes, scales = O.checkpoint(x)
    s = torch.ldexp(torch.ones((), dtype=torch.float64), scales.long() - 127).repeat_interleave(32, 1)
    assert torch.equal(codes.view(torch.float8_e4m3fn).double() * s, values)
    grid = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    grid = torch.where(torch.isnan(grid), torch.full_like(grid, 1e30), grid)
    dist = (x.double()[:, :, None] / s[:, :, None] - grid).abs()
    assert torch.equal((x.double() / s - codes.view(torch.float8_e4m3fn).double()).abs(), dist.amin(2))
    near = dist == dist.amin(2, keepdim=True)
    near[:, :, 128] |= near[:, :, 0]
    tie = (near[:, :, :128].sum(2) > 1) | (near[:, :, 129:].sum(2) > 1)
    assert tie.any() and (codes[tie] & 1 == 0).all()
    top = x.abs().double().reshape(40, 3, 32).amax(2)
    e = scales.double() - 127
    assert (top <= 448 * 2 ** e).all() and ((top > 448 * 2 ** (e - 1)) | (e == -126)).all()


def test_workspace_of_a_product_in_parts():
    """operands beyond 2 GiB: the 32-bit sum of dW comes on top, once; a pitch that no call takes is answered all the same"""
    lib = ffn.load()

    def bytes_of(**over):
        n = C.c_size_t()
        assert lib.zluda_ffn_gated_backward_workspace(C.byref(backward(**over)), C.byref(n)) == 0
        return n.value

    big = dict(tokens=40000, features=16384, model=2048, dz__data=64, dz__type=BF, dz__ld=32768, dx__ld=2048, dw__ld=2048, x__ld=2048, w__ld=2048, dh__ld=16384,
               gate__ld=16384, up__ld=16384)
    assert bytes_of(**big) - bytes_of(**dict(big, tokens=30000)) == 2 * 16384 * 2048 * 4
    assert bytes_of(**dict(big, dw__data=None)) == bytes_of(**dict(big, dw__data=None, tokens=30000))
    for ld in (0, -1, 1 << 62, -(1 << 63)):
        bytes_of(x__ld=ld, dz__data=64, dz__ld=ld)
