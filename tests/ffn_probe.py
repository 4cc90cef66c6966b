"""Builds and loads tests/host_c/ffn_probe.cpp: which kernel a feed-forward call takes on a chip of so many CUs."""
import ctypes as C
import functools
import os
import shutil
import subprocess
import tempfile

import pytest

from zluda_amd import abi, ffn

BASE = 1 << 40   # (an aligned address; nothing is read from it)
CUS = 256
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Gated(C.Structure):
    _fields_ = [("x", C.c_void_p), ("w", C.c_void_p), ("ldx", C.c_int64), ("ldw", C.c_int64), ("tokens", C.c_int32), ("features", C.c_int32), ("model", C.c_int32)]


@functools.lru_cache(None)
def load():
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    with tempfile.TemporaryDirectory() as d:
        so = os.path.join(d, "ffn_probe.so")
        subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-fvisibility=hidden", "-Wl,-Bsymbolic",
                        os.path.join(ROOT, "tests", "host_c", "ffn_probe.cpp"), "-o", so], check=True)
        lib = C.CDLL(so)
    lib.probe_max_side.restype = lib.probe_rows_in_window.restype = C.c_uint64
    lib.probe_column_strips.restype = lib.probe_grad_splits.restype = C.c_uint32
    lib.probe_column_strips.argtypes = [C.c_uint64]
    lib.probe_rows_in_window.argtypes = [C.c_uint64, C.c_int64]
    lib.probe_grad_largest_tiles.argtypes = [C.c_uint64] * 3
    lib.probe_grad_splits.argtypes = [C.POINTER(ffn.zluda_ffn_gated_grad), C.POINTER(ffn.zluda_ffn_matrix), C.c_int64, C.c_void_p, C.c_int, C.POINTER(C.c_uint32)]
    return lib


def gated_tile(tokens, model, features, pad=0, skip=0, cus=CUS):
    """index of the tile of a gated product, -1: at any alignment; rows `pad` elements longer, `skip` elements behind an aligned address"""
    g = Gated(BASE + 2 * skip, 2 * BASE + 2 * skip, model + pad, model + pad, tokens, features, model)
    return load().probe_gated_tile(C.byref(g), cus)


def tile_shape(tile):
    """features, tokens, whether it is the persistent kernel's"""
    f, t = C.c_int(), C.c_int()
    persistent = load().probe_gated_tile_shape(tile, C.byref(f), C.byref(t))
    return f.value, t.value, persistent == 1


def grad_splits(tokens, model, features, pad=0, skip=0, dz_ld=None, x_kept=False, cus=CUS):
    """(shares of dX's K in the launch that makes dX and dW, stages of a share); 0 shares: one after the other.  dz_ld: the caller's own [dG dU]"""
    p, M, bf = ffn.zluda_ffn_gated_grad(0, tokens, features, model), ffn.zluda_ffn_matrix, abi.CUDA_R_16BF
    for i, n in enumerate(("w", "dx", "dw", "x")):
        setattr(p, n, M((i + 1) * BASE + 2 * skip, None, model + pad, 0, bf))
    lines = lambda n: (n + 63) // 64 * 64  # noqa: E731
    x = M(BASE, None, lines(model), 0, bf) if x_kept else p.x
    stages = C.c_uint32()
    own = dz_ld is not None
    n = load().probe_grad_splits(C.byref(p), C.byref(x), dz_ld if own else lines(2 * features), 5 * BASE + 2 * skip * own, cus, C.byref(stages))
    return n, stages.value
