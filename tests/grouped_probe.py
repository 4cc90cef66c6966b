"""Builds and loads tests/host_c/grouped_probe.cpp: which tile a product by expert takes on a chip of so many CUs (operands on 16 bytes)."""
import ctypes as C
import functools
import os
import shutil
import subprocess
import tempfile

import pytest

from zluda_amd import abi as K, ffn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"bf16": K.CUDA_R_16BF, "f16": K.CUDA_R_16F, "f32": K.CUDA_R_32F}


@functools.lru_cache(None)
def load():
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    with tempfile.TemporaryDirectory() as d:
        so = os.path.join(d, "grouped_probe.so")
        subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-fvisibility=hidden", "-Wl,-Bsymbolic",
                        os.path.join(ROOT, "tests", "host_c", "grouped_probe.cpp"), "-o", so], check=True)
        lib = C.CDLL(so)
    lib.probe_grouped_tile.argtypes = [C.POINTER(ffn.zluda_ffn_grouped), C.c_uint64]
    return lib


def tiles():
    return load().probe_grouped_tiles()


def tile(kind, rows, experts, features, model, cus=256):
    """kind: the type of 16-bit operands, or "packed " and that of y"""
    p = ffn.zluda_ffn_grouped(rows, experts, features, model)
    packed, out = kind.startswith("packed"), TYPES[kind.split()[-1]]
    p.x.type = p.w.type = K.CUDA_R_8F_E4M3 if packed else out
    p.y.type = out
    return load().probe_grouped_tile(C.byref(p), cus)
