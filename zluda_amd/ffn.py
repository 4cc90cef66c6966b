"""ctypes binding of the feed-forward operators of libcublaslt.so (include/zluda_ffn.h): a gated feed-forward layer, layer norm, and
activation checkpoints in 8 bits.  As in cublaslt.py, device memory crosses the boundary as integer addresses.

A call object is configured once with a plain dict (types, sizes, pitches) and run with addresses:

  GatedForward   type, tokens, features, model; activation (SILU, GELU, RELU; default SILU), bias (bool), kept (KEPT_NONE, KEPT_PLAIN,
                 KEPT_8BIT); pitches in elements ldx, ldw, ldh, ldgate, ldup and for checkpoints ldgate_scales, ldup_scales
  GatedBackward  the same sizes and activation; bias (bool), kept and x_kept (KEPT_PLAIN or KEPT_8BIT: how the forward pass kept G and U, and x);
                 outputs, all wanted by default but the last two: dx, dw (bool), h, dz (bool)
  NormForward    type, weight_type (default: type), rows, cols, eps; kept (KEPT_NONE or KEPT_8BIT)
  NormBackward   the same; x_kept (KEPT_PLAIN or KEPT_8BIT), add (bool), weights (bool: dweight and dbias, default True)
  Checkpoint     type, rows, cols

A call object writes the addresses into its own structure and hands that to the library: one thread at a time may run it (several threads: an object each).
`workspace` is the number of bytes of device scratch that run() wants.  Pitches default to tight rows, those of checkpoints to what
checkpoint_buffers() makes: codes padded to 32 columns, one scale byte for each 32.  A status other than 0 raises CublasLtError.
"""
import ctypes as C

from . import abi, cublaslt

SILU, GELU, RELU = 0, 1, 2
KEPT_NONE, KEPT_PLAIN, KEPT_8BIT = 0, 1, 2
BLOCK = 32


class zluda_ffn_matrix(C.Structure):
    _fields_ = [("data", C.c_void_p), ("scales", C.c_void_p), ("ld", C.c_int64), ("ld_scales", C.c_int64), ("type", C.c_uint32)]


_M = zluda_ffn_matrix


class zluda_ffn_gated(C.Structure):
    _fields_ = [("activation", C.c_uint32), ("tokens", C.c_uint64), ("features", C.c_uint64), ("model", C.c_uint64),
                ("x", _M), ("w", _M), ("h", _M), ("gate", _M), ("up", _M), ("bias", C.c_void_p)]


class zluda_ffn_gated_grad(C.Structure):
    _fields_ = [("activation", C.c_uint32), ("tokens", C.c_uint64), ("features", C.c_uint64), ("model", C.c_uint64),
                ("dh", _M), ("gate", _M), ("up", _M), ("x", _M), ("w", _M), ("dx", _M), ("dw", _M), ("h", _M), ("dz", _M), ("dbias", C.c_void_p)]


class zluda_ffn_norm(C.Structure):
    _fields_ = [("rows", C.c_uint64), ("cols", C.c_uint64), ("eps", C.c_float), ("weight_type", C.c_uint32),
                ("x", _M), ("y", _M), ("kept", _M), ("weight", C.c_void_p), ("bias", C.c_void_p), ("mean", C.c_void_p), ("rstd", C.c_void_p)]


class zluda_ffn_norm_grad(C.Structure):
    _fields_ = [("rows", C.c_uint64), ("cols", C.c_uint64), ("weight_type", C.c_uint32), ("x", _M), ("dy", _M), ("add", _M), ("dx", _M),
                ("weight", C.c_void_p), ("mean", C.c_void_p), ("rstd", C.c_void_p), ("dweight", C.c_void_p), ("dbias", C.c_void_p)]


_vp, _u32, _u64, _sz, _psz = C.c_void_p, C.c_uint32, C.c_uint64, C.c_size_t, C.POINTER(C.c_size_t)
SIGNATURES = {
    "zluda_ffn_gated_forward": (_u32, [C.POINTER(zluda_ffn_gated), _vp, _sz, _vp]),
    "zluda_ffn_gated_forward_workspace": (_u32, [C.POINTER(zluda_ffn_gated), _psz]),
    "zluda_ffn_gated_backward": (_u32, [C.POINTER(zluda_ffn_gated_grad), _vp, _sz, _vp]),
    "zluda_ffn_gated_backward_workspace": (_u32, [C.POINTER(zluda_ffn_gated_grad), _psz]),
    "zluda_ffn_norm_forward": (_u32, [C.POINTER(zluda_ffn_norm), _vp]),
    "zluda_ffn_norm_backward": (_u32, [C.POINTER(zluda_ffn_norm_grad), _vp, _sz, _vp]),
    "zluda_ffn_norm_backward_workspace": (_u32, [C.POINTER(zluda_ffn_norm_grad), _psz]),
    "zluda_ffn_checkpoint_store": (_u32, [_u64, _u64, C.POINTER(_M), C.POINTER(_M), _vp]),
    "zluda_ffn_checkpoint_load": (_u32, [_u64, _u64, C.POINTER(_M), C.POINTER(_M), _vp]),
}

_lib = None


def load():
    """The library with the operators' signatures (loads libcublaslt.so through cublaslt.load())."""
    global _lib
    if _lib is None:
        lib = cublaslt.load().lib
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _lib = lib
    return _lib


def _check(status, what):
    if status != abi.CUBLAS_STATUS_SUCCESS:
        raise cublaslt.CublasLtError(status, what)


# (A call's cost on the host is what the smallest problems wait for: the structures' members and the function are looked up once.)
def _members(p, names):
    return [getattr(p, n) for n in names.split()]


def checkpoint_pitches(cols):
    """(codes, scales) of a row of a checkpoint"""
    blocks = -(-cols // BLOCK)
    return blocks * BLOCK, blocks


def checkpoint_buffers(rows, cols, device):
    """(codes, scales): torch tensors for a checkpoint of rows x cols"""
    import torch
    ld, lds = checkpoint_pitches(cols)
    return torch.empty((rows, ld), dtype=torch.uint8, device=device), torch.empty((rows, lds), dtype=torch.uint8, device=device)


class _Call:
    """fills the structure's matrices from the spec; subclasses name them"""

    def __init__(self, spec):
        self.spec, self.lib, self.workspace = dict(spec), load(), 0

    def matrix(self, name, cols, type, kept=KEPT_PLAIN):
        m = getattr(self.p, name)
        if kept == KEPT_8BIT:
            ld, lds = checkpoint_pitches(cols)
            m.type, m.ld, m.ld_scales = abi.CUDA_R_8F_E4M3, self.spec.get("ld" + name, ld), self.spec.get("ld" + name + "_scales", lds)
        else:
            m.type, m.ld = type, self.spec.get("ld" + name, cols)

    def query(self, fn):
        n = C.c_size_t(0)
        _check(fn(C.byref(self.p), C.byref(n)), fn.__name__)
        self.workspace = n.value


class GatedForward(_Call):
    def __init__(self, spec):
        super().__init__(spec)
        s, self.p = self.spec, zluda_ffn_gated()
        p, t = self.p, s["type"]
        p.activation, p.tokens, p.features, p.model = s.get("activation", SILU), s["tokens"], s["features"], s["model"]
        self.matrix("x", p.model, t)
        self.matrix("w", p.model, t)
        self.matrix("h", p.features, t)
        for name in ("gate", "up"):
            self.matrix(name, p.features, t, s.get("kept", KEPT_NONE))
        self.query(self.lib.zluda_ffn_gated_forward_workspace)
        self._call, self._ref, self._m = self.lib.zluda_ffn_gated_forward, C.byref(p), _members(p, "x w h gate up")

    def run(self, x, w, h, bias=None, gate=None, gate_scales=None, up=None, up_scales=None, workspace=None, workspace_size=0, stream=None):
        mx, mw, mh, mg, mu = self._m
        mx.data, mw.data, mh.data, self.p.bias = x, w, h, bias
        mg.data, mg.scales, mu.data, mu.scales = gate, gate_scales, up, up_scales
        status = self._call(self._ref, workspace, workspace_size, stream)
        if status:
            _check(status, "zluda_ffn_gated_forward")


class GatedBackward(_Call):
    def __init__(self, spec):
        super().__init__(spec)
        s, self.p = self.spec, zluda_ffn_gated_grad()
        p, t = self.p, s["type"]
        p.activation, p.tokens, p.features, p.model = s.get("activation", SILU), s["tokens"], s["features"], s["model"]
        for name, cols in (("dh", p.features), ("w", p.model), ("dx", p.model), ("dw", p.model), ("h", p.features), ("dz", 2 * p.features)):
            self.matrix(name, cols, t)
        for name in ("gate", "up"):
            self.matrix(name, p.features, t, s.get("kept", KEPT_PLAIN))
        self.matrix("x", p.model, t, s.get("x_kept", KEPT_PLAIN))
        # the workspace depends on which matrices are there: any address stands for one that will be
        for name, default in (("dx", True), ("dw", True), ("h", False), ("dz", False)):
            getattr(p, name).data = 16 if s.get(name, default) else None
        p.dbias = 16 if s.get("bias", False) else None
        self.query(self.lib.zluda_ffn_gated_backward_workspace)
        self._call, self._ref, self._m = self.lib.zluda_ffn_gated_backward, C.byref(p), _members(p, "dh gate up x w dx dw h dz")

    def run(self, dh, gate, up, x=None, w=None, dx=None, dw=None, dbias=None, h=None, dz=None, gate_scales=None, up_scales=None, x_scales=None,
            workspace=None, workspace_size=0, stream=None):
        mdh, mg, mu, mx, mw, mdx, mdw, mh, mdz = self._m
        mdh.data, mg.data, mg.scales, mu.data, mu.scales, mx.data, mx.scales, mw.data = dh, gate, gate_scales, up, up_scales, x, x_scales, w
        mdx.data, mdw.data, self.p.dbias, mh.data, mdz.data = dx, dw, dbias, h, dz
        status = self._call(self._ref, workspace, workspace_size, stream)
        if status:
            _check(status, "zluda_ffn_gated_backward")


class NormForward(_Call):
    def __init__(self, spec):
        super().__init__(spec)
        s, self.p = self.spec, zluda_ffn_norm()
        p, t = self.p, s["type"]
        p.rows, p.cols, p.eps, p.weight_type = s["rows"], s["cols"], s.get("eps", 1e-5), s.get("weight_type", t)
        self.matrix("x", p.cols, t)
        self.matrix("y", p.cols, t)
        self.matrix("kept", p.cols, t, KEPT_8BIT)
        self._call, self._ref, self._m = self.lib.zluda_ffn_norm_forward, C.byref(p), _members(p, "x y kept")

    def run(self, x, y, weight=None, bias=None, mean=None, rstd=None, kept=None, kept_scales=None, stream=None):
        p, (mx, my, mk) = self.p, self._m
        mx.data, my.data, p.weight, p.bias, p.mean, p.rstd, mk.data = x, y, weight, bias, mean, rstd, kept
        if kept is not None:
            mk.scales = kept_scales
        status = self._call(self._ref, stream)
        if status:
            _check(status, "zluda_ffn_norm_forward")


class NormBackward(_Call):
    def __init__(self, spec):
        super().__init__(spec)
        s, self.p = self.spec, zluda_ffn_norm_grad()
        p, t = self.p, s["type"]
        p.rows, p.cols, p.weight_type = s["rows"], s["cols"], s.get("weight_type", t)
        self.matrix("x", p.cols, t, s.get("x_kept", KEPT_PLAIN))
        for name in ("dy", "add", "dx"):
            self.matrix(name, p.cols, t)
        p.dweight = p.dbias = 16 if s.get("weights", True) else None
        self.query(self.lib.zluda_ffn_norm_backward_workspace)
        self._call, self._ref, self._m = self.lib.zluda_ffn_norm_backward, C.byref(p), _members(p, "x dy add dx")

    def run(self, x, dy, mean, rstd, weight=None, add=None, dx=None, dweight=None, dbias=None, x_scales=None, workspace=None, workspace_size=0, stream=None):
        p, (mx, my, ma, md) = self.p, self._m
        mx.data, mx.scales, my.data, ma.data, md.data = x, x_scales, dy, add, dx
        p.weight, p.mean, p.rstd, p.dweight, p.dbias = weight, mean, rstd, dweight, dbias
        status = self._call(self._ref, workspace, workspace_size, stream)
        if status:
            _check(status, "zluda_ffn_norm_backward")


class Checkpoint(_Call):
    def __init__(self, spec):
        super().__init__(spec)
        s = self.spec
        self.rows, self.cols = s["rows"], s["cols"]
        ld, lds = checkpoint_pitches(self.cols)
        self.x = _M(None, None, s.get("ldx", self.cols), 0, s["type"])
        self.c = _M(None, None, s.get("ldcodes", ld), s.get("ldscales", lds), abi.CUDA_R_8F_E4M3)
        self._store, self._load, self._refs = self.lib.zluda_ffn_checkpoint_store, self.lib.zluda_ffn_checkpoint_load, (C.byref(self.x), C.byref(self.c))

    def store(self, x, codes, scales, stream=None):
        self.x.data, self.c.data, self.c.scales = x, codes, scales
        status = self._store(self.rows, self.cols, self._refs[0], self._refs[1], stream)
        if status:
            _check(status, "zluda_ffn_checkpoint_store")

    def load(self, codes, scales, x, stream=None):
        self.x.data, self.c.data, self.c.scales = x, codes, scales
        status = self._load(self.rows, self.cols, self._refs[1], self._refs[0], stream)
        if status:
            _check(status, "zluda_ffn_checkpoint_load")
