"""ctypes binding of the feed-forward operators of libcublaslt.so (include/zluda_ffn.h): a gated feed-forward layer, layer norm,
activation checkpoints in 8 bits, RMS norm, packing with scales for each 128, and products grouped by expert.  As in cublaslt.py, device memory
crosses the boundary as integer addresses.

A call object is configured once with a plain dict (types, sizes, pitches) and run with addresses:

  GatedForward   type, tokens, features, model; activation (SILU, GELU, RELU; default SILU), bias (bool), kept (KEPT_NONE, KEPT_PLAIN,
                 KEPT_8BIT); pitches in elements ldx, ldw, ldh, ldgate, ldup and for checkpoints ldgate_scales, ldup_scales
  GatedBackward  the same sizes and activation; bias (bool), kept and x_kept (KEPT_PLAIN or KEPT_8BIT: how the forward pass kept G and U, and x);
                 outputs, all wanted by default but the last two: dx, dw (bool), h, dz (bool)
  NormForward    type, weight_type (default: type), rows, cols, eps; kept (KEPT_NONE or KEPT_8BIT)
  NormBackward   the same; x_kept (KEPT_PLAIN or KEPT_8BIT), add (bool), weights (bool: dweight and dbias, default True)
  Checkpoint     type, rows, cols
  RmsForward     type, weight_type (default: type), rows, cols, eps; which of residual, sum, y, codes and scales (packed), rstd there are is
                 told by run()'s arguments
  RmsBackward    type, weight_type, rows, cols
  Activate       type, rows, cols; activation (SILU, GELU, RELU, COPY; default SILU), block_rows (1 or 128; default 1)
  Unpack         type, rows, cols; block_rows
  GroupedForward   type (of x, w and y; packed: of y), rows, experts, model, features; packed (bool)
  GroupedBackward  type, rows, experts, model, features; outputs, wanted by default: dx, dw (bool).  run() may leave one out; dx alone can take more scratch
                   than both of them do (its sums are shared out further): `workspace_dx` bytes

A call object writes the addresses into its own structure and hands that to the library: one thread at a time may run it (several threads: an object each).
`workspace` is the number of bytes of device scratch that run() wants.  Pitches default to tight rows, those of checkpoints to what
checkpoint_buffers() makes: codes padded to 32 columns, one scale byte for each 32; those of packed matrices to what packed_buffers() makes.  A status other than 0 raises CublasLtError.
"""
import ctypes as C

from . import abi, cublaslt

SILU, GELU, RELU, COPY = 0, 1, 2, 3
KEPT_NONE, KEPT_PLAIN, KEPT_8BIT = 0, 1, 2
BLOCK = 32
PACK = 128


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


class zluda_ffn_rms(C.Structure):
    _fields_ = [("rows", C.c_uint64), ("cols", C.c_uint64), ("eps", C.c_float), ("weight_type", C.c_uint32),
                ("x", _M), ("residual", _M), ("sum", _M), ("y", _M), ("packed", _M), ("weight", C.c_void_p), ("rstd", C.c_void_p)]


class zluda_ffn_rms_grad(C.Structure):
    _fields_ = [("rows", C.c_uint64), ("cols", C.c_uint64), ("weight_type", C.c_uint32), ("h", _M), ("dy", _M), ("add", _M), ("dx", _M),
                ("weight", C.c_void_p), ("rstd", C.c_void_p), ("dweight", C.c_void_p)]


class zluda_ffn_activation(C.Structure):
    _fields_ = [("activation", C.c_uint32), ("block_rows", C.c_uint32), ("rows", C.c_uint64), ("cols", C.c_uint64),
                ("gate", _M), ("up", _M), ("y", _M), ("packed", _M)]


class zluda_ffn_grouped(C.Structure):
    _fields_ = [("rows", C.c_uint64), ("experts", C.c_uint64), ("features", C.c_uint64), ("model", C.c_uint64), ("offsets", C.c_void_p),
                ("x", _M), ("w", _M), ("y", _M)]


class zluda_ffn_grouped_grad(C.Structure):
    _fields_ = [("rows", C.c_uint64), ("experts", C.c_uint64), ("features", C.c_uint64), ("model", C.c_uint64), ("offsets", C.c_void_p),
                ("dy", _M), ("x", _M), ("w", _M), ("dx", _M), ("dw", _M)]


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
    "zluda_ffn_rms_forward": (_u32, [C.POINTER(zluda_ffn_rms), _vp]),
    "zluda_ffn_rms_backward": (_u32, [C.POINTER(zluda_ffn_rms_grad), _vp, _sz, _vp]),
    "zluda_ffn_rms_backward_workspace": (_u32, [C.POINTER(zluda_ffn_rms_grad), _psz]),
    "zluda_ffn_activate": (_u32, [C.POINTER(zluda_ffn_activation), _vp]),
    "zluda_ffn_unpack": (_u32, [_u64, _u64, _u32, C.POINTER(_M), C.POINTER(_M), _vp]),
    "zluda_ffn_grouped_forward": (_u32, [C.POINTER(zluda_ffn_grouped), _vp, _sz, _vp]),
    "zluda_ffn_grouped_forward_workspace": (_u32, [C.POINTER(zluda_ffn_grouped), _psz]),
    "zluda_ffn_grouped_backward": (_u32, [C.POINTER(zluda_ffn_grouped_grad), _vp, _sz, _vp]),
    "zluda_ffn_grouped_backward_workspace": (_u32, [C.POINTER(zluda_ffn_grouped_grad), _psz]),
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


def packed_pitches(rows, cols, block_rows=1):
    """(codes of a row, scales): rows of codes on 16 bytes; scales in the layout of cublasLtMatmul's VEC128_32F or (block_rows 128) BLK128x128_32F"""
    blocks = -(-cols // PACK)
    return -(-cols // 16) * 16, rows if block_rows == 1 else -(-blocks // 4) * 4


def packed_buffers(rows, cols, device, block_rows=1):
    """(codes, scales): torch tensors for a packed matrix of rows x cols"""
    import torch
    ld, lds = packed_pitches(rows, cols, block_rows)
    lines = -(-cols // PACK) if block_rows == 1 else -(-rows // PACK)
    # (zeros: what pads the codes of a row, and the scales of a block row, is part of a matmul's operands but never written)
    return torch.zeros((rows, ld), dtype=torch.uint8, device=device), torch.zeros((lines, lds), dtype=torch.float32, device=device)


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

    def packed(self, m, name, rows, cols, block_rows=1):
        ld, lds = packed_pitches(rows, cols, block_rows)
        m.type, m.ld, m.ld_scales = abi.CUDA_R_8F_E4M3, self.spec.get("ld" + name, ld), self.spec.get("ld" + name + "_scales", lds)

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


class RmsForward(_Call):
    def __init__(self, spec):
        super().__init__(spec)
        s, self.p = self.spec, zluda_ffn_rms()
        p, t = self.p, s["type"]
        p.rows, p.cols, p.eps, p.weight_type = s["rows"], s["cols"], s.get("eps", 1e-5), s.get("weight_type", t)
        for name in ("x", "residual", "sum", "y"):
            self.matrix(name, p.cols, t)
        self.packed(p.packed, "codes", p.rows, p.cols)
        self._call, self._ref, self._m = self.lib.zluda_ffn_rms_forward, C.byref(p), _members(p, "x residual sum y packed")

    def run(self, x, weight=None, residual=None, sum=None, y=None, codes=None, scales=None, rstd=None, stream=None):
        p, (mx, mr, ms, my, mk) = self.p, self._m
        mx.data, mr.data, ms.data, my.data, mk.data, mk.scales, p.weight, p.rstd = x, residual, sum, y, codes, scales, weight, rstd
        status = self._call(self._ref, stream)
        if status:
            _check(status, "zluda_ffn_rms_forward")


class RmsBackward(_Call):
    def __init__(self, spec):
        super().__init__(spec)
        s, self.p = self.spec, zluda_ffn_rms_grad()
        p, t = self.p, s["type"]
        p.rows, p.cols, p.weight_type = s["rows"], s["cols"], s.get("weight_type", t)
        for name in ("h", "dy", "add", "dx"):
            self.matrix(name, p.cols, t)
        p.dweight = 16
        self.query(self.lib.zluda_ffn_rms_backward_workspace)
        self._call, self._ref, self._m = self.lib.zluda_ffn_rms_backward, C.byref(p), _members(p, "h dy add dx")

    def run(self, h, dy, rstd, weight=None, add=None, dx=None, dweight=None, workspace=None, workspace_size=0, stream=None):
        p, (mh, my, ma, md) = self.p, self._m
        mh.data, my.data, ma.data, md.data, p.weight, p.rstd, p.dweight = h, dy, add, dx, weight, rstd, dweight
        status = self._call(self._ref, workspace, workspace_size, stream)
        if status:
            _check(status, "zluda_ffn_rms_backward")


class Activate(_Call):
    def __init__(self, spec):
        super().__init__(spec)
        s, self.p = self.spec, zluda_ffn_activation()
        p, t = self.p, s["type"]
        p.activation, p.block_rows, p.rows, p.cols = s.get("activation", SILU), s.get("block_rows", 1), s["rows"], s["cols"]
        for name in ("gate", "up", "y"):
            self.matrix(name, p.cols, t)
        self.packed(p.packed, "codes", p.rows, p.cols, p.block_rows)
        self._call, self._ref, self._m = self.lib.zluda_ffn_activate, C.byref(p), _members(p, "gate up y packed")

    def run(self, gate, up=None, y=None, codes=None, scales=None, stream=None):
        mg, mu, my, mk = self._m
        mg.data, mu.data, my.data, mk.data, mk.scales = gate, up, y, codes, scales
        status = self._call(self._ref, stream)
        if status:
            _check(status, "zluda_ffn_activate")


class Unpack(_Call):
    def __init__(self, spec):
        super().__init__(spec)
        s = self.spec
        self.rows, self.cols, self.block_rows = s["rows"], s["cols"], s.get("block_rows", 1)
        self.y, self.c = _M(None, None, s.get("ldy", self.cols), 0, s["type"]), _M()
        self.packed(self.c, "codes", self.rows, self.cols, self.block_rows)
        self._call, self._refs = self.lib.zluda_ffn_unpack, (C.byref(self.c), C.byref(self.y))

    def run(self, codes, scales, y, stream=None):
        self.c.data, self.c.scales, self.y.data = codes, scales, y
        status = self._call(self.rows, self.cols, self.block_rows, self._refs[0], self._refs[1], stream)
        if status:
            _check(status, "zluda_ffn_unpack")


class GroupedForward(_Call):
    def __init__(self, spec):
        super().__init__(spec)
        s, self.p = self.spec, zluda_ffn_grouped()
        p, t = self.p, s["type"]
        p.rows, p.experts, p.features, p.model = s["rows"], s["experts"], s["features"], s["model"]
        if s.get("packed", False):
            self.packed(p.x, "x", p.rows, p.model)
            self.packed(p.w, "w", p.experts * p.features, p.model, PACK)
        else:
            self.matrix("x", p.model, t)
            self.matrix("w", p.model, t)
        self.matrix("y", p.features, t)
        self.query(self.lib.zluda_ffn_grouped_forward_workspace)
        self._call, self._ref, self._m = self.lib.zluda_ffn_grouped_forward, C.byref(p), _members(p, "x w y")

    def run(self, offsets, x, w, y, x_scales=None, w_scales=None, workspace=None, workspace_size=0, stream=None):
        mx, mw, my = self._m
        self.p.offsets, mx.data, mx.scales, mw.data, mw.scales, my.data = offsets, x, x_scales, w, w_scales, y
        status = self._call(self._ref, workspace, workspace_size, stream)
        if status:
            _check(status, "zluda_ffn_grouped_forward")


class GroupedBackward(_Call):
    def __init__(self, spec):
        super().__init__(spec)
        s, self.p = self.spec, zluda_ffn_grouped_grad()
        p, t = self.p, s["type"]
        p.rows, p.experts, p.features, p.model = s["rows"], s["experts"], s["features"], s["model"]
        for name, cols in (("dy", p.features), ("x", p.model), ("w", p.model), ("dx", p.model), ("dw", p.model)):
            self.matrix(name, cols, t)
        for name in ("dx", "dw"):
            getattr(p, name).data = 16 if s.get(name, True) else None
        wanted = p.dx.data, p.dw.data
        p.dx.data, p.dw.data = 16, None
        self.query(self.lib.zluda_ffn_grouped_backward_workspace)
        self.workspace_dx = self.workspace
        p.dx.data, p.dw.data = wanted
        self.query(self.lib.zluda_ffn_grouped_backward_workspace)
        self._call, self._ref, self._m = self.lib.zluda_ffn_grouped_backward, C.byref(p), _members(p, "dy x w dx dw")

    def run(self, offsets, dy, x=None, w=None, dx=None, dw=None, workspace=None, workspace_size=0, stream=None):
        if dx and not dw and workspace_size < self.workspace_dx:
            raise cublaslt.CublasLtError(abi.CUBLAS_STATUS_ALLOC_FAILED, "zluda_ffn_grouped_backward of dx alone, which takes a workspace of %d bytes," % self.workspace_dx)
        my, mx, mw, mdx, mdw = self._m
        self.p.offsets, my.data, mx.data, mw.data, mdx.data, mdw.data = offsets, dy, x, w, dx, dw
        status = self._call(self._ref, workspace, workspace_size, stream)
        if status:
            _check(status, "zluda_ffn_grouped_backward")
