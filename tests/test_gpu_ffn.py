"""The feed-forward operators (include/zluda_ffn.h) on the GPU against their definitions in 64 bits (ffn_oracle.py): element by
element within bounds that follow from the arithmetic, checkpoints bit for bit, at sizes around every edge of the tiles, any
alignment and pitch, with guard bytes around and between the rows of every output."""
import pytest
import torch

import ffn_oracle as O
from zluda_amd import abi, ffn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": (torch.bfloat16, abi.CUDA_R_16BF), "f16": (torch.float16, abi.CUDA_R_16F), "f32": (torch.float32, abi.CUDA_R_32F)}
ACT = {"silu": ffn.SILU, "gelu": ffn.GELU, "relu": ffn.RELU}


class Mat:
    """rows x cols with a pitch, `skip` elements behind a 256-byte boundary, in a buffer of guard bytes"""

    def __init__(self, rows, cols, dtype, ld=None, skip=0, data=None):
        self.rows, self.cols, self.ld = rows, cols, cols if ld is None else ld
        self.size = torch.empty((), dtype=dtype).element_size()
        self.skip = 64 + skip
        n = self.skip + rows * self.ld + 64
        self.raw = torch.full((n * self.size,), 0xCD, dtype=torch.uint8, device=DEV)
        self.flat = self.raw.view(dtype)
        self.view = self.flat[self.skip:self.skip + rows * self.ld].view(rows, self.ld)[:, :cols]
        if data is not None:
            self.view.copy_(data)

    @property
    def ptr(self):
        return self.flat.data_ptr() + self.skip * self.size

    def guards(self):
        """nothing but the matrix's elements has been written"""
        keep = self.raw.clone()
        m = keep.view(self.flat.dtype)[self.skip:self.skip + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols]
        m.copy_(torch.full((m.element_size(),), 0xCD, dtype=torch.uint8, device=DEV).view(self.flat.dtype).expand_as(m))
        return bool((keep == 0xCD).all())


class Ckpt:
    """a checkpoint with guard bytes behind the rows"""

    def __init__(self, rows, cols, wide=0):
        ld, lds = ffn.checkpoint_pitches(cols)
        self.rows, self.cols = rows, cols
        self.codes, self.scales = Mat(rows, ld, torch.uint8, ld + 32 * wide), Mat(rows, lds, torch.uint8, lds + wide)

    def guards(self):
        return self.codes.guards() and self.scales.guards()

    def matches(self, x):
        """bit for bit the checkpoint of x (a NaN code may have either sign)"""
        _, codes, scales = O.checkpoint(x)
        got = self.codes.view.cpu()
        nan = (codes & 0x7F) == 0x7F
        return torch.equal(got[~nan], codes[~nan]) and bool(((got[nan] & 0x7F) == 0x7F).all()) and torch.equal(self.scales.view.cpu(), scales)

    def values(self):
        c = self.codes.view.contiguous().view(torch.float8_e4m3fn).double()
        s = torch.ldexp(torch.ones((), dtype=torch.float64), self.scales.view.cpu().long() - 127).to(DEV)
        return (c * s.repeat_interleave(32, 1))[:, :self.cols]


def randn(seed, *shape, std=1.0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return torch.randn(shape, device=DEV, generator=gen) * std


def stream():
    return torch.cuda.current_stream().cuda_stream


def scratch(call):
    ws = torch.empty(max(16, call.workspace), dtype=torch.uint8, device=DEV)
    return dict(workspace=ws.data_ptr(), workspace_size=call.workspace), ws


# ---- gated feed-forward -----------------------------------------------------------------------------------------------------

def run_gated(typ, act, t, d, f, bias, kept, pad=0, skip=0, seed=0, x=None):
    dt, code = TYPES[typ]
    x = Mat(t, d, dt, d + pad, skip, randn(seed, t, d) if x is None else x)
    w = Mat(2 * f, d, dt, d + pad, skip, randn(seed + 1, 2 * f, d, std=1.5 * d ** -0.5))
    b = Mat(1, 2 * f, dt, None, skip, randn(seed + 2, 1, 2 * f, std=0.3)) if bias else None
    h = Mat(t, f, dt, f + pad, skip)
    if kept == ffn.KEPT_8BIT:
        g, u = Ckpt(t, f, pad), Ckpt(t, f, pad)
        ptrs = dict(gate=g.codes.ptr, gate_scales=g.scales.ptr, up=u.codes.ptr, up_scales=u.scales.ptr)
        pitch = dict(ldgate=g.codes.ld, ldgate_scales=g.scales.ld, ldup=u.codes.ld, ldup_scales=u.scales.ld)
    elif kept == ffn.KEPT_PLAIN:
        g, u = Mat(t, f, dt, f + pad, skip), Mat(t, f, dt, f + 2 * pad, skip)
        ptrs, pitch = dict(gate=g.ptr, up=u.ptr), dict(ldgate=g.ld, ldup=u.ld)
    else:
        g = u = None
        ptrs, pitch = {}, {}
    call = ffn.GatedForward(dict(type=code, activation=ACT[act], tokens=t, features=f, model=d, kept=kept, ldx=x.ld, ldw=w.ld, ldh=h.ld, **pitch))
    ws, _keep = scratch(call)
    call.run(x=x.ptr, w=w.ptr, bias=b.ptr if b else None, h=h.ptr, stream=stream(), **ws, **ptrs)
    torch.cuda.synchronize()
    ref = O.gated_forward(act, x.view, w.view, b.view[0] if b else None)
    return x, w, b, h, g, u, ref


def check_gated(h, g, u, kept, ref, what):
    O.check(h.view, ref["h"], what + " h")
    assert h.guards(), what
    for m, name in ((g, "g"), (u, "u")):
        if kept == ffn.KEPT_PLAIN:
            O.check(m.view, ref[name], what + " " + name)
            assert m.guards(), what + " " + name
        elif kept == ffn.KEPT_8BIT:
            # within one grid step of the block's scale from a value inside the bound, scales within a factor of two
            assert m.guards(), what + " " + name
            value, bound = ref[name]
            top = torch.nn.functional.pad(value.abs() + bound, (0, -value.shape[1] % 32)).reshape(value.shape[0], -1, 32).amax(2).repeat_interleave(32, 1)
            top = top[:, :value.shape[1]]
            # e4m3: half a step is 2^-4 of a value (relative), 2^-10 of the scale at least; the scale is at most top / 224
            allowed = bound + (value.abs() + bound) * 2.0 ** -4 + top / 224 * 2.0 ** -10
            assert ((m.values() - value).abs() <= allowed * 1.001).all(), what + " " + name
            assert (m.codes.view[:, value.shape[1]:] == 0).all()


SIZES = [(1, 8, 1), (1, 64, 32), (2, 31, 33), (5, 256, 688), (16, 512, 128), (17, 96, 40), (33, 264, 96), (48, 1024, 96), (63, 200, 7), (64, 128, 64), (65, 128, 65),
         (100, 1000, 129), (128, 64, 256), (129, 72, 127), (257, 136, 300), (300, 320, 520)]


@pytest.mark.parametrize("t,d,f", SIZES)
@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_gated_forward_sizes(gpu_api, typ, t, d, f):
    for i, act in enumerate(O.ACTS):
        for kept in (ffn.KEPT_NONE, ffn.KEPT_PLAIN, ffn.KEPT_8BIT):
            what = "gated %s %s %d x %d x %d kept %d" % (typ, act, t, d, f, kept)
            print(what, flush=True)
            _, _, _, h, g, u, ref = run_gated(typ, act, t, d, f, i != 1, kept, seed=10 * t + i)
            check_gated(h, g, u, kept, ref, what)


# every tile of gated_tile(): one, two and three token rows of each, K with a tail, of an odd number of stages, shorter than the ring
@pytest.mark.parametrize("t,d,f", [(7, 328, 4100), (33, 64, 4100), (50, 200, 8200), (65, 8, 4100), (120, 328, 12000), (128, 64, 12000), (257, 328, 6000), (250, 136, 12800)])
@pytest.mark.parametrize("typ,act,kept", [("bf16", "silu", ffn.KEPT_8BIT), ("f16", "gelu", ffn.KEPT_PLAIN), ("bf16", "relu", ffn.KEPT_NONE)])
def test_gated_forward_tiles(gpu_api, t, d, f, typ, act, kept):
    for bias, skip in ((True, 0), (False, 8)):
        what = "gated %s %s %d x %d x %d kept %d" % (typ, act, t, d, f, kept)
        print(what, flush=True)
        _, _, _, h, g, u, ref = run_gated(typ, act, t, d, f, bias, kept, skip, skip, seed=t)
        check_gated(h, g, u, kept, ref, what)


# enough tiles for the persistent kernel: ragged in every direction, K of two stages, of an odd number, with a tail
@pytest.mark.parametrize("t,d,f", [(1100, 200, 3400), (1025, 72, 3401), (2049, 64, 2056), (769, 328, 4100), (300, 512, 8200)])
@pytest.mark.parametrize("typ,act,kept", [("bf16", "silu", ffn.KEPT_8BIT), ("f16", "gelu", ffn.KEPT_PLAIN), ("bf16", "relu", ffn.KEPT_NONE)])
def test_gated_forward_many_tiles(gpu_api, t, d, f, typ, act, kept):
    for bias, skip in ((True, 0), (False, 0), (True, 8)):
        what = "gated %s %s %d x %d x %d kept %d" % (typ, act, t, d, f, kept)
        print(what, flush=True)
        _, _, _, h, g, u, ref = run_gated(typ, act, t, d, f, bias, kept, skip, skip, seed=t)
        check_gated(h, g, u, kept, ref, what)


@pytest.mark.parametrize("t,d,f", [(384, 136, 14300), (2000, 200, 5601), (4000, 64, 2816)])   # 192 tokens a tile
@pytest.mark.parametrize("typ,act,kept", [("bf16", "silu", ffn.KEPT_8BIT), ("f16", "gelu", ffn.KEPT_PLAIN)])
def test_gated_forward_many_narrow_tiles(gpu_api, t, d, f, typ, act, kept):
    for bias in (True, False):
        what = "gated %s %s %d x %d x %d kept %d" % (typ, act, t, d, f, kept)
        print(what, flush=True)
        _, _, _, h, g, u, ref = run_gated(typ, act, t, d, f, bias, kept, seed=t)
        check_gated(h, g, u, kept, ref, what)


@pytest.mark.parametrize("pad,skip", [(0, 1), (1, 0), (3, 5), (8, 0), (8, 8), (4, 4)])
@pytest.mark.parametrize("t,d,f", [(1, 128, 64), (9, 80, 72), (150, 256, 160), (520, 192, 264)])
def test_gated_forward_pitches_and_alignments(gpu_api, t, d, f, pad, skip):
    for kept in (ffn.KEPT_PLAIN, ffn.KEPT_8BIT):
        what = "gated pad %d skip %d %d x %d x %d" % (pad, skip, t, d, f)
        print(what, flush=True)
        _, _, _, h, g, u, ref = run_gated("bf16", "silu", t, d, f, True, kept, pad, skip, seed=t)
        check_gated(h, g, u, kept, ref, what)


@pytest.mark.parametrize("t", [3, 40, 300])
def test_gated_forward_rows_keep_to_themselves(gpu_api, t):
    """what is not finite in one token's row stays in that row"""
    d, f = 256, 160
    x = randn(5, t, d)
    x[t // 2, 7] = float("nan")
    x[t // 3, 9] = float("inf")
    for kept in (ffn.KEPT_NONE, ffn.KEPT_8BIT):
        _, _, _, h, g, _, ref = run_gated("bf16", "silu", t, d, f, False, kept, x=x)
        bad = torch.zeros(t, dtype=torch.bool, device=DEV)
        bad[[t // 2, t // 3]] = True
        assert torch.isfinite(h.view[~bad].float()).all() and torch.isnan(h.view[t // 2].float()).all()
        ok = {k: (v[0][~bad], v[1][~bad]) for k, v in ref.items()}
        O.check(h.view[~bad], ok["h"])
        if g:
            assert torch.isnan(g.values()[t // 2]).all()


def run_gated_backward(typ, act, t, d, f, kept, pad=0, skip=0, seed=0, want=("dx", "dw", "dbias", "h", "dz"), on=None):
    dt, code = TYPES[typ]
    dh = Mat(t, f, dt, f + pad, skip, randn(seed, t, f, std=0.5))
    w = Mat(2 * f, d, dt, d + pad, skip, randn(seed + 1, 2 * f, d, std=d ** -0.5))
    g0, u0, x0 = (randn(seed + 2 + i, t, n, std=1.3) for i, n in enumerate((f, f, d)))
    ins, pitch, vals = {}, {}, {}
    for name, data, n in (("gate", g0, f), ("up", u0, f), ("x", x0, d)):
        if kept == ffn.KEPT_8BIT:
            c = Ckpt(t, n, pad)
            data = data.to(dt)
            s = ffn.Checkpoint(dict(type=code, rows=t, cols=n, ldcodes=c.codes.ld, ldscales=c.scales.ld))
            s.store(x=data.data_ptr(), codes=c.codes.ptr, scales=c.scales.ptr, stream=stream())
            torch.cuda.synchronize()
            ins[name], ins[name + "_scales"] = c.codes.ptr, c.scales.ptr
            pitch["ld" + name], pitch["ld" + name + "_scales"] = c.codes.ld, c.scales.ld
            vals[name] = c.values()
            vals["_" + name] = c
        else:
            m = Mat(t, n, dt, n + pad, skip, data)
            ins[name], pitch["ld" + name], vals[name], vals["_" + name] = m.ptr, m.ld, m.view, m
    outs = {"dx": Mat(t, d, dt, d + pad, skip), "dw": Mat(2 * f, d, dt, d + pad, skip), "dbias": Mat(1, 2 * f, dt, None, skip), "h": Mat(t, f, dt, f + pad, skip),
            "dz": Mat(t, 2 * f, dt, 2 * f + pad, skip)}
    outs = {k: outs[k] for k in want}
    call = ffn.GatedBackward(dict(type=code, activation=ACT[act], tokens=t, features=f, model=d, kept=kept, x_kept=kept, bias="dbias" in want, lddh=dh.ld, ldw=w.ld,
                                  **{n: n in want for n in ("dx", "dw", "h", "dz")}, **pitch, **{"ld" + k: m.ld for k, m in outs.items() if k != "dbias"}))
    ws, _keep = scratch(call)
    call.run(dh=dh.ptr, w=w.ptr, stream=stream(), **ins, **{k: m.ptr for k, m in outs.items()}, **ws)
    torch.cuda.synchronize()
    return outs, O.gated_backward(act, dh.view, vals["gate"], vals["up"], vals["x"], w.view), (call, dh, w, ins, ws, vals, _keep)


def check_gated_backward(outs, ref, what):
    for k, m in outs.items():
        O.check(m.view if k != "dbias" else m.view[0], ref[k], what + " " + k)
        assert m.guards(), what + " " + k


@pytest.mark.parametrize("t,d,f", [(1, 8, 8), (1, 31, 1), (3, 64, 33), (16, 96, 40), (65, 37, 63), (130, 256, 96), (257, 72, 520), (513, 128, 264), (700, 264, 1040)])
@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_gated_backward_sizes(gpu_api, typ, t, d, f):
    for i, act in enumerate(O.ACTS):
        for kept in (ffn.KEPT_PLAIN, ffn.KEPT_8BIT):
            what = "gated backward %s %s %d x %d x %d kept %d" % (typ, act, t, d, f, kept)
            print(what, flush=True)
            outs, ref, _ = run_gated_backward(typ, act, t, d, f, kept, seed=t + i)
            check_gated_backward(outs, ref, what)


# sizes of the launch that makes dx and dw together (16-byte pieces): edges of its tiles and stages, and K of dx in one share and in many
@pytest.mark.parametrize("t,d,f", [(1, 8, 4), (2, 136, 60), (63, 128, 64), (64, 128, 68), (65, 120, 132), (127, 256, 200), (128, 264, 64), (129, 136, 300), (300, 520, 256),
                                   (1000, 136, 2052), (640, 1032, 128), (1, 1024, 4096)])
@pytest.mark.parametrize("pad", [0, 8, 72])
@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_gated_backward_products_together(gpu_api, typ, pad, t, d, f):
    for kept in (ffn.KEPT_PLAIN, ffn.KEPT_8BIT):
        what = "gated backward %s %d x %d x %d pad %d kept %d" % (typ, t, d, f, pad, kept)
        print(what, flush=True)
        outs, ref, _ = run_gated_backward(typ, "gelu", t, d, f, kept, pad, pad, seed=t)
        check_gated_backward(outs, ref, what)


@pytest.mark.parametrize("pad,skip", [(1, 0), (0, 3), (8, 8)])
@pytest.mark.parametrize("want", [("dx",), ("dw",), ("dx", "dw"), ("dbias",), ("h", "dz"), ("dw", "dbias")])
def test_gated_backward_pitches_and_choices(gpu_api, want, pad, skip):
    for kept in (ffn.KEPT_PLAIN, ffn.KEPT_8BIT):
        outs, ref, _ = run_gated_backward("bf16", "silu", 77, 80, 72, kept, pad, skip, want=want)
        check_gated_backward(outs, ref, "%s pad %d skip %d" % (want, pad, skip))


def test_gated_backward_of_no_tokens_is_zero(gpu_api):
    d, f = 40, 24
    dw, db = Mat(2 * f, d, torch.bfloat16, d + 3), Mat(1, 2 * f, torch.bfloat16)
    call = ffn.GatedBackward(dict(type=abi.CUDA_R_16BF, tokens=0, features=f, model=d, bias=True, lddw=dw.ld))
    ws, _keep = scratch(call)
    call.run(dh=None, gate=None, up=None, x=None, w=16, dx=16, dw=dw.ptr, dbias=db.ptr, stream=stream(), **ws)
    torch.cuda.synchronize()
    assert (dw.view == 0).all() and (db.view == 0).all() and dw.guards() and db.guards()
    ffn.GatedForward(dict(type=abi.CUDA_R_16BF, tokens=0, features=f, model=d)).run(x=None, w=16, h=None, stream=stream())


@pytest.mark.parametrize("act", O.ACTS)
def test_gated_gradients_against_differences(gpu_api, act):
    """the loss sum(dH * H) along random directions of X and W: central differences of the definition in 64 bits"""
    t, d, f = 33, 48, 40
    dt, code = TYPES["f16"]
    x, w = randn(1, t, d).to(dt), randn(2, 2 * f, d, std=d ** -0.5).to(dt)
    dh = randn(3, t, f, std=0.5).to(dt)
    z = x.double() @ w.double().t()
    g, u = z[:, :f].to(dt), z[:, f:].to(dt)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    call = ffn.GatedBackward(dict(type=code, activation=ACT[act], tokens=t, features=f, model=d))
    ws, _keep = scratch(call)
    call.run(dh=dh.data_ptr(), gate=g.contiguous().data_ptr(), up=u.contiguous().data_ptr(), x=x.data_ptr(), w=w.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(), stream=stream(), **ws)
    torch.cuda.synchronize()

    def loss(x, w):
        z = x @ w.t()
        return (dh.double() * O.act(act, z[:, :f])[0] * z[:, f:]).sum().item()

    step = 1e-5
    for k in range(3):
        vx, vw = randn(20 + k, t, d).double(), randn(30 + k, 2 * f, d).double() * d ** -0.5
        for vx_, vw_, grad, v in ((vx, 0 * vw, dx, vx), (0 * vx, vw, dw, vw)):
            num = (loss(x.double() + step * vx_, w.double() + step * vw_) - loss(x.double() - step * vx_, w.double() - step * vw_)) / (2 * step)
            ana = (grad.double() * v).sum().item()
            # G, U, dG, dU and the gradient are rounded to 11 bits each: five relative errors of 2^-11 at most on each of the
            # terms, which are random in sign: allowed is that of the norms
            allowed = 5 * 2.0 ** -11 * (grad.double().norm() * v.norm()).item()
            assert abs(num - ana) <= allowed, (act, num, ana, allowed)


# ---- layer norm -------------------------------------------------------------------------------------------------------------

NORM_SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 65), (9, 511), (8, 512), (7, 513), (70, 1001), (6, 1024), (5, 1025), (33, 2048), (4, 2050), (40, 4096), (3, 4099),
              (11, 8192), (2, 8200), (5, 12345), (3, 16384), (1000, 40), (2500, 96), (1300, 2000)]


def run_norm(typ, wtyp, rows, cols, pad=0, skip=0, seed=0, vectors=True, keep=True, x=None, eps=1e-5):
    dt, code = TYPES[typ]
    wt, wcode = TYPES[wtyp]
    if x is None:
        x = randn(seed, rows, cols) * (0.1 + 5 * torch.rand((rows, 1), device=DEV)) + 2.0 * randn(seed + 1, rows, 1)
    x = Mat(rows, cols, dt, cols + pad, skip, x)
    w, b = (Mat(1, cols, wt, None, skip, randn(seed + 2 + i, 1, cols) * 0.3 + 1 - i) for i in range(2))
    y, mean, rstd = Mat(rows, cols, dt, cols + 2 * pad, skip), Mat(1, rows, torch.float32), Mat(1, rows, torch.float32)
    c = Ckpt(rows, cols, pad)
    call = ffn.NormForward(dict(type=code, weight_type=wcode, rows=rows, cols=cols, eps=eps, ldx=x.ld, ldy=y.ld, ldkept=c.codes.ld, ldkept_scales=c.scales.ld))
    call.run(x=x.ptr, y=y.ptr, weight=w.ptr if vectors else None, bias=b.ptr if vectors else None, mean=mean.ptr, rstd=rstd.ptr, kept=c.codes.ptr if keep else None,
             kept_scales=c.scales.ptr if keep else None, stream=stream())
    torch.cuda.synchronize()
    ref = O.norm_forward(x.view, w.view[0] if vectors else None, b.view[0] if vectors else None, eps)
    return x, w, b, y, mean, rstd, c, ref


@pytest.mark.parametrize("rows,cols", NORM_SIZES)
@pytest.mark.parametrize("typ,wtyp", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")])
def test_norm_forward(gpu_api, typ, wtyp, rows, cols):
    print("norm", typ, rows, cols, flush=True)
    x, _, _, y, mean, rstd, c, ref = run_norm(typ, wtyp, rows, cols, seed=rows)
    O.check(y.view, ref["y"], "y")
    O.check(mean.view[0], ref["mean"], "mean")
    O.check(rstd.view[0], ref["rstd"], "rstd")
    assert c.matches(x.view)
    assert y.guards() and mean.guards() and rstd.guards() and c.guards()


@pytest.mark.parametrize("pad,skip", [(1, 0), (0, 1), (8, 8), (3, 5)])
@pytest.mark.parametrize("rows,cols", [(5, 72), (9, 1000), (6, 3000), (3, 9000)])
def test_norm_forward_pitches_and_options(gpu_api, rows, cols, pad, skip):
    for vectors, keep in ((True, True), (False, False)):
        x, _, _, y, mean, rstd, c, ref = run_norm("bf16", "f32", rows, cols, pad, skip, vectors=vectors, keep=keep)
        O.check(y.view, ref["y"], "y")
        assert y.guards() and c.guards() and (not keep or c.matches(x.view))


def test_norm_forward_in_place(gpu_api):
    for rows, cols in ((3, 100), (1000, 520), (700, 4096), (600, 9001)):
        x, w, b, y, _, _, c, ref = run_norm("bf16", "f32", rows, cols)
        call = ffn.NormForward(dict(type=abi.CUDA_R_16BF, weight_type=abi.CUDA_R_32F, rows=rows, cols=cols))
        kept = Ckpt(rows, cols)
        call.run(x=x.ptr, y=x.ptr, weight=w.ptr, bias=b.ptr, kept=kept.codes.ptr, kept_scales=kept.scales.ptr, stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(x.view, y.view) and torch.equal(kept.codes.view, c.codes.view) and x.guards()


def test_norm_forward_of_rows_far_from_zero_and_constant_rows(gpu_api):
    """the variance comes from differences to the mean: a mean 1000 times the spread costs no more than the bound says, and a
    constant row gives its bias"""
    x = randn(3, 6, 700) + 1000.0
    x[2] = 5.5
    _, _, b, y, _, rstd, _, ref = run_norm("f32", "f32", 6, 700, x=x)
    O.check(y.view, ref["y"], "y")
    O.check(rstd.view[0], ref["rstd"], "rstd")
    assert (y.view[2] - b.view[0]).abs().max() < 1e-3


def test_norm_rows_keep_to_themselves(gpu_api):
    x = randn(3, 9, 600)
    x[4, 100] = float("inf")
    x[6, 3] = float("nan")
    xm, _, _, y, _, _, c, _ = run_norm("bf16", "bf16", 9, 600, x=x)
    good = [0, 1, 2, 3, 5, 7, 8]
    assert torch.isfinite(y.view[good].float()).all() and torch.isnan(y.view[6].float()).all() and c.matches(xm.view)


def run_norm_backward(typ, wtyp, rows, cols, ck, add, pad=0, skip=0, seed=0, vectors=True, want_dx=True, want_w=True):
    dt, code = TYPES[typ]
    wt, wcode = TYPES[wtyp]
    x0 = (randn(seed, rows, cols) * 2 + 0.5).to(dt)
    if ck:
        c = Ckpt(rows, cols, pad)
        ffn.Checkpoint(dict(type=code, rows=rows, cols=cols, ldcodes=c.codes.ld, ldscales=c.scales.ld)).store(x=x0.data_ptr(), codes=c.codes.ptr, scales=c.scales.ptr, stream=stream())
        xv, ins, pitch = c.values(), dict(x=c.codes.ptr, x_scales=c.scales.ptr), dict(ldx=c.codes.ld, ldx_scales=c.scales.ld)
    else:
        c = Mat(rows, cols, dt, cols + pad, skip, x0)
        xv, ins, pitch = c.view, dict(x=c.ptr), dict(ldx=c.ld)
    torch.cuda.synchronize()
    mean = x0.float().mean(1).contiguous()
    rstd = (x0.float().var(1, unbiased=False) + 1e-5).rsqrt().contiguous()
    dy, a = (Mat(rows, cols, dt, cols + pad, skip, randn(seed + 5 + i, rows, cols, std=0.5)) for i in range(2))
    w = Mat(1, cols, wt, None, skip, randn(seed + 9, 1, cols) * 0.3 + 1)
    outs = {}
    if want_dx:
        outs["dx"] = Mat(rows, cols, dt, cols + 2 * pad, skip)
    if want_w:
        outs["dweight"], outs["dbias"] = Mat(1, cols, wt, None, skip), Mat(1, cols, wt, None, skip)
    call = ffn.NormBackward(dict(type=code, weight_type=wcode, rows=rows, cols=cols, x_kept=ffn.KEPT_8BIT if ck else ffn.KEPT_PLAIN, weights=want_w, lddy=dy.ld, ldadd=a.ld,
                                 lddx=cols + 2 * pad, **pitch))
    ws, _keep = scratch(call)
    run = lambda: call.run(dy=dy.ptr, mean=mean.data_ptr(), rstd=rstd.data_ptr(), weight=w.ptr if vectors else None, add=a.ptr if add else None, stream=stream(),  # noqa: E731
                           **ins, **ws, **{k: m.ptr for k, m in outs.items()})
    run()
    torch.cuda.synchronize()
    ref = O.norm_backward(xv, dy.view, w.view[0] if vectors else None, mean, rstd, a.view if add else None)
    return outs, ref, run, (dy, a, w, mean, rstd, c, _keep)


def check_norm_backward(outs, ref, what):
    for k, m in outs.items():
        O.check(m.view if k == "dx" else m.view[0], ref[k], what + " " + k)
        assert m.guards(), what + " " + k


@pytest.mark.parametrize("rows,cols", NORM_SIZES)
@pytest.mark.parametrize("typ,wtyp", [("bf16", "f32"), ("f16", "f16"), ("f32", "f32")])
def test_norm_backward(gpu_api, typ, wtyp, rows, cols):
    for ck in (False, True):
        what = "norm backward %s %d x %d ck %d" % (typ, rows, cols, ck)
        print(what, flush=True)
        outs, ref, run, _ = run_norm_backward(typ, wtyp, rows, cols, ck, add=ck, seed=rows)
        check_norm_backward(outs, ref, what)
        first = {k: m.view.clone() for k, m in outs.items()}
        run()
        torch.cuda.synchronize()
        assert all(torch.equal(first[k], m.view) for k, m in outs.items()), "the same call gives the same bits"


@pytest.mark.parametrize("pad,skip", [(1, 0), (0, 1), (8, 8)])
@pytest.mark.parametrize("rows,cols", [(5, 72), (90, 1000), (6, 3000), (3, 9000)])
def test_norm_backward_pitches_and_choices(gpu_api, rows, cols, pad, skip):
    for add, vectors, want_dx, want_w in ((True, False, True, False), (False, True, False, True), (True, True, True, True)):
        outs, ref, _, _ = run_norm_backward("bf16", "bf16", rows, cols, False, add, pad, skip, vectors=vectors, want_dx=want_dx, want_w=want_w)
        check_norm_backward(outs, ref, "pad %d skip %d" % (pad, skip))


def test_norm_backward_in_place_and_of_no_rows(gpu_api):
    rows, cols = 37, 700
    outs, ref, _, (dy, a, w, mean, rstd, x, _) = run_norm_backward("f32", "f32", rows, cols, False, True)
    call = ffn.NormBackward(dict(type=abi.CUDA_R_32F, rows=rows, cols=cols, weights=False))
    for target in (a, dy):
        keep = target.view.clone()
        call.run(x=x.ptr, dy=dy.ptr, mean=mean.data_ptr(), rstd=rstd.data_ptr(), weight=w.ptr, add=a.ptr, dx=target.ptr, stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(target.view, outs["dx"].view)
        target.view.copy_(keep)
    dw, db = Mat(1, cols, torch.float32), Mat(1, cols, torch.float32)
    ffn.NormBackward(dict(type=abi.CUDA_R_32F, rows=0, cols=cols)).run(x=None, dy=None, mean=None, rstd=None, dweight=dw.ptr, dbias=db.ptr, stream=stream())
    torch.cuda.synchronize()
    assert (dw.view == 0).all() and (db.view == 0).all() and dw.guards() and db.guards()


def test_norm_gradients_against_differences(gpu_api):
    """the loss sum(dY * Y) along random directions of x, the weight and the bias"""
    rows, cols, eps = 7, 90, 1e-5
    x, dy, w, b = randn(1, rows, cols) * 2 + 0.5, randn(2, rows, cols), randn(3, 1, cols)[0] + 1, randn(4, 1, cols)[0]
    mean, rstd = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    y, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    spec = dict(type=abi.CUDA_R_32F, rows=rows, cols=cols, eps=eps)
    ffn.NormForward(spec).run(x=x.data_ptr(), y=y.data_ptr(), weight=w.data_ptr(), bias=b.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr(), stream=stream())
    call = ffn.NormBackward(spec)
    ws, _keep = scratch(call)
    call.run(x=x.data_ptr(), dy=dy.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr(), weight=w.data_ptr(), dx=dx.data_ptr(), dweight=dw.data_ptr(), dbias=db.data_ptr(),
             stream=stream(), **ws)
    torch.cuda.synchronize()
    loss = lambda x, w, b: (dy.double() * O.norm_forward(x, w, b, eps)["y"][0]).sum().item()  # noqa: E731
    step = 1e-5
    base = [t.double() for t in (x, w, b)]
    for i, grad in enumerate((dx, dw, db)):
        for k in range(3):
            v = randn(50 + k, *grad.shape).double()
            plus, minus = list(base), list(base)
            plus[i], minus[i] = base[i] + step * v, base[i] - step * v
            num = (loss(*plus) - loss(*minus)) / (2 * step)
            ana = (grad.double() * v).sum().item()
            assert abs(num - ana) <= 1e-5 * (grad.double().norm() * v.norm()).item(), (i, num, ana)   # 32-bit rounding, 100 terms deep


# ---- checkpoints ------------------------------------------------------------------------------------------------------------

def special_values(dt):
    """rows of 64: zeros, the type's ends, ties of the e4m3 grid, block tops around 448, infinities and NaN"""
    fin = torch.finfo(dt)
    rows = [torch.zeros(64), torch.full((64,), -0.0), torch.full((64,), fin.max), torch.full((64,), fin.tiny), torch.full((64,), fin.tiny / 4),
            torch.linspace(-460, 460, 64), torch.linspace(440, 456, 64), torch.arange(64) * 0.03125 + 1, torch.arange(64) * 2.0 ** -10, torch.arange(64) / 16.0 * fin.tiny]
    for top in (1.0, 1.7421875, 1.75, 1.7578125, 1.9921875, 448.0):
        r = torch.arange(64) / 64.0
        r[5] = top
        rows.append(r)
    bad = torch.arange(64) / 7.0
    bad[3], bad[11], bad[40] = float("inf"), float("-inf"), float("nan")
    all_bad = torch.full((64,), float("nan"))
    return torch.stack(rows + [bad, all_bad]).to(dt)


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
def test_checkpoint_special_values(gpu_api, typ):
    dt, code = TYPES[typ]
    x = special_values(dt).to(DEV)
    rows, cols = x.shape
    c, back = Ckpt(rows, cols), Mat(rows, cols, dt)
    call = ffn.Checkpoint(dict(type=code, rows=rows, cols=cols))
    call.store(x=x.data_ptr(), codes=c.codes.ptr, scales=c.scales.ptr, stream=stream())
    call.load(codes=c.codes.ptr, scales=c.scales.ptr, x=back.ptr, stream=stream())
    torch.cuda.synchronize()
    values, codes, scales = O.checkpoint(x)
    nan = torch.isnan(values)
    pad = torch.nn.functional.pad(nan, (0, codes.shape[1] - cols))
    assert torch.equal(c.scales.view.cpu(), scales)
    assert torch.equal(c.codes.view.cpu()[~pad], codes[~pad]) and ((c.codes.view.cpu()[pad] & 0x7F) == 0x7F).all()
    assert torch.equal(back.view.cpu()[~nan], values.to(dt)[~nan]) and torch.isnan(back.view.cpu()[nan].float()).all()


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (5, 33), (2, 100), (7, 511), (4, 513), (130, 777), (66, 2048), (9, 20000)])
@pytest.mark.parametrize("typ,pad,skip", [("bf16", 0, 0), ("f16", 1, 1), ("f32", 3, 1), ("bf16", 8, 8)])
def test_checkpoint_round_trip(gpu_api, rows, cols, typ, pad, skip):
    dt, code = TYPES[typ]
    x = Mat(rows, cols, dt, cols + pad, skip, randn(rows, rows, cols) * torch.exp(4 * randn(7, rows, 1)))
    c, back = Ckpt(rows, cols, pad), Mat(rows, cols, dt, cols + pad, skip)
    call = ffn.Checkpoint(dict(type=code, rows=rows, cols=cols, ldx=x.ld, ldcodes=c.codes.ld, ldscales=c.scales.ld))
    call.store(x=x.ptr, codes=c.codes.ptr, scales=c.scales.ptr, stream=stream())
    call.load(codes=c.codes.ptr, scales=c.scales.ptr, x=back.ptr, stream=stream())
    torch.cuda.synchronize()
    assert c.matches(x.view) and c.guards() and back.guards()
    assert torch.equal(torch.nan_to_num(back.view.cpu(), nan=-1.25), torch.nan_to_num(O.checkpoint(x.view)[0].to(dt), nan=-1.25))


# ---- offsets beyond 32 bits -------------------------------------------------------------------------------------------------

def test_norm_and_checkpoint_beyond_32_bits(gpu_api):
    """2.4e9 elements: the first and last rows, and some between"""
    rows, cols = 290000, 8192
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    x.copy_(randn(1, 1000, cols).to(torch.bfloat16).repeat(rows // 1000, 1))
    x[-1] = randn(2, cols) * 3
    y, (codes, scales), back = torch.empty_like(x), ffn.checkpoint_buffers(rows, cols, DEV), torch.empty_like(x)
    spec = dict(type=abi.CUDA_R_16BF, rows=rows, cols=cols)
    ffn.NormForward(spec).run(x=x.data_ptr(), y=y.data_ptr(), stream=stream())
    c = ffn.Checkpoint(spec)
    c.store(x=x.data_ptr(), codes=codes.data_ptr(), scales=scales.data_ptr(), stream=stream())
    c.load(codes=codes.data_ptr(), scales=scales.data_ptr(), x=back.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    for at in ([0, 1], [262143, 262144], [rows - 2, rows - 1]):
        O.check(y[at], O.norm_forward(x[at], None, None, 1e-5)["y"], str(at))
        value, code, scale = O.checkpoint(x[at])
        assert torch.equal(codes[at].cpu(), code) and torch.equal(scales[at].cpu(), scale) and torch.equal(back[at].cpu(), value.to(torch.bfloat16))
    mean, rstd = torch.zeros(rows, device=DEV), torch.ones(rows, device=DEV)
    ffn.NormBackward(dict(spec, weights=False)).run(x=x.data_ptr(), dy=y.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr(), dx=back.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    for at in ([0, 1], [262143, 262144], [rows - 2, rows - 1]):
        O.check(back[at], O.norm_backward(x[at], y[at], None, mean[at], rstd[at])["dx"], str(at))


@pytest.mark.parametrize("which", ["x", "h"])
def test_gated_forward_pitches_beyond_32_bits(gpu_api, which):
    """rows 16 MiB apart: X (which leaves the 2 GiB windows), H and what is kept"""
    t, d, f = 300, 128, 200
    wide = 8 << 20
    big = torch.empty(t * wide, dtype=torch.bfloat16, device=DEV)
    far = big.view(t, wide)
    x, w = randn(1, t, d).to(torch.bfloat16), randn(2, 2 * f, d, std=d ** -0.5).to(torch.bfloat16)
    h = torch.empty(t, f, dtype=torch.bfloat16, device=DEV)
    spec = dict(type=abi.CUDA_R_16BF, tokens=t, features=f, model=d, kept=ffn.KEPT_PLAIN)
    if which == "x":
        far[:, :d] = x
        ffn.GatedForward(dict(spec, ldx=wide, kept=ffn.KEPT_NONE)).run(x=big.data_ptr(), w=w.data_ptr(), h=h.data_ptr(), stream=stream())
        outs = {"h": h}
    else:
        ffn.GatedForward(dict(spec, ldh=wide, ldgate=wide, ldup=wide)).run(x=x.data_ptr(), w=w.data_ptr(), h=big.data_ptr(), gate=big.data_ptr() + 2000, up=big.data_ptr() + 4000,
                                                                          stream=stream())
        outs = {"h": far[:, :f], "g": far[:, 1000:1000 + f], "u": far[:, 2000:2000 + f]}
    torch.cuda.synchronize()
    ref = O.gated_forward("silu", x, w, None)
    for k, v in outs.items():
        O.check(v, ref[k], k)


def test_gated_backward_beyond_32_bits(gpu_api):
    """[dG dU] of 2.3e9 bytes: its last rows, the gradients that come from them, and a bias gradient over all rows"""
    t, d, f = 42000, 64, 14336
    bf = torch.bfloat16
    rows = 500
    dh, g, u = (randn(i, rows, f, std=0.7).to(bf).repeat(t // rows, 1) for i in range(3))
    x, w = randn(4, t, d).to(bf), randn(5, 2 * f, d, std=0.1).to(bf)
    dz, dx, dw, db = (torch.empty(s, dtype=bf, device=DEV) for s in ((t, 2 * f), (t, d), (2 * f, d), (2 * f,)))
    call = ffn.GatedBackward(dict(type=abi.CUDA_R_16BF, tokens=t, features=f, model=d, bias=True, dz=True))
    ws, _keep = scratch(call)
    call.run(dh=dh.data_ptr(), gate=g.data_ptr(), up=u.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(), dbias=db.data_ptr(), dz=dz.data_ptr(),
             stream=stream(), **ws)
    torch.cuda.synchronize()
    for at in (slice(0, 3), slice(t - 3, t)):
        ref = O.gated_backward("silu", dh[at], g[at], u[at], x[at], w)
        O.check(dz[at], ref["dz"], "dz")
        O.check(dx[at], ref["dx"], "dx")
    # the rows repeat: their sums are those of one period times the periods, and dw that with X summed over the periods
    one = O.gated_backward("silu", dh[:rows], g[:rows], u[:rows], x[:rows], w)
    n = t // rows
    value, bound = one["dbias"]
    O.check(db, (n * value, n * bound + (t + 1) * O.E32 * n * (one["dz"][0].abs() + one["dz"][1]).sum(0)), "dbias")
    xs = x.double().reshape(n, rows, d)
    z, ez = one["dz"]
    er = ez + O.UNIT[bf] * (z.abs() + ez) + O.TINY[bf]
    mag = (z.abs() + er).t() @ xs.abs().sum(0)
    O.check(dw, (z.t() @ xs.sum(0), er.t() @ xs.abs().sum(0) + (t + 1) * O.E32 * mag), "dw")


# ---- streams and graphs -----------------------------------------------------------------------------------------------------

def test_operators_in_a_graph_on_another_stream(gpu_api):
    """a step (norm, gated layer with 8-bit checkpoints, its backward) captured once and replayed with new inputs, other work and
    synchronisations in between: every replay gives the bits of the eager calls"""
    t, d, f = 96, 256, 320
    bf, code = TYPES["bf16"]
    x, y, h, dh = (torch.empty(t, n, dtype=bf, device=DEV) for n in (d, d, f, f))
    w = randn(1, 2 * f, d, std=d ** -0.5).to(bf)
    dx, dw = torch.empty(t, d, dtype=bf, device=DEV), torch.empty(2 * f, d, dtype=bf, device=DEV)
    dn, dwt, dbs = torch.empty(t, d, dtype=bf, device=DEV), torch.empty(d, device=DEV), torch.empty(d, device=DEV)
    mean, rstd = torch.empty(t, device=DEV), torch.empty(t, device=DEV)
    (g, gs), (u, us), (c, cs), (k, ks) = (ffn.checkpoint_buffers(t, n, DEV) for n in (f, f, d, d))
    spec = dict(type=code, tokens=t, features=f, model=d)
    fwd, bwd = ffn.GatedForward(dict(spec, kept=ffn.KEPT_8BIT)), ffn.GatedBackward(dict(spec, kept=ffn.KEPT_8BIT, x_kept=ffn.KEPT_8BIT))
    nspec = dict(type=code, weight_type=abi.CUDA_R_32F, rows=t, cols=d, x_kept=ffn.KEPT_8BIT)
    nf, nb, ck = ffn.NormForward(nspec), ffn.NormBackward(nspec), ffn.Checkpoint(dict(type=code, rows=t, cols=d))
    ws = torch.empty(max(16, fwd.workspace, bwd.workspace, nb.workspace), dtype=torch.uint8, device=DEV)

    def step():
        s, p = stream(), lambda a: a.data_ptr()  # noqa: E731
        w_ = dict(workspace=p(ws), workspace_size=ws.numel(), stream=s)
        nf.run(x=p(x), y=p(y), mean=p(mean), rstd=p(rstd), kept=p(k), kept_scales=p(ks), stream=s)
        ck.store(x=p(y), codes=p(c), scales=p(cs), stream=s)
        fwd.run(x=p(y), w=p(w), h=p(h), gate=p(g), gate_scales=p(gs), up=p(u), up_scales=p(us), **w_)
        bwd.run(dh=p(dh), gate=p(g), gate_scales=p(gs), up=p(u), up_scales=p(us), x=p(c), x_scales=p(cs), w=p(w), dx=p(dx), dw=p(dw), **w_)
        nb.run(x=p(k), x_scales=p(ks), dy=p(dx), mean=p(mean), rstd=p(rstd), dx=p(dn), dweight=p(dwt), dbias=p(dbs), **w_)

    outs = (h, dw, dn, dwt, dbs)
    x.copy_(randn(100, t, d)); dh.copy_(randn(101, t, f))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step()
    for r in range(4):
        x.copy_(randn(200 + r, t, d)); dh.copy_(randn(300 + r, t, f))
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, outs)), "replay %d" % r
        assert all(torch.isfinite(a.float()).all() for a in got)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("which", ["x", "dz", "x_8bit"])
def test_gated_in_parts(gpu_api, which, dt):
    """rows so far apart that the matmuls take the tokens in two parts: X of the forward product, [dG dU] or X of the backward pass"""
    t, d, f, wide = 2900, 136, 200, 400000
    code = {torch.bfloat16: abi.CUDA_R_16BF, torch.float16: abi.CUDA_R_16F}[dt]
    big = torch.empty(t * wide, dtype=dt, device=DEV)
    far = big.view(t, wide)
    x, w = randn(1, t, d).to(dt), randn(2, 2 * f, d, std=d ** -0.5).to(dt)
    kept = ffn.KEPT_8BIT if which == "x_8bit" else ffn.KEPT_PLAIN
    if which != "dz":
        far[:, :d] = x
        g, u = ([Ckpt(t, f), Ckpt(t, f)] if which == "x_8bit" else [Mat(t, f, dt), Mat(t, f, dt)])
        h = torch.empty(t, f, dtype=dt, device=DEV)
        args = dict(gate=g.codes.ptr, up=u.codes.ptr, gate_scales=g.scales.ptr, up_scales=u.scales.ptr) if which == "x_8bit" else dict(gate=g.ptr, up=u.ptr)
        lds = dict(ldgate=g.codes.ld, ldup=u.codes.ld, ldgate_scales=g.scales.ld, ldup_scales=u.scales.ld) if which == "x_8bit" else dict(ldgate=g.ld, ldup=u.ld)
        ffn.GatedForward(dict(type=code, tokens=t, features=f, model=d, ldx=wide, kept=kept, **lds)).run(x=big.data_ptr(), w=w.data_ptr(), h=h.data_ptr(), stream=stream(), **args)
        torch.cuda.synchronize()
        ref = O.gated_forward("silu", x, w, None)
        O.check(h, ref["h"], "h")
        if which == "x_8bit":
            for m, name in ((g, "g"), (u, "u")):  # (half a step, as for the checkpoints of run_gated())
                value, bound = ref[name]
                top = torch.nn.functional.pad(value.abs() + bound, (0, -f % 32)).reshape(t, -1, 32).amax(2).repeat_interleave(32, 1)[:, :f]
                assert ((m.values() - value).abs() <= (bound + (value.abs() + bound) * 2.0 ** -4 + top / 224 * 2.0 ** -10) * 1.001).all() and m.guards(), name
            return
        O.check(g.view, ref["g"], "g")
        O.check(u.view, ref["u"], "u")
    dh, gate, up = (randn(i, t, f, std=0.7).to(dt) for i in range(3, 6))
    dx, dw, db = (torch.empty(s, dtype=dt, device=DEV) for s in ((t, d), (2 * f, d), (2 * f,)))
    spec = dict(type=code, tokens=t, features=f, model=d, bias=True, dz=which == "dz", **({"lddz": wide} if which == "dz" else {"ldx": wide}))
    call = ffn.GatedBackward(spec)
    ws, _keep = scratch(call)
    call.run(dh=dh.data_ptr(), gate=gate.data_ptr(), up=up.data_ptr(), x=big.data_ptr() if which == "x" else x.data_ptr(), w=w.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(),
             dbias=db.data_ptr(), dz=big.data_ptr() if which == "dz" else None, stream=stream(), **ws)
    torch.cuda.synchronize()
    ref = O.gated_backward("silu", dh, gate, up, x, w)
    for name, out in (("dx", dx), ("dw", dw), ("dbias", db)) + ((("dz", far[:, :2 * f]),) if which == "dz" else ()):
        O.check(out, ref[name], name)
