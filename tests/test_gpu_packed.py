"""RMS norm, packing and unpacking (include/zluda_ffn.h) on the GPU against their definitions in 64 bits (packed_oracle.py), at sizes around every edge of
the kernels, any alignment and pitch, with guard bytes around and between the rows of every output."""
import pytest
import torch

import ffn_oracle as O
import packed_oracle as P
from test_gpu_ffn import ACT, DEV, Mat, TYPES, randn, stream
from zluda_amd import ffn

pytestmark = pytest.mark.gpu


class Packed:
    """a packed matrix with guard bytes: codes rows x cols, scales as the header lays them out"""

    def __init__(self, rows, cols, pad=0, skip=0, block_rows=1):
        ld, lds = ffn.packed_pitches(rows, cols, block_rows)
        self.rows, self.cols, self.block_rows = rows, cols, block_rows
        self.codes = Mat(rows, cols, torch.uint8, (cols if pad else ld) + pad, skip)
        lines = P.blocks(cols) if block_rows == 1 else P.blocks(rows)
        width = rows if block_rows == 1 else P.blocks(cols)
        self.scales = Mat(lines, width, torch.float32, lds + pad)
        self.pitch = dict(ldcodes=self.codes.ld, ldcodes_scales=self.scales.ld)
        self.ptrs = dict(codes=self.codes.ptr, scales=self.scales.ptr)

    def guards(self):
        return self.codes.guards() and self.scales.guards()

    def by_block(self):
        """scales as [row block][block]"""
        return self.scales.view.t() if self.block_rows == 1 else self.scales.view

    def check(self, value, bound, what):
        P.check_packed(self.codes.view, self.by_block(), value, bound, self.cols, self.block_rows, what)
        assert self.guards(), what


def residual_sum(x, r, dt):
    """rounded once from 32 bits, as the operator does"""
    return x if r is None else (x.float() + r.float()).to(dt)


SHAPES = [(1, 1), (1, 7), (2, 8), (3, 127), (5, 128), (4, 129), (9, 500), (17, 512), (33, 513), (6, 1001), (3, 1024), (5, 1025), (7, 2048), (4, 2056), (3, 4096), (2, 4104),
          (3, 8192), (2, 8200), (2, 16384), (700, 64), (300, 1000)]


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_rms_forward(typ, rows, cols):
    dt, code = TYPES[typ]
    for pad, skip, res, wt in ((0, 0, True, typ), (3, 1, True, "f32"), (8, 0, False, typ), (0, 8, False, None)):
        x, r = Mat(rows, cols, dt, cols + pad, skip, randn(rows + cols, rows, cols)), Mat(rows, cols, dt, cols + 2 * pad, skip, randn(7, rows, cols, std=3.0))
        w = None if wt is None else Mat(1, cols, TYPES[wt][0], None, skip, 1 + randn(9, 1, cols, std=0.3))
        s, y = Mat(rows, cols, dt, cols + pad, skip), Mat(rows, cols, dt, cols + pad, skip)
        rstd, packed = Mat(1, rows, torch.float32), Packed(rows, cols, pad, skip)
        call = ffn.RmsForward(dict(type=code, weight_type=TYPES[wt or typ][1], rows=rows, cols=cols, eps=1e-6, ldx=x.ld, ldresidual=r.ld, ldsum=s.ld, ldy=y.ld, **packed.pitch))
        call.run(x=x.ptr, residual=r.ptr if res else None, weight=None if w is None else w.ptr, sum=s.ptr, y=y.ptr, rstd=rstd.ptr, stream=stream(), **packed.ptrs)
        torch.cuda.synchronize()
        what = "%s %dx%d pad %d" % (typ, rows, cols, pad)
        h = residual_sum(x.view, r.view if res else None, dt)
        assert torch.equal(s.view, h), what
        ref = P.rms_forward(h, None if w is None else w.view[0], 1e-6)
        O.check(y.view, ref["y"], what + " y")
        O.check(rstd.view[0], ref["rstd"], what + " rstd")
        packed.check(*ref["y"], what)
        assert s.guards() and y.guards() and rstd.guards(), what


def test_rms_forward_in_place_and_single_outputs():
    rows, cols, dt, code = 37, 1000, *TYPES["bf16"]
    x, r = randn(1, rows, cols).to(dt), randn(2, rows, cols).to(dt)
    h = residual_sum(x, r, dt)
    ref = P.rms_forward(h, None, 1e-5)
    call = ffn.RmsForward(dict(type=code, rows=rows, cols=cols))
    a, b = x.clone(), r.clone()
    call.run(x=a.data_ptr(), residual=b.data_ptr(), sum=b.data_ptr(), y=a.data_ptr(), stream=stream())      # the sum over the residual, y over x
    assert torch.equal(b, h)
    O.check(a, ref["y"], "in place")
    b = r.clone()
    call.run(x=x.data_ptr(), residual=b.data_ptr(), y=b.data_ptr(), stream=stream())
    O.check(b, ref["y"], "y over the residual")
    p = Packed(rows, cols)
    call.run(x=x.data_ptr(), residual=r.data_ptr(), stream=stream(), **p.ptrs)
    torch.cuda.synchronize()
    p.check(*ref["y"], "packed alone")
    s = torch.empty_like(x)
    call.run(x=x.data_ptr(), residual=r.data_ptr(), sum=s.data_ptr(), stream=stream())
    assert torch.equal(s, h)


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_rms_backward(typ, rows, cols):
    dt, code = TYPES[typ]
    for pad, skip, add, wt in ((0, 0, True, typ), (3, 1, False, "f32"), (8, 0, True, None)):
        mat = lambda seed, std=1.0: Mat(rows, cols, dt, cols + pad, skip, randn(seed, rows, cols, std=std))  # noqa: E731
        h, dy, more = mat(1, 2.0), mat(2, 0.1), mat(3, 0.1)
        w = None if wt is None else Mat(1, cols, TYPES[wt][0], None, skip, 1 + randn(9, 1, cols, std=0.3))
        rstd = P.rms_forward(h.view, None, 1e-5)["rstd"][0].float()
        dx, dw = Mat(rows, cols, dt, cols + pad, skip), Mat(1, cols, TYPES[wt or typ][0], None, skip)
        call = ffn.RmsBackward(dict(type=code, weight_type=TYPES[wt or typ][1], rows=rows, cols=cols, ldh=h.ld, lddy=dy.ld, ldadd=more.ld, lddx=dx.ld))
        ws = torch.empty(max(16, call.workspace), dtype=torch.uint8, device=DEV)
        args = dict(h=h.ptr, dy=dy.ptr, rstd=rstd.data_ptr(), weight=None if w is None else w.ptr, add=more.ptr if add else None, workspace=ws.data_ptr(),
                    workspace_size=call.workspace, stream=stream())
        call.run(dx=dx.ptr, dweight=dw.ptr, **args)
        torch.cuda.synchronize()
        what = "%s %dx%d pad %d" % (typ, rows, cols, pad)
        ref = P.rms_backward(h.view, dy.view, None if w is None else w.view[0], rstd, more.view if add else None)
        O.check(dx.view, ref["dx"], what + " dx")
        O.check(dw.view[0], ref["dweight"], what + " dweight")
        assert dx.guards() and dw.guards(), what
        first = dw.view.clone()
        dw.view.zero_()
        call.run(dweight=dw.ptr, **args)                                          # alone, and the same bits again
        assert torch.equal(dw.view, first), what
        call.run(dx=dy.ptr, **args)                                               # over dy
        torch.cuda.synchronize()
        O.check(dy.view, ref["dx"], what + " dx over dy")


def test_rms_of_no_rows():
    dw = torch.full((64,), 7.0, dtype=torch.bfloat16, device=DEV)
    call = ffn.RmsBackward(dict(type=TYPES["bf16"][1], rows=0, cols=64))
    call.run(h=None, dy=None, rstd=None, dweight=dw.data_ptr(), stream=stream())
    assert (dw == 0).all()
    ffn.RmsForward(dict(type=TYPES["bf16"][1], rows=0, cols=64)).run(x=None, y=None, stream=stream())


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("act", [None, "silu", "gelu", "relu"])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_activate(typ, act, block_rows):
    dt, code = TYPES[typ]
    for rows, cols, pad, skip in ((1, 1, 0, 0), (3, 130, 3, 1), (130, 127, 0, 0), (127, 257, 5, 0), (257, 640, 8, 0), (5, 520, 0, 3), (1100, 136, 0, 0)):
        for gated in (False, True) if act else (False,):
            z = Mat(rows, 2 * cols, dt, 2 * cols + pad, skip, randn(rows, rows, 2 * cols, std=1.5))
            gate, up = z.view[:, :cols], z.view[:, cols:] if gated else None
            y, packed = Mat(rows, cols, dt, cols + pad, skip), Packed(rows, cols, pad, skip, block_rows)
            call = ffn.Activate(dict(type=code, activation=ffn.COPY if act is None else ACT[act], rows=rows, cols=cols, block_rows=block_rows, ldgate=z.ld, ldup=z.ld, ldy=y.ld,
                                     **packed.pitch))
            call.run(gate=z.ptr, up=z.ptr + cols * z.size if gated else None, y=y.ptr, stream=stream(), **packed.ptrs)
            torch.cuda.synchronize()
            what = "%s %s %dx%d pad %d gated %s" % (typ, act, rows, cols, pad, gated)
            value, bound = P.activated(act, gate, up)
            O.check(y.view, (value, bound), what)
            packed.check(value, bound, what)
            assert y.guards(), what
            back = Mat(rows, cols, dt, cols + pad, skip)
            un = ffn.Unpack(dict(type=code, rows=rows, cols=cols, block_rows=block_rows, ldy=back.ld, **packed.pitch))
            un.run(y=back.ptr, stream=stream(), **packed.ptrs)
            torch.cuda.synchronize()
            exact = P.decode(packed.codes.view, packed.by_block(), cols, block_rows)
            O.check(back.view, (exact, exact.abs() * O.E32), what + " back")
            assert back.guards(), what


@pytest.mark.parametrize("block_rows", [1, 128])
def test_codes_are_the_nearest(block_rows):
    """a copy: scales to the bit, codes to the bit but within 2^-22 of a border, what is not finite as NaN, the smallest and largest blocks"""
    rows, cols = 256, 1024
    v = randn(5, rows, cols) * torch.exp2(torch.arange(rows, device=DEV)[:, None] / 2 - 64)
    v[3, 5], v[3, 300], v[200, 700], v[200, 701] = float("inf"), float("-inf"), float("nan"), 1e38
    v[7] = 0
    v[9, :256] = 1e-40
    v[11, 128:256] = 3.4028234e38
    v[12, 1000] = -3.0e38
    p = Packed(rows, cols, block_rows=block_rows)
    ffn.Activate(dict(type=TYPES["f32"][1], activation=ffn.COPY, rows=rows, cols=cols, block_rows=block_rows, **p.pitch)).run(gate=v.data_ptr(), stream=stream(), **p.ptrs)
    back = torch.empty_like(v)
    ffn.Unpack(dict(type=TYPES["f32"][1], rows=rows, cols=cols, block_rows=block_rows, **p.pitch)).run(y=back.data_ptr(), stream=stream(), **p.ptrs)
    torch.cuda.synchronize()
    s = P.scale_of(v.double(), block_rows)
    assert torch.equal(p.by_block().double(), s)
    want, off = P.quantise(v.double() / P.spread(s, rows, cols, block_rows))
    got = p.codes.view.contiguous().view(torch.float8_e4m3fn).double()
    odd = ~torch.isfinite(v)
    assert torch.isnan(got[odd]).all() and torch.isfinite(got[~odd]).all()
    wrong = (got != want) & ~odd & (off > 2.0 ** -22)
    assert not wrong.any(), (got[wrong][:5], want[wrong][:5])
    assert ((got != want) & ~odd).float().mean() < 1e-4
    assert torch.isfinite(back[~odd]).all() and torch.isnan(back[odd]).all()
    assert back[11, 200].item() >= 3.4e38


def test_long_matrices():
    """offsets past 32 bits: codes and plain rows behind 4 GiB"""
    rows, cols = 70000, 32768
    dt, code = TYPES["bf16"]
    x = torch.zeros((rows, cols), dtype=dt, device=DEV)
    x[-5:] = randn(3, 5, cols).to(dt)
    codes, scales = ffn.packed_buffers(rows, cols, DEV)
    ffn.Activate(dict(type=code, activation=ffn.COPY, rows=rows, cols=cols)).run(gate=x.data_ptr(), codes=codes.data_ptr(), scales=scales.data_ptr(), stream=stream())
    back = torch.empty_like(x)
    ffn.Unpack(dict(type=code, rows=rows, cols=cols)).run(codes=codes.data_ptr(), scales=scales.data_ptr(), y=back.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert not back[:-5].any()
    value = x[-5:].double()
    P.check_packed(codes[-5:], scales[:, -5:].t(), value, torch.zeros_like(value), cols)
    exact = P.decode(codes[-5:], scales[:, -5:].t(), cols)
    O.check(back[-5:], (exact, exact.abs() * O.E32))
