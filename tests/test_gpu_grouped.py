"""Products grouped by expert (include/zluda_ffn.h) on the GPU against their definitions in 64 bits (packed_oracle.py): counts around every edge of the tiles,
experts without rows, rows without an expert, any alignment and pitch, guard bytes around and between the rows of every output."""
import pytest
import torch

import ffn_oracle as O
import packed_oracle as P
from test_gpu_ffn import DEV, Mat, TYPES, randn, stream
from test_gpu_packed import Packed
from zluda_amd import ffn

pytestmark = pytest.mark.gpu

# rows of each expert, rows behind the last one's
COUNTS = [([1], 0), ([0, 0, 1], 0), ([3, 0, 5], 2), ([16, 17, 0, 15], 0), ([31, 33, 1, 0, 0, 64], 5), ([65, 63], 0), ([0, 129, 127, 0], 1), ([300, 1, 0, 255, 257], 30),
          ([1] * 70, 0), ([0] * 40 + [7] + [0] * 100 + [130, 2], 3), ([0, 0], 9), ([600], 0)]
SIZES = [(64, 64), (72, 136), (128, 256), (264, 520), (1000, 200), (8, 1024), (328, 2048)]      # features, model


def offsets_of(counts):
    o = [0]
    for n in counts:
        o.append(o[-1] + n)
    return o, torch.tensor(o, dtype=torch.int32, device=DEV)


def run_forward(typ, counts, spare, f, d, pad=0, skip=0, seed=0):
    dt, code = TYPES[typ]
    o, dev = offsets_of(counts)
    rows, e = o[-1] + spare, len(counts)
    x = Mat(rows, d, dt, d + pad, skip, randn(seed + 1, rows, d))
    w = Mat(e * f, d, dt, d + pad, skip, randn(seed + 2, e * f, d, std=d ** -0.5))
    y = Mat(rows, f, dt, f + pad, skip)
    call = ffn.GroupedForward(dict(type=code, rows=rows, experts=e, features=f, model=d, ldx=x.ld, ldw=w.ld, ldy=y.ld))
    ws = torch.empty(max(16, call.workspace), dtype=torch.uint8, device=DEV)
    call.run(offsets=dev.data_ptr(), x=x.ptr, w=w.ptr, y=y.ptr, workspace=ws.data_ptr(), workspace_size=call.workspace, stream=stream())
    torch.cuda.synchronize()
    return o, x, w, y


def untouched(m, first):
    """the rows from `first` on hold the guard bytes still"""
    return bool((m.view[first:].contiguous().view(torch.uint8) == 0xCD).all())


def check_forward(o, x, w, y, f, what):
    assert y.guards() and untouched(y, o[-1]), what
    for e in range(len(o) - 1):
        r = slice(o[e], o[e + 1])
        if o[e + 1] > o[e]:
            O.check(y.view[r], P.product(x.view[r].double(), w.view[e * f:(e + 1) * f].double()), "%s expert %d" % (what, e))


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("counts,spare", COUNTS)
def test_forward(typ, counts, spare):
    for f, d in SIZES if len(counts) < 10 else SIZES[:3]:
        check_forward(*run_forward(typ, counts, spare, f, d), f, "%s %dx%d" % (typ, f, d))


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("f,d,pad,skip", [(64, 64, 8, 8), (65, 72, 0, 0), (72, 63, 0, 0), (30, 17, 3, 1), (129, 128, 1, 0), (128, 136, 0, 4), (1, 1, 0, 0)])
def test_forward_at_any_alignment(typ, f, d, pad, skip):
    for counts, spare in (([5, 0, 70], 3), ([130, 1], 0)):
        check_forward(*run_forward(typ, counts, spare, f, d, pad, skip), f, "%s %dx%d pad %d skip %d" % (typ, f, d, pad, skip))


def pack(rows, cols, block_rows, seed, std=1.0, pad=0, skip=0, experts=1):
    """a packed matrix of random values; with blocks of 128 rows each of `experts` parts starts anew"""
    p = Packed(rows, cols, pad, skip) if block_rows == 1 else None
    v = randn(seed, rows, cols, std=std)
    if block_rows == 1:
        ffn.Activate(dict(type=TYPES["f32"][1], activation=ffn.COPY, rows=rows, cols=cols, **p.pitch)).run(gate=v.data_ptr(), stream=stream(), **p.ptrs)
        return p.codes, p.scales, P.spread(p.by_block().double(), rows, cols)
    f = rows // experts
    ld, lds = ffn.packed_pitches(f, cols, 128)
    codes, scales = Mat(rows, cols, torch.uint8, (cols if pad else ld) + pad, skip), Mat(experts * P.blocks(f), P.blocks(cols), torch.float32, lds + pad)
    call = ffn.Activate(dict(type=TYPES["f32"][1], activation=ffn.COPY, rows=f, cols=cols, block_rows=128, ldcodes=codes.ld, ldcodes_scales=scales.ld))
    for e in range(experts):
        call.run(gate=v[e * f:].data_ptr(), codes=codes.ptr + e * f * codes.ld, scales=scales.ptr + e * P.blocks(f) * scales.ld * 4, stream=stream())
    torch.cuda.synchronize()
    spread = torch.cat([P.spread(scales.view[e * P.blocks(f):(e + 1) * P.blocks(f)].double(), f, cols, 128) for e in range(experts)])
    return codes, scales, spread


def values(codes):
    return codes.view.contiguous().view(torch.float8_e4m3fn).double()


def run_packed(out, counts, spare, f, d, pad=0, skip=0):
    o, dev = offsets_of(counts)
    rows, e = o[-1] + spare, len(counts)
    x, xs, sx = pack(rows, d, 1, 5, 1.0, pad, skip)
    w, ws_, sw = pack(e * f, d, 128, 6, d ** -0.5, pad, skip, e)
    y = Mat(rows, f, TYPES[out][0], f + pad, skip)
    call = ffn.GroupedForward(dict(type=TYPES[out][1], packed=True, rows=rows, experts=e, features=f, model=d, ldx=x.ld, ldx_scales=xs.ld, ldw=w.ld, ldw_scales=ws_.ld, ldy=y.ld))
    ws = torch.empty(max(16, call.workspace), dtype=torch.uint8, device=DEV)
    call.run(offsets=dev.data_ptr(), x=x.ptr, x_scales=xs.ptr, w=w.ptr, w_scales=ws_.ptr, y=y.ptr, workspace=ws.data_ptr(), workspace_size=call.workspace, stream=stream())
    torch.cuda.synchronize()
    what = "%s %dx%d pad %d" % (out, f, d, pad)
    assert y.guards() and untouched(y, o[-1]), what
    vx, vw = values(x), values(w)
    for i in range(e):
        r, q = slice(o[i], o[i + 1]), slice(i * f, (i + 1) * f)
        if o[i + 1] > o[i]:
            O.check(y.view[r], P.scaled_product(vx[r], vw[q], sx[r], sw[q], out == "f32"), "%s expert %d" % (what, i))


@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("counts,spare", COUNTS)
def test_packed_forward(out, counts, spare):
    for f, d in SIZES if len(counts) < 10 else SIZES[:3]:
        run_packed(out, counts, spare, f, d)


@pytest.mark.parametrize("f,d,pad,skip", [(64, 64, 16, 16), (65, 80, 0, 0), (72, 63, 0, 0), (30, 17, 3, 1), (129, 144, 1, 0), (200, 136, 0, 4), (1, 1, 0, 0)])
def test_packed_forward_at_any_alignment(f, d, pad, skip):
    for out, (counts, spare) in (("bf16", ([5, 0, 70], 3)), ("f32", ([130, 1], 0))):
        run_packed(out, counts, spare, f, d, pad, skip)


def run_backward(typ, counts, spare, f, d, pad=0, skip=0, dx=True, dw=True):
    dt, code = TYPES[typ]
    o, dev = offsets_of(counts)
    rows, e = o[-1] + spare, len(counts)
    dy = Mat(rows, f, dt, f + pad, skip, randn(1, rows, f, std=0.1))
    x = Mat(rows, d, dt, d + pad, skip, randn(2, rows, d))
    w = Mat(e * f, d, dt, d + pad, skip, randn(3, e * f, d, std=f ** -0.5))
    gx, gw = Mat(rows, d, dt, d + pad, skip), Mat(e * f, d, dt, d + pad, skip)
    call = ffn.GroupedBackward(dict(type=code, rows=rows, experts=e, features=f, model=d, dx=dx, dw=dw, lddy=dy.ld, ldx=x.ld, ldw=w.ld, lddx=gx.ld, lddw=gw.ld))
    ws = torch.empty(max(16, call.workspace), dtype=torch.uint8, device=DEV)
    call.run(offsets=dev.data_ptr(), dy=dy.ptr, x=x.ptr if dw else None, w=w.ptr if dx else None, dx=gx.ptr if dx else None, dw=gw.ptr if dw else None,
             workspace=ws.data_ptr(), workspace_size=call.workspace, stream=stream())
    torch.cuda.synchronize()
    what = "%s %dx%d pad %d" % (typ, f, d, pad)
    assert gx.guards() and gw.guards(), what
    if dx:
        assert untouched(gx, o[-1]), what
    for i in range(e):
        r, q = slice(o[i], o[i + 1]), slice(i * f, (i + 1) * f)
        g = dy.view[r].double()
        if dx and o[i + 1] > o[i]:
            O.check(gx.view[r], P.product(g, w.view[q].double().t()), "%s dx, expert %d" % (what, i))
        if dw:
            O.check(gw.view[q], P.product(g.t(), x.view[r].double().t()), "%s dw, expert %d" % (what, i))


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("counts,spare", COUNTS)
def test_backward(typ, counts, spare):
    for f, d in SIZES if len(counts) < 10 else SIZES[:3]:
        run_backward(typ, counts, spare, f, d)


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("f,d,pad,skip", [(64, 64, 8, 8), (65, 72, 0, 0), (72, 63, 0, 0), (30, 17, 3, 1), (129, 128, 1, 0), (128, 136, 0, 4), (1, 1, 0, 0)])
def test_backward_at_any_alignment(typ, f, d, pad, skip):
    for counts, spare in (([5, 0, 70], 3), ([130, 1], 0)):
        run_backward(typ, counts, spare, f, d, pad, skip)


def test_one_gradient_alone():
    for dx, dw in ((True, False), (False, True)):
        run_backward("bf16", [20, 0, 150], 4, 136, 264, dx=dx, dw=dw)


def test_no_rows_at_all():
    """dw of experts that have none is zeros"""
    f, d = 40, 72
    dw = torch.full((3 * f, d), 5.0, dtype=torch.bfloat16, device=DEV)
    o = torch.zeros(4, dtype=torch.int32, device=DEV)
    call = ffn.GroupedBackward(dict(type=TYPES["bf16"][1], rows=0, experts=3, features=f, model=d, dx=False))
    ws = torch.empty(max(16, call.workspace), dtype=torch.uint8, device=DEV)
    call.run(offsets=o.data_ptr(), dy=None, x=None, dw=dw.data_ptr(), workspace=ws.data_ptr(), workspace_size=call.workspace, stream=stream())
    torch.cuda.synchronize()
    assert (dw == 0).all()


def test_offsets_that_break_the_rule_stay_inside():
    """decreasing, negative and past the end: other results, nothing outside the matrices"""
    f, d, rows, e = 136, 264, 100, 5
    dt, code = TYPES["bf16"]
    x, w = Mat(rows, d, dt, None, 0, randn(1, rows, d)), Mat(e * f, d, dt, None, 0, randn(2, e * f, d))
    dy = Mat(rows, f, dt, None, 0, randn(3, rows, f))
    for bad in ([0, 90, 20, 100, 50, 100], [-7, 30, 30, 60, 90, 4000], [90, 0, 0, 0, 0, 0], [2 ** 31 - 1] * 6, [-2 ** 31, 2 ** 31 - 1, 0, -1, 5, 2 ** 31 - 1]):
        o = torch.tensor(bad, dtype=torch.int32, device=DEV)
        y, dx, dw = Mat(rows, f, dt), Mat(rows, d, dt), Mat(e * f, d, dt)
        fwd = ffn.GroupedForward(dict(type=code, rows=rows, experts=e, features=f, model=d))
        bwd = ffn.GroupedBackward(dict(type=code, rows=rows, experts=e, features=f, model=d))
        ws = torch.empty(max(16, fwd.workspace, bwd.workspace), dtype=torch.uint8, device=DEV)
        kw = dict(workspace=ws.data_ptr(), workspace_size=ws.numel(), stream=stream())
        fwd.run(offsets=o.data_ptr(), x=x.ptr, w=w.ptr, y=y.ptr, **kw)
        bwd.run(offsets=o.data_ptr(), dy=dy.ptr, x=x.ptr, w=w.ptr, dx=dx.ptr, dw=dw.ptr, **kw)
        torch.cuda.synchronize()
        assert y.guards() and dx.guards() and dw.guards()
