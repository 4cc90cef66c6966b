"""Checkpoints of values near the type's largest.  E4M3 rounds [248, 256) times a block's scale up to 256 times, so a finite value may
stand there as 65536 (f16) or 2^128 (bf16, f32), which the type does not have.  What the backward passes read stays finite: such a value counts as
the largest one, and only what was not finite is NaN."""
import pytest
import torch

import ffn_oracle as O
from test_gpu_ffn import DEV, TYPES, Ckpt, randn, scratch, stream
from zluda_amd import ffn

pytestmark = pytest.mark.gpu


def store(typ, x):
    dt, code = TYPES[typ]
    c = Ckpt(*x.shape)
    ffn.Checkpoint(dict(type=code, rows=x.shape[0], cols=x.shape[1])).store(x=x.to(dt).contiguous().data_ptr(), codes=c.codes.ptr, scales=c.scales.ptr, stream=stream())
    torch.cuda.synchronize()
    return c


@pytest.mark.parametrize("t,d,f", [(40, 64, 48), (33, 75, 41), (300, 128, 200)])   # the products in one launch, off 16 bytes, one after the other
@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_x_of_the_gated_backward(gpu_api, typ, t, d, f):
    dt, code = TYPES[typ]
    top = torch.finfo(dt).max
    x = randn(1, t, d).to(dt)
    x[3, 5], x[4, 6], x[5, 40], x[6, 7] = top, -top, top * 0.98, top / 2
    x[7, 9] = float("inf")
    c = store(typ, x)
    values = c.values()
    assert values[3, 5] > top and values[4, 6] < -top and values[6, 7] < top and torch.isnan(values[7, 9])
    values = values.clamp(-top, top)                  # (NaN stays)
    dh, g, u, w = (randn(2 + i, *s, std=std).to(dt) for i, (s, std) in enumerate((((t, f), 1e-3), ((t, f), 1.0), ((t, f), 1.0), ((2 * f, d), d ** -0.5))))
    dx, dw = torch.empty(t, d, dtype=dt, device=DEV), torch.empty(2 * f, d, dtype=dt, device=DEV)
    call = ffn.GatedBackward(dict(type=code, tokens=t, features=f, model=d, x_kept=ffn.KEPT_8BIT))
    ws, _keep = scratch(call)
    call.run(dh=dh.data_ptr(), gate=g.data_ptr(), up=u.data_ptr(), x=c.codes.ptr, x_scales=c.scales.ptr, w=w.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(), stream=stream(), **ws)
    torch.cuda.synchronize()
    ref = O.gated_backward("silu", dh, g, u, values, w)
    O.check(dx, ref["dx"], "dx")
    rest = [j for j in range(d) if j != 9]
    O.check(dw[:, rest], tuple(v[:, rest] for v in ref["dw"]), "dw")
    assert torch.isnan(dw[:, 9]).all()


def test_gate_and_up_of_the_gated_backward(gpu_api):
    """(an f16 value of 65536 is an ordinary one in 32 bits)"""
    t, d, f = 20, 64, 70
    dt, code = TYPES["bf16"]
    top = torch.finfo(dt).max
    gate, up = randn(1, t, f).to(dt), randn(2, t, f).to(dt)
    gate[2, 3], gate[4, 65], up[5, 40], gate[7, 8] = top, -top, top, float("-inf")
    g, u = store("bf16", gate), store("bf16", up)
    dh = randn(3, t, f, std=1e-3).to(dt)
    dz, h = torch.empty(t, 2 * f, dtype=dt, device=DEV), torch.empty(t, f, dtype=dt, device=DEV)
    call = ffn.GatedBackward(dict(type=code, activation=ffn.RELU, tokens=t, features=f, model=d, kept=ffn.KEPT_8BIT, dx=False, dw=False, dz=True, h=True))
    ws, _keep = scratch(call)
    call.run(dh=dh.data_ptr(), gate=g.codes.ptr, gate_scales=g.scales.ptr, up=u.codes.ptr, up_scales=u.scales.ptr, dz=dz.data_ptr(), h=h.data_ptr(), stream=stream(), **ws)
    torch.cuda.synchronize()
    m = torch.finfo(torch.float32).max
    gv, uv = g.values().clamp(-m, m), u.values().clamp(-m, m)
    assert torch.isnan(gv[7, 8])
    gv[7, 8] = 0.0
    ref = O.gated_backward("relu", dh, gv, uv, torch.zeros(t, d, device=DEV), torch.zeros(2 * f, d, device=DEV))
    dz[7, f + 8] = 0.0                                # (dU = dH act(NaN))
    h[7, 8] = 0.0
    O.check(dz, ref["dz"], "dz")
    keep = ref["h"][0].abs() < top                    # (a product of the largest U may be past the type's range by itself)
    O.check(torch.where(keep, h, torch.zeros_like(h)), tuple(torch.where(keep, v, torch.zeros_like(v)) for v in ref["h"]), "h")
    assert keep.sum() >= keep.numel() - 2


@pytest.mark.parametrize("typ", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(9, 100), (6, 700), (4, 1500), (5, 3000), (3, 6000), (3, 9000)])
def test_x_of_the_norm_backward(gpu_api, typ, rows, cols):
    dt, code = TYPES[typ]
    top, m = torch.finfo(dt).max, torch.finfo(torch.float32).max
    x = randn(1, rows, cols).to(dt)
    x[1, 7], x[2, cols - 1] = top, -top
    c = store(typ, x)
    values = c.values()
    assert values[1, 7] > m and values[2, cols - 1] < -m
    values = values.clamp(-m, m)
    dy, mean, rstd = randn(2, rows, cols, std=0.5).to(dt), torch.zeros(rows, device=DEV), torch.ones(rows, device=DEV)
    rstd[1:3] = 1e-30
    dx, dw, db = torch.empty(rows, cols, dtype=dt, device=DEV), torch.empty(cols, dtype=dt, device=DEV), torch.empty(cols, dtype=dt, device=DEV)
    call = ffn.NormBackward(dict(type=code, rows=rows, cols=cols, x_kept=ffn.KEPT_8BIT))
    ws, _keep = scratch(call)
    call.run(x=c.codes.ptr, x_scales=c.scales.ptr, dy=dy.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr(), dx=dx.data_ptr(), dweight=dw.data_ptr(), dbias=db.data_ptr(),
             stream=stream(), **ws)
    torch.cuda.synchronize()
    ref = O.norm_backward(values, dy, None, mean, rstd)
    for k, v in (("dx", dx), ("dweight", dw), ("dbias", db)):
        O.check(v, ref[k], k)
