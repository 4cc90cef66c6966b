"""The gated layer's backward pass with G and U kept in one form and X in the other: plain beside 8-bit checkpoints."""
import pytest
import torch

import ffn_oracle as O
import ffn_probe
from test_gpu_ffn import ACT, TYPES, Ckpt, Mat, check_gated_backward, randn, scratch, stream
from zluda_amd import ffn

pytestmark = pytest.mark.gpu

# the products in one launch (a share of dX's K, several), one after the other, rows off 16 bytes, odd widths
SIZES = [(1, 64, 33, 0), (100, 1024, 2816, 0), (257, 1032, 1100, 8), (300, 128, 200, 0), (130, 256, 96, 3), (65, 37, 63, 1)]


@pytest.mark.parametrize("t,d,f,pad", SIZES)
@pytest.mark.parametrize("typ,act", [("bf16", "silu"), ("f16", "gelu")])
@pytest.mark.parametrize("products,x_kept", [(ffn.KEPT_PLAIN, ffn.KEPT_8BIT), (ffn.KEPT_8BIT, ffn.KEPT_PLAIN)])
def test_mixed_forms(gpu_api, products, x_kept, typ, act, t, d, f, pad):
    dt, code = TYPES[typ]
    ins, pitch, vals, keep = {}, {}, {}, []
    for i, (name, n, kept) in enumerate((("gate", f, products), ("up", f, products), ("x", d, x_kept))):
        data = randn(t + i, t, n, std=1.3).to(dt)
        if kept == ffn.KEPT_8BIT:
            m = Ckpt(t, n, pad)
            ffn.Checkpoint(dict(type=code, rows=t, cols=n, ldcodes=m.codes.ld, ldscales=m.scales.ld)).store(x=data.data_ptr(), codes=m.codes.ptr, scales=m.scales.ptr, stream=stream())
            torch.cuda.synchronize()
            ins[name], ins[name + "_scales"], pitch["ld" + name], pitch["ld" + name + "_scales"], vals[name] = m.codes.ptr, m.scales.ptr, m.codes.ld, m.scales.ld, m.values()
        else:
            m = Mat(t, n, dt, n + pad, pad, data)
            ins[name], pitch["ld" + name], vals[name] = m.ptr, m.ld, m.view
        keep += [m, data]
    dh, w = Mat(t, f, dt, f + pad, pad, randn(7, t, f, std=0.5)), Mat(2 * f, d, dt, d + pad, pad, randn(8, 2 * f, d, std=d ** -0.5))
    outs = {"dx": Mat(t, d, dt, d + pad, pad), "dw": Mat(2 * f, d, dt, d + pad, pad), "dbias": Mat(1, 2 * f, dt, None, pad), "h": Mat(t, f, dt, f + pad, pad)}
    call = ffn.GatedBackward(dict(type=code, activation=ACT[act], tokens=t, features=f, model=d, kept=products, x_kept=x_kept, bias=True, h=True, lddh=dh.ld, ldw=w.ld, **pitch,
                                  **{"ld" + k: m.ld for k, m in outs.items() if k != "dbias"}))
    ws, _keep = scratch(call)
    call.run(dh=dh.ptr, w=w.ptr, stream=stream(), **ins, **{k: m.ptr for k, m in outs.items()}, **ws)
    torch.cuda.synchronize()
    check_gated_backward(outs, O.gated_backward(act, dh.view, vals["gate"], vals["up"], vals["x"], w.view), "%s %s" % (typ, (t, d, f)))


def test_sizes_take_both_ways(gpu_api):
    cus = gpu_api.zluda_gemm_device_cu_count()
    shares = [ffn_probe.grad_splits(t, d, f, pad, pad, cus=cus)[0] for t, d, f, pad in SIZES]
    assert 0 in shares and max(shares) > 1
