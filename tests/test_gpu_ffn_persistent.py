"""The gated forward products in tiles of 128 features and 256 tokens, the persistent kernel's wider ones, which large layers run on: last tiles
ragged in both directions, one and several tiles a workgroup, K of one stage, of two, three, four and six, with a tail."""
import pytest
import torch

import ffn_oracle as O
import ffn_probe
from test_gpu_ffn import ACT, DEV, TYPES, Ckpt, Mat, check_gated, randn, stream
from zluda_amd import ffn

pytestmark = pytest.mark.gpu

WIDE = 5     # (index in kGatedTiles)
SIZES = [(497, 64, 10897), (1157, 8, 9750), (1157, 72, 9751), (1751, 136, 9787), (398, 200, 11008), (2741, 328, 4385)]


@pytest.mark.parametrize("t,d,f", SIZES)
@pytest.mark.parametrize("kept", [ffn.KEPT_NONE, ffn.KEPT_PLAIN, ffn.KEPT_8BIT])
@pytest.mark.parametrize("typ,act", [("bf16", "silu"), ("f16", "gelu"), ("bf16", "relu"), ("f16", "silu")])
def test_wide_tiles(gpu_api, typ, act, kept, t, d, f):
    cus = gpu_api.zluda_gemm_device_cu_count()
    assert ffn_probe.gated_tile(t, d, f, cus=cus) == WIDE
    assert ffn_probe.tile_shape(WIDE) == (128, 256, True)
    dt, code = TYPES[typ]
    x, w = Mat(t, d, dt, data=randn(t, t, d)), Mat(2 * f, d, dt, data=randn(t + 1, 2 * f, d, std=1.5 * d ** -0.5))
    # the bias from an even and from an odd element on (Wu's half starts the other way round where the features are odd), and none
    for bias_skip in (0, 1, None):
        what = "gated %s %s %d x %d x %d kept %d bias %s" % (typ, act, t, d, f, kept, bias_skip)
        print(what, flush=True)
        b = None if bias_skip is None else Mat(1, 2 * f, dt, None, bias_skip, randn(t + 2, 1, 2 * f, std=0.3))
        h = Mat(t, f, dt, f + 3, 1)
        ptrs, pitch, g, u = {}, {}, None, None
        if kept == ffn.KEPT_8BIT:
            g, u = Ckpt(t, f, 1), Ckpt(t, f, 2)
            ptrs = dict(gate=g.codes.ptr, gate_scales=g.scales.ptr, up=u.codes.ptr, up_scales=u.scales.ptr)
            pitch = dict(ldgate=g.codes.ld, ldgate_scales=g.scales.ld, ldup=u.codes.ld, ldup_scales=u.scales.ld)
        elif kept == ffn.KEPT_PLAIN:
            g, u = Mat(t, f, dt, f + 8), Mat(t, f, dt, f + 5, 3)
            ptrs, pitch = dict(gate=g.ptr, up=u.ptr), dict(ldgate=g.ld, ldup=u.ld)
        call = ffn.GatedForward(dict(type=code, activation=ACT[act], tokens=t, features=f, model=d, kept=kept, ldh=h.ld, **pitch))
        call.run(x=x.ptr, w=w.ptr, bias=b.ptr if b else None, h=h.ptr, stream=stream(), **ptrs)
        torch.cuda.synchronize()
        check_gated(h, g, u, kept, O.gated_forward(act, x.view, w.view, b.view[0] if b else None), what)


@pytest.mark.parametrize("kept", [ffn.KEPT_NONE, ffn.KEPT_8BIT])
def test_rows_of_wide_tiles_keep_to_themselves(gpu_api, kept):
    """what is not finite in one token's row stays in that row, in tiles with every token and in the last ones"""
    t, d, f = 1157, 136, 9750
    assert ffn_probe.gated_tile(t, d, f, cus=gpu_api.zluda_gemm_device_cu_count()) == WIDE
    dt, code = TYPES["bf16"]
    x, w = randn(1, t, d).to(dt), randn(2, 2 * f, d, std=d ** -0.5).to(dt)
    bad = [0, 255, 700, t - 1]
    x[bad, 7] = float("nan")
    h = torch.empty(t, f, dtype=dt, device=DEV)
    g, u = Ckpt(t, f), Ckpt(t, f)
    ptrs = dict(gate=g.codes.ptr, gate_scales=g.scales.ptr, up=u.codes.ptr, up_scales=u.scales.ptr) if kept else {}
    ffn.GatedForward(dict(type=code, tokens=t, features=f, model=d, kept=kept)).run(x=x.data_ptr(), w=w.data_ptr(), h=h.data_ptr(), stream=stream(), **ptrs)
    torch.cuda.synchronize()
    good = [i for i in range(t) if i not in bad]
    ref = O.gated_forward("silu", x[good], w, None)
    O.check(h[good], ref["h"], "h")
    assert torch.isnan(h[bad]).all()
    if kept:
        assert torch.isnan(g.values()[bad]).all() and torch.isfinite(g.values()[good]).all() and torch.isfinite(u.values()[good]).all()
