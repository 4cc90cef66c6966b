"""The launch that makes dX and dW together, at sizes where both run their loops: three to sixteen stages of K for dW, one to sixteen shares of dX's K with
several tiles of tokens, sums of the shares, ragged in every direction."""
import pytest
import torch

import ffn_probe
from test_gpu_ffn import DEV, TYPES, check_gated_backward, run_gated_backward, stream
from zluda_amd import ffn

pytestmark = pytest.mark.gpu

SIZES = [(129, 1960, 260), (193, 1544, 312), (129, 392, 1216), (129, 152, 2424), (200, 152, 2452), (257, 1032, 1100), (300, 1024, 1400), (330, 1288, 496), (330, 800, 780),
         (400, 1000, 1040), (449, 2064, 1164), (640, 776, 920), (700, 1032, 804), (1001, 680, 1292)]


@pytest.mark.parametrize("t,d,f", SIZES)
@pytest.mark.parametrize("typ,act", [("bf16", "silu"), ("f16", "gelu")])
@pytest.mark.parametrize("pad", [0, 8])
def test_products_together_in_their_loops(gpu_api, pad, typ, act, t, d, f):
    cus = gpu_api.zluda_gemm_device_cu_count()
    for kept in (ffn.KEPT_PLAIN, ffn.KEPT_8BIT):
        for want in (("dx", "dw"), ("dx", "dw", "dbias"), ("dx", "dw", "dbias", "h", "dz")):
            what = "gated backward %s %s %d x %d x %d pad %d kept %d %s" % (typ, act, t, d, f, pad, kept, ",".join(want))
            print(what, flush=True)
            assert ffn_probe.grad_splits(t, d, f, pad, pad, 2 * f + pad if "dz" in want else None, kept == ffn.KEPT_8BIT, cus)[0] > 0
            outs, ref, _ = run_gated_backward(typ, act, t, d, f, kept, pad, pad, seed=t, want=want)
            check_gated_backward(outs, ref, what)


def integers(seed, low, high, *shape):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return torch.randint(low, high + 1, shape, device=DEV, generator=gen).double()


@pytest.mark.parametrize("t,d,f", SIZES)
@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_products_together_of_integers_are_exact(gpu_api, typ, t, d, f):
    """small integers, ReLU: every product and sum is exact in 32 bits, so that the outputs are the exact sums rounded to the type, bit for bit, and a single
    term too many or too few shows"""
    assert ffn_probe.grad_splits(t, d, f, cus=gpu_api.zluda_gemm_device_cu_count())[0] > 0
    dt, code = TYPES[typ]
    dh, g, u, x, w = integers(1, -3, 3, t, f), integers(2, -2, 3, t, f), integers(3, -3, 3, t, f), integers(4, -3, 3, t, d), integers(5, -3, 3, 2 * f, d)
    on = (g > 0).double()
    dz = torch.cat([dh * u * on, dh * g * on], 1)
    outs = {k: torch.empty(s, dtype=dt, device=DEV) for k, s in (("dx", (t, d)), ("dw", (2 * f, d)), ("dbias", (2 * f,)))}
    call = ffn.GatedBackward(dict(type=code, activation=ffn.RELU, tokens=t, features=f, model=d, bias=True))
    ws = torch.full((call.workspace,), 0xFF, dtype=torch.uint8, device=DEV)
    ins = {k: v.to(dt) for k, v in dict(dh=dh, gate=g, up=u, x=x, w=w).items()}
    call.run(**{k: v.data_ptr() for k, v in {**ins, **outs}.items()}, workspace=ws.data_ptr(), workspace_size=ws.numel(), stream=stream())
    torch.cuda.synchronize()
    for k, want in (("dx", dz @ w), ("dw", dz.t() @ x), ("dbias", dz.sum(0))):
        assert torch.equal(outs[k].double() + 0.0, want.to(dt).double() + 0.0), k     # (+ 0.0: zeros of either sign)
