"""The backward products one after the other on the matmuls' 256 x 256 tiles, which the gated layer asks for wherever they fill the chip twice: dW and dX each
for itself, ragged, and dW summed over two parts of the tokens in 32 bits.  On small integers, bit for bit."""
import pytest
import torch

import ffn_probe
from test_gpu_ffn import DEV, TYPES, stream
from test_gpu_ffn_products import integers
from zluda_amd import ffn

pytestmark = pytest.mark.gpu

# which product, tokens, model, features, pitch of x
CASES = [("dw", 70, 4104, 3900, None), ("dw", 200, 8200, 2000, 8208), ("dx", 8200, 4104, 40, None), ("dx", 5000, 7000, 100, None), ("dw", 2900, 4104, 3900, 400000)]


@pytest.mark.parametrize("which,t,d,f,ldx", CASES)
@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_largest_tiles(gpu_api, typ, which, t, d, f, ldx):
    cus = gpu_api.zluda_gemm_device_cu_count()
    assert ffn_probe.load().probe_grad_largest_tiles(d, t if which == "dx" else 2 * f, cus)
    dt, code = TYPES[typ]
    parts = ldx is not None and ffn_probe.load().probe_rows_in_window(t, ldx) < t
    assert parts == (ldx == 400000)
    dh, g, u = integers(1, -3, 3, t, f), integers(2, -2, 3, t, f), integers(3, -3, 3, t, f)
    on = (g > 0).double()
    dz = torch.cat([dh * u * on, dh * g * on], 1)
    ins = {k: v.to(dt) for k, v in dict(dh=dh, gate=g, up=u).items()}
    if which == "dx":
        other = integers(5, -3, 3, 2 * f, d)
        ins["w"], want = other.to(dt), dz @ other
    else:
        other = integers(4, -3, 3, t, d)
        ins["x"], want = torch.empty(t, ldx or d, dtype=dt, device=DEV), dz.t() @ other
        ins["x"][:, :d] = other
    out = torch.full((want.shape[0] + 1, d), float("nan"), dtype=dt, device=DEV)
    call = ffn.GatedBackward(dict(type=code, activation=ffn.RELU, tokens=t, features=f, model=d, dx=which == "dx", dw=which == "dw", **({"ldx": ldx} if ldx else {})))
    ws = torch.full((call.workspace,), 0xFF, dtype=torch.uint8, device=DEV)
    call.run(**{k: v.data_ptr() for k, v in ins.items()}, **{which: out.data_ptr()}, workspace=ws.data_ptr(), workspace_size=ws.numel(), stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(out[:-1].double() + 0.0, want.to(dt).double() + 0.0)     # (+ 0.0: zeros of either sign)
    assert torch.isnan(out[-1]).all()
