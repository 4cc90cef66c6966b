"""A backward pass of the gated layer gives its bits again: whatever another call left in the workspace and in the outputs, and whatever the
call object ran in between."""
import pytest
import torch

from test_gpu_ffn import DEV, TYPES, randn, stream
from zluda_amd import ffn

pytestmark = pytest.mark.gpu


# products in one launch (dx in one share of K, in several) and one after the other, 16-byte rows and none
@pytest.mark.parametrize("t,d,f", [(5, 64, 48), (100, 1024, 2816), (1001, 1024, 2816), (300, 128, 200), (77, 75, 41)])
@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_gated_backward_repeats_its_bits(gpu_api, typ, t, d, f):
    dt, code = TYPES[typ]
    sets = [[randn(10 * s + i, *shape, std=std).to(dt) for i, (shape, std) in enumerate((((t, f), 0.5), ((t, f), 1.3), ((t, f), 1.3), ((t, d), 1.0), ((2 * f, d), d ** -0.5)))]
            for s in range(2)]
    call = ffn.GatedBackward(dict(type=code, tokens=t, features=f, model=d, bias=True, h=True))
    outs = {k: torch.empty(s, dtype=dt, device=DEV) for k, s in (("dx", (t, d)), ("dw", (2 * f, d)), ("dbias", (2 * f,)), ("h", (t, f)))}
    ws = torch.empty(call.workspace, dtype=torch.uint8, device=DEV)

    def run(inputs):
        call.run(**{k: v.data_ptr() for k, v in zip(("dh", "gate", "up", "x", "w"), inputs)}, **{k: v.data_ptr() for k, v in outs.items()}, workspace=ws.data_ptr(),
                 workspace_size=ws.numel(), stream=stream())
        torch.cuda.synchronize()
        return {k: v.clone() for k, v in outs.items()}

    ws.zero_()
    first = run(sets[0])
    other = run(sets[1])
    assert all(torch.isfinite(v.float()).all() and not torch.equal(v, first[k]) for k, v in other.items())
    for byte in (None, 0xFF, 0x00):
        if byte is not None:
            ws.fill_(byte)
            for v in outs.values():
                v.fill_(float("nan"))
        again = run(sets[0])
        assert all(torch.equal(v, first[k]) for k, v in again.items()), byte
