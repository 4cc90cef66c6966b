"""A workspace that a call has no use for may lie anywhere: gradients by expert and of the RMS norm."""
import ctypes as C

import pytest
import torch

from test_packed import IV, NOINIT, grouped_grad, rms_grad
from zluda_amd import abi as K, ffn

WANTS = [("grouped_backward", grouped_grad, {}, 0), ("grouped_backward", grouped_grad, dict(features=4096, model=512, dy__ld=4096, x__ld=512, w__ld=512, dx__ld=512, dw__ld=512), 1),
         ("rms_backward", rms_grad, dict(rows=1), 0), ("rms_backward", rms_grad, dict(rows=4000), 1), ("rms_backward", rms_grad, dict(rows=4000, dweight=None), 0)]


@pytest.mark.parametrize("name,make,over,wants", WANTS)
def test_alignment_counts_where_there_is_a_use(api, name, make, over, wants):
    if torch.cuda.is_available():
        pytest.skip("there is a device")
    p, n, lib = make(**over), C.c_size_t(), ffn.load()
    assert getattr(lib, "zluda_ffn_%s_workspace" % name)(C.byref(p), C.byref(n)) == 0 and (n.value > 0) == bool(wants)
    for off in (0, 4, 8):
        assert getattr(lib, "zluda_ffn_" + name)(C.byref(p), (1 << 20) + off, 1 << 40, None) == (IV if wants and off else NOINIT)


@pytest.mark.gpu
def test_gradients_beside_a_workspace_of_no_use(gpu_api):
    import ffn_oracle as O
    import packed_oracle as P
    from test_gpu_ffn import DEV, randn, stream
    bf, f, d, rows = torch.bfloat16, 130, 72, 50                # (a width that is no multiple of eight: no shares)
    offsets, raw = torch.tensor([0, 20, 50], dtype=torch.int32, device=DEV), torch.full((4096,), 0xCD, dtype=torch.uint8, device=DEV)
    dy, x, w = randn(1, rows, f).to(bf), randn(2, rows, d).to(bf), randn(3, 2 * f, d).to(bf)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    call = ffn.GroupedBackward(dict(type=K.CUDA_R_16BF, rows=rows, experts=2, features=f, model=d))
    assert call.workspace == 0
    call.run(offsets=offsets.data_ptr(), dy=dy.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(), workspace=raw.data_ptr() + 8, workspace_size=4088,
             stream=stream())
    h, gy = randn(4, 3, 1000).to(bf), randn(5, 3, 1000).to(bf)
    rstd, gx, gw = h.float().square().mean(1).rsqrt(), torch.empty_like(h), torch.empty(1000, dtype=bf, device=DEV)
    ffn.RmsBackward(dict(type=K.CUDA_R_16BF, rows=3, cols=1000)).run(h=h.data_ptr(), dy=gy.data_ptr(), rstd=rstd.data_ptr(), dx=gx.data_ptr(), dweight=gw.data_ptr(),
                                                                     workspace=raw.data_ptr() + 4, workspace_size=4092, stream=stream())
    torch.cuda.synchronize()
    for r, q in ((slice(0, 20), slice(0, f)), (slice(20, 50), slice(f, 2 * f))):
        O.check(dx[r], P.product(dy[r].double(), w[q].double().t()), "dx")
        O.check(dw[q], P.product(dy[r].double().t(), x[r].double().t()), "dw")
    ref = P.rms_backward(h, gy, None, rstd)
    O.check(gx, ref["dx"], "dx of the norm")
    O.check(gw, ref["dweight"], "dweight")
    assert (raw == 0xCD).all()
