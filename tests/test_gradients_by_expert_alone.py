"""Gradients by expert, one of the two alone, on a call object that was made for both: which workspace it takes."""
import pytest
import torch

from zluda_amd import abi as K, cublaslt, ffn

SIZES = [(64, 8, 5632, 2048), (692, 2, 4744, 2688), (3459, 16, 3696, 416), (64, 1, 4096, 4096), (2000, 2, 1024, 1024)]      # rows, experts, features, model


def call_of(rows, experts, features, model, **over):
    return ffn.GroupedBackward(dict(type=K.CUDA_R_16BF, rows=rows, experts=experts, features=features, model=model, **over))


@pytest.mark.parametrize("size", SIZES)
def test_workspaces_of_both_and_of_one(size):
    both, dx, dw = call_of(*size), call_of(*size, dw=False), call_of(*size, dx=False)
    assert both.workspace_dx == dx.workspace_dx == dx.workspace == dw.workspace_dx and dw.workspace == 0
    assert both.p.dx.data and both.p.dw.data and dx.p.dx.data and not dx.p.dw.data and not dw.p.dx.data


def test_sizes_where_dx_alone_takes_more():
    assert sum(call_of(*s).workspace_dx > call_of(*s).workspace for s in SIZES) >= 3


@pytest.mark.parametrize("size", [s for s in SIZES if s != (2000, 2, 1024, 1024)])
def test_too_little_for_dx_alone_says_how_much(size):
    call = call_of(*size)
    with pytest.raises(cublaslt.CublasLtError) as e:
        call.run(offsets=64, dy=256, w=512, dx=1024, workspace=4096, workspace_size=call.workspace_dx - 1)
    assert e.value.status == K.CUBLAS_STATUS_ALLOC_FAILED and "%d bytes" % call.workspace_dx in str(e.value)


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES)
def test_one_after_the_other_on_one_object(gpu_api, size):
    """dx alone, dw alone and both, each with the workspace that is named for it, of which nothing behind is written"""
    import ffn_oracle as O
    import packed_oracle as P
    from test_gpu_ffn import DEV, randn, stream
    rows, experts, f, d = size
    o = [rows * i // experts for i in range(experts + 1)]
    offsets = torch.tensor(o, dtype=torch.int32, device=DEV)
    dy, x, w = (randn(i, *shape, std=std).bfloat16() for i, shape, std in ((1, (rows, f), 0.1), (2, (rows, d), 1.0), (3, (experts * f, d), f ** -0.5)))
    call = call_of(*size)
    ws = torch.full((max(call.workspace, call.workspace_dx) + 256,), 0xCD, dtype=torch.uint8, device=DEV)
    args = dict(offsets=offsets.data_ptr(), dy=dy.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), workspace=ws.data_ptr(), stream=stream())
    outs = []
    for with_dx, with_dw, size in ((True, False, call.workspace_dx), (False, True, 0), (True, True, call.workspace)):
        dx, dw = torch.full_like(x, 7), torch.full_like(w, 7)
        ws.fill_(0xCD)
        call.run(dx=dx.data_ptr() if with_dx else None, dw=dw.data_ptr() if with_dw else None, workspace_size=size, **args)
        torch.cuda.synchronize()
        assert (ws[size:] == 0xCD).all() and (with_dx or (dx == 7).all()) and (with_dw or (dw == 7).all())
        outs.append((dx if with_dx else None, dw if with_dw else None))
    for i in range(experts):
        r, q = slice(o[i], o[i + 1]), slice(i * f, (i + 1) * f)
        want_dx, want_dw = P.product(dy[r].double(), w[q].double().t()), P.product(dy[r].double().t(), x[r].double().t())
        for dx, dw in outs:
            if dx is not None:
                O.check(dx[r], want_dx, "dx, expert %d" % i)
            if dw is not None:
                O.check(dw[q], want_dw, "dw, expert %d" % i)
