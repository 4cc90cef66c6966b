"""The call objects of zluda_amd.ffn hand on the addresses of the call at hand and nothing of an earlier one."""
import pytest

from zluda_amd import abi, cublaslt, ffn

IV = abi.CUBLAS_STATUS_INVALID_VALUE


def addresses(structure):
    """every pointer in the structure"""
    out = {}
    for name, typ in structure._fields_:
        v = getattr(structure, name)
        if isinstance(v, ffn.zluda_ffn_matrix):
            out.update({name: v.data, name + "_scales": v.scales})
        elif typ is ffn._vp:
            out[name] = v
    return out


SPEC = dict(type=abi.CUDA_R_16BF, tokens=4, features=64, model=32, rows=4, cols=64, kept=ffn.KEPT_8BIT, x_kept=ffn.KEPT_8BIT)
FULL = {
    ffn.GatedForward: dict(x=32, w=64, h=96, bias=128, gate=160, gate_scales=192, up=224, up_scales=256),
    ffn.GatedBackward: dict(dh=32, gate=64, up=96, x=128, w=160, dx=192, dw=224, dbias=256, h=288, dz=320, gate_scales=352, up_scales=384, x_scales=416),
    ffn.NormForward: dict(x=32, y=64, weight=96, bias=128, mean=160, rstd=192, kept=224, kept_scales=256),
    ffn.NormBackward: dict(x=32, dy=64, mean=96, rstd=128, weight=160, add=192, dx=224, dweight=256, dbias=288, x_scales=320),
}


@pytest.mark.parametrize("make", FULL)
def test_a_call_leaves_no_address_behind(make):
    call = make(SPEC)
    if hasattr(call.p, "activation"):   # (refused before anything else is looked at: nothing is launched, with or without a device)
        call.p.activation = 99
    else:
        call.p.cols = 0
    run = lambda **a: refused(call, a)  # noqa: E731
    run(**FULL[make])
    for left_out in FULL[make]:
        args = dict(FULL[make])
        positional = make.run.__code__.co_varnames[1:make.run.__code__.co_argcount - len(make.run.__defaults__)]
        if left_out in positional:
            continue
        run(**FULL[make])
        args.pop(left_out)
        run(**args)
        got = addresses(call.p)
        assert got[left_out] is None, left_out
        assert {k: got[k] for k in args} == args


def refused(call, args):
    with pytest.raises(cublaslt.CublasLtError) as e:
        call.run(**args)
    assert e.value.status == IV


def test_a_kept_product_without_scales_is_refused_the_second_time_too():
    call = ffn.GatedForward(dict(SPEC, tokens=4))
    args = dict(FULL[ffn.GatedForward])
    refused(call, dict(args, x=33))      # (refused for x: nothing is launched)
    for name in ("gate_scales", "up_scales"):
        args.pop(name)
    with pytest.raises(cublaslt.CublasLtError) as e:
        call.run(**args)
    assert e.value.status == IV
