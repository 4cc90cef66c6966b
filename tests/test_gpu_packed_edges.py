"""Products by expert and norms where one row must not reach another, on large tiles, and their gradients against differences of the forward pass."""
import pytest
import torch

import ffn_oracle as O
import packed_oracle as P
from test_gpu_ffn import DEV, Mat, TYPES, randn, stream
from test_gpu_grouped import check_forward, offsets_of, pack, run_backward, run_forward, untouched
from zluda_amd import cublaslt, ffn

pytestmark = pytest.mark.gpu
BF = TYPES["bf16"]


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("counts,spare,f,d", [([1100, 0, 900, 1500, 3, 290, 256, 500], 40, 5640, 2056), ([1500, 2500, 0, 257], 0, 1000, 4104), ([8000, 5], 0, 520, 1032),
                                              ([64] * 60 + [0, 900], 7, 2824, 1000)])
def test_large_tiles(typ, counts, spare, f, d):
    run_backward(typ, counts, spare, f, d)
    check_forward(*run_forward(typ, counts, spare, f, d), f, "%s %dx%d" % (typ, f, d))


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("counts,spare,f,d", [([9, 7, 8, 0, 10, 8, 14, 8], 0, 5632, 2048), ([40, 0, 37, 200], 23, 2816, 1032), ([64], 0, 4096, 4096), ([692], 8, 4744, 520),
                                              ([3, 1], 0, 2048, 136), ([700, 1, 600, 699], 5, 4096, 512)])
def test_shares_of_a_long_k(typ, counts, spare, f, d):
    """few tiles of dx with a long K: shares of it, summed up behind; nothing is written past the workspace that was asked for, and less of it is refused"""
    dt, code = TYPES[typ]
    o, dev = offsets_of(counts)
    rows, e = o[-1] + spare, len(counts)
    dy, x, w = Mat(rows, f, dt, None, 0, randn(1, rows, f, std=0.1)), Mat(rows, d, dt, None, 0, randn(2, rows, d)), Mat(e * f, d, dt, None, 0, randn(3, e * f, d, std=f ** -0.5))
    dx, dw = Mat(rows, d, dt, d + 8), Mat(e * f, d, dt)
    call = ffn.GroupedBackward(dict(type=code, rows=rows, experts=e, features=f, model=d, lddx=dx.ld))
    assert call.workspace > 0
    ws = torch.full((call.workspace + 4096,), 0xCD, dtype=torch.uint8, device=DEV)
    args = dict(offsets=dev.data_ptr(), dy=dy.ptr, x=x.ptr, w=w.ptr, dx=dx.ptr, dw=dw.ptr, stream=stream())
    for bad in (dict(workspace=ws.data_ptr(), workspace_size=call.workspace - 1), dict(workspace=None, workspace_size=call.workspace), dict()):
        with pytest.raises(cublaslt.CublasLtError):
            call.run(**args, **bad)
    call.run(**args, workspace=ws.data_ptr(), workspace_size=call.workspace)
    torch.cuda.synchronize()
    assert dx.guards() and dw.guards() and untouched(dx, o[-1]) and bool((ws[call.workspace:] == 0xCD).all())
    for i in range(e):
        r, q = slice(o[i], o[i + 1]), slice(i * f, (i + 1) * f)
        if counts[i]:
            O.check(dx.view[r], P.product(dy.view[r].double(), w.view[q].double().t()), "dx, expert %d" % i)
        O.check(dw.view[q], P.product(dy.view[r].double().t(), x.view[r].double().t()), "dw, expert %d" % i)


@pytest.mark.parametrize("f,d", [(64, 72), (40, 33)])
def test_most_experts(f, d):
    """as many experts as there may be, few of which have rows"""
    counts = [0] * 4096
    for e, n in ((0, 3), (63, 1), (64, 2), (1000, 70), (2047, 1), (2048, 130), (4094, 5), (4095, 1)):
        counts[e] = n
    o, dev = offsets_of(counts)
    rows, live = o[-1] + 2, [e for e in range(4096) if counts[e]]
    x, dy, w = randn(1, rows, d).to(BF[0]), randn(2, rows, f).to(BF[0]), randn(3, 4096 * f, d, std=d ** -0.5).to(BF[0])
    y, dx, dw = torch.full_like(dy, 7), torch.full_like(x, 7), torch.full_like(w, 7)
    spec = dict(type=BF[1], rows=rows, experts=4096, features=f, model=d)
    fwd, bwd = ffn.GroupedForward(spec), ffn.GroupedBackward(spec)
    ws = torch.empty(max(16, bwd.workspace), dtype=torch.uint8, device=DEV)
    fwd.run(offsets=dev.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), y=y.data_ptr(), stream=stream())
    bwd.run(offsets=dev.data_ptr(), dy=dy.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(), workspace=ws.data_ptr(), workspace_size=ws.numel(),
            stream=stream())
    torch.cuda.synchronize()
    for e in live:
        r, q = slice(o[e], o[e + 1]), slice(e * f, (e + 1) * f)
        O.check(y[r], P.product(x[r].double(), w[q].double()), "y")
        O.check(dx[r], P.product(dy[r].double(), w[q].double().t()), "dx")
        O.check(dw[q], P.product(dy[r].double().t(), x[r].double().t()), "dw")
    assert (y[-2:] == 7).all() and (dx[-2:] == 7).all()
    others = dw.view(4096, f, d)[[e for e in range(4096) if not counts[e]]]
    assert not others.any()


BAD = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("counts,spare,f,d", [([5, 3, 0, 9], 4, 72, 136), ([130, 40, 300], 20, 264, 264), ([2000, 1, 3000, 300], 100, 2056, 2056), ([5, 3, 0, 9], 4, 63, 65)])
@pytest.mark.parametrize("bad", BAD)
def test_rows_keep_to_themselves(counts, spare, f, d, bad):
    """infinities and NaN in one row, in one expert's matrix, and in the rows without an expert change nothing else"""
    o, dev = offsets_of(counts)
    rows, e = o[-1] + spare, len(counts)
    x, dy, w = randn(1, rows, d).to(BF[0]), randn(2, rows, f).to(BF[0]), randn(3, e * f, d, std=d ** -0.5).to(BF[0])
    spec = dict(type=BF[1], rows=rows, experts=e, features=f, model=d)
    fwd, bwd = ffn.GroupedForward(spec), ffn.GroupedBackward(spec)
    ws = torch.empty(max(16, bwd.workspace), dtype=torch.uint8, device=DEV)

    def run():
        y, dx, dw = torch.zeros_like(dy), torch.zeros_like(x), torch.zeros_like(w)
        fwd.run(offsets=dev.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), y=y.data_ptr(), stream=stream())
        bwd.run(offsets=dev.data_ptr(), dy=dy.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(), workspace=ws.data_ptr(), workspace_size=ws.numel(), stream=stream())
        torch.cuda.synchronize()
        return y, dx, dw.view(e, f, d)
    y0, dx0, dw0 = run()
    row, expert = o[1] - 1, 0                               # the last row of expert 0, next to the first of the next one
    x[row, ::3], dy[row, 1::5] = bad, bad
    x[o[-1]:], dy[o[-1]:] = bad, bad
    w[-f + 1::7] = bad                                      # the last expert's
    y, dx, dw = run()
    others = [r for r in range(o[-2]) if r != row]
    assert torch.equal(y[others], y0[others]) and torch.equal(dx[others], dx0[others]) and torch.equal(y[o[-1]:], y0[o[-1]:])
    assert torch.equal(dw[1:], dw0[1:])
    assert not y[row].isfinite().any() and not dx[row].isfinite().any()
    assert not dw[expert, :, ::3].isfinite().any() and not dw[expert, 1::5].isfinite().any()
    assert not y[o[-2]:o[-1], 1::7].isfinite().any()
    keep = torch.ones(f, dtype=torch.bool, device=DEV)
    keep[1::7] = False
    assert torch.equal(y[o[-2]:o[-1], keep], y0[o[-2]:o[-1], keep])


@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_packed_rows_keep_to_themselves(out):
    counts, f, d = [5, 130, 0, 9, 300], 264, 400
    o, dev = offsets_of(counts)
    rows, e = o[-1] + 3, len(counts)
    x, xs, _ = pack(rows, d, 1, 5)
    w, ws, _ = pack(e * f, d, 128, 6, d ** -0.5, experts=e)
    call = ffn.GroupedForward(dict(type=TYPES[out][1], packed=True, rows=rows, experts=e, features=f, model=d, ldx=x.ld, ldx_scales=xs.ld, ldw=w.ld, ldw_scales=ws.ld))

    def run():
        y = torch.zeros((rows, f), dtype=TYPES[out][0], device=DEV)
        call.run(offsets=dev.data_ptr(), x=x.ptr, x_scales=xs.ptr, w=w.ptr, w_scales=ws.ptr, y=y.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        return y
    y0 = run()
    x.view[4, 77] = 0x7F                                    # NaN
    x.view[o[-1]:] = 0x7F
    xs.view[:, 6] = float("nan")
    xs.view[:, o[-1]:rows] = float("inf")
    y = run()
    others = [r for r in range(rows) if r not in (4, 6)]
    assert torch.equal(y[others], y0[others]) and y[4].isnan().all() and y[6].isnan().all()


@pytest.mark.parametrize("counts,f,d", [([20, 0, 100, 3], 200, 64), ([100, 33], 136, 56), ([7, 1], 63, 33)])
def test_gradients_of_experts_are_differences(counts, f, d):
    """the product is linear in each operand and these are small integers, so that differences of the forward pass are exact"""
    o, dev = offsets_of(counts)
    rows, e = o[-1], len(counts)

    def ints(seed, most, *s):
        gen = torch.Generator(device=DEV)
        gen.manual_seed(seed)
        return torch.randint(-most, most + 1, s, device=DEV, generator=gen).to(BF[0])
    x, w, dy, vx, vw = ints(1, 2, rows, d), ints(2, 1, e * f, d), ints(3, 1, rows, f), ints(4, 1, rows, d), ints(5, 1, e * f, d)
    spec = dict(type=BF[1], rows=rows, experts=e, features=f, model=d)
    fwd, bwd = ffn.GroupedForward(spec), ffn.GroupedBackward(spec)
    ws = torch.empty(max(16, bwd.workspace), dtype=torch.uint8, device=DEV)

    def loss(x, w):
        y = torch.empty_like(dy)
        fwd.run(offsets=dev.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), y=y.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        assert y.abs().max() <= 256                         # (integers up to here are bfloat16 values)
        return (y.double() * dy.double()).sum()
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    bwd.run(offsets=dev.data_ptr(), dy=dy.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(), workspace=ws.data_ptr(), workspace_size=ws.numel(), stream=stream())
    torch.cuda.synchronize()
    assert dx.abs().max() <= 256 and dw.abs().max() <= 256
    assert loss(x + vx, w) - loss(x, w) == (dx.double() * vx.double()).sum()
    assert loss(x, w + vw) - loss(x, w) == (dw.double() * vw.double()).sum()


@pytest.mark.parametrize("rows,cols", [(1, 200), (37, 1001), (64, 4096)])
def test_gradients_of_the_norm_are_differences(rows, cols):
    x, dy, v = randn(1, rows, cols), randn(2, rows, cols), randn(3, rows, cols)
    weight, vw = 1 + 0.2 * randn(4, cols), randn(5, cols)
    spec = dict(type=TYPES["f32"][1], weight_type=TYPES["f32"][1], rows=rows, cols=cols)
    fwd, bwd = ffn.RmsForward(spec), ffn.RmsBackward(spec)
    rstd = torch.empty(rows, device=DEV)

    def own(x, w):
        y = torch.empty_like(x)
        fwd.run(x=x.data_ptr(), weight=w.data_ptr(), y=y.data_ptr(), rstd=rstd.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        return (y.double() * dy.double()).sum().item(), (y.double() * dy.double()).norm().item()

    def plain(x, w):
        x, w = x.double(), w.double()
        return (x * (x.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w * dy.double()).sum().item()
    own(x, weight)
    dx, dw = torch.empty_like(x), torch.empty(cols, device=DEV)
    ws = torch.empty(max(16, bwd.workspace), dtype=torch.uint8, device=DEV)
    bwd.run(h=x.data_ptr(), dy=dy.data_ptr(), rstd=rstd.data_ptr(), weight=weight.data_ptr(), dx=dx.data_ptr(), dweight=dw.data_ptr(), workspace=ws.data_ptr(), workspace_size=ws.numel(),
            stream=stream())
    torch.cuda.synchronize()
    h = 2.0 ** -6
    for grad, at in (((dx.double() * v.double()).sum().item(), lambda t: (x + t * v, weight)), ((dw.double() * vw.double()).sum().item(), lambda t: (x, weight + t * vw))):
        (hi, size), (lo, _) = own(*at(h)), own(*at(-h))
        q = [(plain(*at(t)) - plain(*at(-t))) / (2 * t) for t in (h, 2 * h)]
        # a quotient over h is off by a multiple of h^2, so that those over h and 2 h differ by three times as much; the inputs x + t v (2^-24 of them), each value of
        # y and the gradients' own are off by a few 2^-24, independent of each other (a norm; the row's common factor, the number of a row's columns, by the root of it)
        bound = abs(q[1] - q[0]) + 8 * O.E32 * size * cols ** 0.5 / h
        assert abs((hi - lo) / (2 * h) - grad) <= bound, (rows, cols, (hi - lo) / (2 * h), grad, bound)
