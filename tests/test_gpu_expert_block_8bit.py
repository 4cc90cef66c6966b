"""zluda_amd.expert_block in 8 bits, operator by operator: each against the definition in 64 bits of what the one in front of it left; and which calls may follow it."""
import pytest
import torch

import ffn_oracle as O
import packed_oracle as P
from packed_norms import norm_check
from test_gpu_ffn import DEV
from zluda_amd import expert_block

pytestmark = pytest.mark.gpu


def codes_of(packed, cols):
    return packed[0].contiguous().view(torch.float8_e4m3fn).double()[..., :cols]


def check_packed_weights(w, packed):
    e, f, d = w.shape
    for i in range(e):
        v = w[i].double()
        P.check_packed(packed[0][i], packed[1][i][:, :P.blocks(d)], v, torch.zeros_like(v), d, 128, "weights of expert %d" % i)


def check_products(y, x, x_scales, w, offsets, what):
    """y of the experts' rows: x (values, rows x model) with its scales (spread), w packed"""
    e, f, d = w[0].shape[0], y.shape[1], x.shape[1]
    for i in range(e):
        r = slice(offsets[i], offsets[i + 1])
        if offsets[i + 1] > offsets[i]:
            ref = P.scaled_product(x[r], codes_of((w[0][i], None), d), x_scales[r], P.spread(w[1][i].double(), f, d, 128))
            O.check(y[r], ref, "%s, expert %d" % (what, i))
            norm_check(y[r], ref, "%s, expert %d" % (what, i))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,model,features,experts,top", [(1, 64, 96, 4, 2), (77, 200, 264, 3, 1), (300, 256, 320, 16, 4), (700, 512, 704, 8, 2), (1500, 1024, 640, 8, 2)])
def test_operator_by_operator(gpu_api, dtype, tokens, model, features, experts, top):
    block, x, residual, chosen, share, _ = expert_block.example(tokens, model, features, experts, top, dtype=dtype)
    block.pack()
    out = block.forward8(x, residual, chosen, share)
    torch.cuda.synchronize()
    check_packed_weights(block.params["w"], block.w8)
    check_packed_weights(block.params["down"], block.d8)
    h = (x.float() + residual.float()).to(dtype)
    assert torch.equal(block.s, h)
    y, bound = P.rms_forward(h, block.params["norm_weight"], 1e-5)["y"]
    P.check_packed(block.codes_n[0], block.codes_n[1].t(), y, bound, model, what="n")
    # rows of the experts, as the sort leaves them
    flat = chosen.reshape(-1)
    order = torch.argsort(flat, stable=True)
    token, offsets = order // top, [0] + torch.cumsum(torch.bincount(flat, minlength=experts), 0).tolist()
    n, sn = codes_of(block.codes_n, model)[token], P.spread(block.codes_n[1].t().double(), tokens, model)[token]
    check_products(block.z, n, sn, block.w8, offsets, "z")
    P.check_packed(block.codes_h[0], block.codes_h[1].t(), *P.activated("silu", block.z[:, :features], block.z[:, features:]), features, what="h")
    rows = tokens * top
    check_products(block.y, codes_of(block.codes_h, features), P.spread(block.codes_h[1].t().double(), rows, features), block.d8, offsets, "y")
    # out = s + sum of share times y over a token's experts: each product, the sum of `top` and the last addition in 32 bits
    back = torch.zeros(rows, model, dtype=torch.float64, device=DEV)
    back[order] = block.y.double() * share.reshape(-1, 1)[order].double()
    back = back.reshape(tokens, top, model)
    value, mag = block.s.double() + back.sum(1), block.s.double().abs() + back.abs().sum(1)
    O.check(out, (value, (top + 2) * 2 * O.E32 * mag), "out")


def test_no_gradients_of_an_8_bit_pass(gpu_api):
    """what the 8-bit pass leaves is not what backward() reads: it says so, until the next forward()"""
    block, x, residual, chosen, share, dout = expert_block.example(40, 128, 96, 4, 2)
    with pytest.raises(RuntimeError):
        block.backward(dout)
    block.pack()
    block.forward(x, residual, chosen, share)
    first = [t.clone() for t in block.backward(dout)] + [g.clone() for g in block.grads.values()]
    block.forward8(x, residual, chosen, share)
    with pytest.raises(RuntimeError):
        block.backward(dout)
    block.forward(x, residual, chosen, share)
    again = list(block.backward(dout)) + list(block.grads.values())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
