"""zluda_amd.ffn_block, the operators together as a program uses them: output and gradients against 64-bit autograd, and that it
learns with 8-bit checkpoints what it learns with 16-bit ones."""
import pytest
import torch

from zluda_amd import ffn_block

pytestmark = pytest.mark.gpu


def reference(block, r, dout):
    p = {k: v.double().requires_grad_() for k, v in block.params.items()}
    r = r.double().requires_grad_()
    n = torch.nn.functional.layer_norm(r, (r.shape[1],), p["norm_weight"], p["norm_bias"], 1e-5)
    f = p["down"].shape[1]
    out = r + (torch.nn.functional.silu(n @ p["w"][:f].t()) * (n @ p["w"][f:].t())) @ p["down"].t()
    out.backward(dout.double())
    return out.detach(), r.grad, {k: v.grad for k, v in p.items()}


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("tokens,model,features", [(1, 64, 96), (77, 200, 264), (700, 512, 1400)])
@pytest.mark.parametrize("keep8", [False, True])
def test_block_against_autograd(gpu_api, tokens, model, features, keep8):
    block = ffn_block.FeedForwardBlock(tokens, model, features, keep8=keep8)
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(tokens)
    r, dout = (torch.randn(tokens, model, device="cuda:0", generator=gen).to(torch.bfloat16) for _ in range(2))
    block.params["norm_weight"].add_(torch.randn(model, device="cuda:0", generator=gen) * 0.2)
    out = block.forward(r).clone()
    dr = block.backward(dout)
    torch.cuda.synchronize()
    ro, rr, rg = reference(block, r, dout)
    # bf16 rounds by 2^-8 of a value at most: out passes n, H and its own rounding, a gradient dh, G, U, n, dz (or H) and its own, each
    # a relative error of that size on factors whose relative errors add up
    assert rel(out, ro) <= 3 * 2.0 ** -8
    # an 8-bit checkpoint rounds by 2^-4 at most; r, n, G and U each enter a gradient, and act' of a value off by a
    # relative e is off by less than e
    allowed = 4 * 2.0 ** -4 if keep8 else 6 * 2.0 ** -8
    assert rel(dr, rr) <= allowed
    for k, v in block.grads.items():
        assert rel(v, rg[k]) <= allowed, k
    block.close()


def test_block_learns_with_8_bit_checkpoints(gpu_api):
    tokens, model, features = 500, 128, 344
    torch.manual_seed(0)
    r = torch.randn(tokens, model, device="cuda:0").to(torch.bfloat16)
    target = r.float() + torch.tanh(r.float() @ torch.randn(model, model, device="cuda:0") / model ** 0.5)
    losses = []
    for keep8 in (False, True):
        block = ffn_block.FeedForwardBlock(tokens, model, features, keep8=keep8)
        losses.append(ffn_block.descend(block, r, target, 40, 30.0))
        # r, n, G, U and the rows' two statistics; checkpoints pad rows to 32 and add a byte for each 32
        cols = [-(-c // 32) * 33 if keep8 else 2 * c for c in (model, model, features, features)]
        assert block.kept_bytes() == tokens * (sum(cols) + 8)
        block.close()
    plain, eight = losses
    assert plain[-1] < 0.5 * plain[0] and abs(eight[-1] - plain[-1]) < 0.05 * plain[0]
