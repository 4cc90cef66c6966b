"""zluda_amd.expert_block, the operators together as a program uses them: output and gradients against 64-bit autograd, and the forward pass in 8 bits."""
import pytest
import torch

from zluda_amd import expert_block

pytestmark = pytest.mark.gpu


def reference(block, x, residual, chosen, share, dout):
    p = {k: v.double().requires_grad_() for k, v in block.params.items()}
    s = (x.float() + residual.float()).to(x.dtype).double().requires_grad_()
    share = share.double().requires_grad_()
    n = s * (s.square().mean(1, keepdim=True) + 1e-5).rsqrt() * p["norm_weight"]
    f, out = block.features, s
    for e in range(block.experts):
        weight = (share * (chosen == e)).sum(1, keepdim=True)
        z = n @ p["w"][e].t()
        out = out + weight * ((torch.nn.functional.silu(z[:, :f]) * z[:, f:]) @ p["down"][e].t())
    out.backward(dout.double())
    return s.detach(), out.detach(), s.grad, share.grad, {k: v.grad for k, v in p.items()}


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,model,features,experts,top", [(1, 64, 96, 4, 2), (77, 200, 264, 3, 1), (300, 256, 320, 16, 4), (700, 512, 704, 8, 2)])
def test_block_against_autograd(gpu_api, dtype, tokens, model, features, experts, top):
    block, x, residual, chosen, share, dout = expert_block.example(tokens, model, features, experts, top, dtype=dtype)
    out = block.forward(x, residual, chosen, share)
    ds, dshare = block.backward(dout)
    torch.cuda.synchronize()
    s, ro, rs, rshare, rg = reference(block, x, residual, chosen, share, dout)
    # a 16-bit type rounds by `unit` of a value at most.  What the experts add passes n, Z, H, Y and its own rounding, a gradient dY, dH (Z, H, n), dZ, dX, dN and
    # its own, each a relative error of that size on factors whose relative errors add up
    unit = torch.finfo(dtype).eps / 2
    assert torch.equal(block.s.double(), s)
    assert rel(out.double() - s, ro - s) <= 6 * unit * (1 + ro.norm().item() / (ro - s).norm().item())
    assert rel(ds, rs) <= 8 * unit and rel(dshare, rshare) <= 8 * unit
    for k, v in block.grads.items():
        assert rel(v, rg[k]) <= 8 * unit, k
    block.pack()
    out8 = block.forward8(x, residual, chosen, share)
    # E4M3 rounds by 2^-4 of a value at most: n, W, H and D
    assert rel(out8.double() - s, ro - s) <= 4 * 2.0 ** -4
