"""zluda_amd.expert_block at the ends: no tokens at all, one token, one expert for all of them, every expert for each."""
import pytest
import torch

from test_gpu_expert_block import reference, rel
from zluda_amd import expert_block

pytestmark = pytest.mark.gpu


def test_no_tokens(gpu_api):
    """outputs without rows, gradients of zeros"""
    block, x, residual, chosen, share, dout = expert_block.example(0, 64, 96, 4, 2)
    for g in block.grads.values():
        g.fill_(7)
    assert block.forward(x, residual, chosen, share).shape == (0, 64)
    ds, dshare = block.backward(dout)
    block.pack()
    assert block.forward8(x, residual, chosen, share).shape == (0, 64)
    torch.cuda.synchronize()
    assert ds.shape == (0, 64) and dshare.shape == (0, 2) and not any(g.any() for g in block.grads.values())


@pytest.mark.parametrize("tokens,experts,top", [(1, 1, 1), (1, 4, 4), (130, 4, 4), (65, 1, 1)])
def test_few_choices(gpu_api, tokens, experts, top):
    block, x, residual, chosen, share, dout = expert_block.example(tokens, 136, 72, experts, top)
    out = block.forward(x, residual, chosen, share)
    ds, dshare = block.backward(dout)
    torch.cuda.synchronize()
    s, ro, rs, rshare, rg = reference(block, x, residual, chosen, share, dout)
    unit = torch.finfo(x.dtype).eps / 2                        # (bounds as in test_block_against_autograd)
    assert rel(out.double() - s, ro - s) <= 6 * unit * (1 + ro.norm().item() / (ro - s).norm().item())
    assert rel(ds, rs) <= 8 * unit and rel(dshare, rshare) <= 8 * unit
    for k, v in block.grads.items():
        assert rel(v, rg[k]) <= 8 * unit, k


def test_one_expert_of_many(gpu_api):
    """all tokens choose the same one: the others' gradients are zeros"""
    block, x, residual, chosen, share, dout = expert_block.example(100, 128, 64, 5, 1)
    chosen.fill_(3)
    block.forward(x, residual, chosen, share)
    for g in block.grads.values():
        g.fill_(7)
    block.backward(dout)
    torch.cuda.synchronize()
    rg = reference(block, x, residual, chosen, share, dout)[4]
    for k in ("w", "down"):
        assert not block.grads[k][:3].any() and not block.grads[k][4:].any() and rel(block.grads[k], rg[k]) <= 8 * torch.finfo(x.dtype).eps / 2
