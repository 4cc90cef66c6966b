"""zluda_amd.expert_block hands addresses on: tensors of another shape, type, layout or device than the block's are refused before anything is launched."""
import pytest
import torch

from zluda_amd import expert_block

T, D, F, E, TOP = 6, 64, 32, 4, 2


def inputs():
    g = torch.Generator().manual_seed(1)
    rand = lambda: torch.randn(T, D, generator=g).bfloat16()  # noqa: E731
    share, chosen = torch.rand(T, E, generator=g).softmax(1).topk(TOP, 1)
    return dict(x=rand(), residual=rand(), chosen=chosen, share=share)


BAD = [lambda t: t[:-1].contiguous(), lambda t: t.repeat(2, 1), lambda t: t[:, :-1].contiguous(), lambda t: t.half(), lambda t: t.float(),
       lambda t: t.t().contiguous().t(), lambda t: t[:1].expand(T, D), lambda t: t.reshape(1, T, D), lambda t: t.to("meta")]


@pytest.mark.parametrize("which", ["x", "residual"])
@pytest.mark.parametrize("bad", range(len(BAD)))
@pytest.mark.parametrize("call", ["forward", "forward8"])
def test_matrices(which, bad, call):
    block, args = expert_block.ExpertBlock(T, D, F, E, TOP, device="cpu"), inputs()
    args[which] = BAD[bad](args[which])
    with pytest.raises(ValueError, match=which):
        getattr(block, call)(**args)


@pytest.mark.parametrize("bad", range(len(BAD)))
def test_gradient(bad):
    block = expert_block.ExpertBlock(T, D, F, E, TOP, device="cpu")
    block.share = inputs()["share"]          # (as forward() leaves it)
    with pytest.raises(ValueError, match="dout"):
        block.backward(BAD[bad](inputs()["x"]))


@pytest.mark.parametrize("which", ["chosen", "share"])
@pytest.mark.parametrize("call", ["forward", "forward8"])
def test_choices(which, call):
    block = expert_block.ExpertBlock(T, D, F, E, TOP, device="cpu")
    for bad in (lambda t: t[:-1], lambda t: t[:, :1], lambda t: t.reshape(-1), lambda t: torch.cat([t, t])):
        args = inputs()
        args[which] = bad(args[which])
        with pytest.raises(ValueError, match=which):
            getattr(block, call)(**args)
