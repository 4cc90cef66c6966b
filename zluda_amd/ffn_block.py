"""The feed-forward half of a transformer block on this library's operators, forward and backward:

    out = r + (act(n Wg^T) * (n Wu^T)) Wd^T,   n = norm(r)

norm and the gated products through zluda_amd.ffn, the down projection and its two gradients through cublasLtMatmul (the residual is its
C, with beta 1).  `keep8` keeps what the backward pass needs -- r, n, G and U -- as 8-bit checkpoints; H is computed again from G and U.

    python -m zluda_amd.ffn_block      a few steps of gradient descent with 16- and with 8-bit checkpoints, and what they kept
"""
import ctypes as C

import torch

from . import abi, cublaslt, ffn

_TYPES = {torch.bfloat16: abi.CUDA_R_16BF, torch.float16: abi.CUDA_R_16F}
_WORKSPACE = 32 << 20


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


class FeedForwardBlock:
    """One block for a fixed number of tokens.  Parameters: norm_weight, norm_bias (32 bits), w (2 features x model: Wg's rows, then
    Wu's), down (model x features); their gradients after backward(): the same names in `grads`."""

    def __init__(self, tokens, model, features, dtype=torch.bfloat16, activation=ffn.SILU, keep8=True, device="cuda:0", seed=0):
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)
        rand = lambda *s, std: (torch.randn(s, device=device, generator=gen) * std).to(dtype)  # noqa: E731
        empty = lambda *s, t=dtype: torch.empty(s, dtype=t, device=device)  # noqa: E731
        self.keep8 = keep8
        self.params = {"norm_weight": torch.ones(model, device=device), "norm_bias": torch.zeros(model, device=device),
                       "w": rand(2 * features, model, std=model ** -0.5), "down": rand(model, features, std=features ** -0.5)}
        self.grads = {k: torch.empty_like(v) for k, v in self.params.items()}
        typ = _TYPES[dtype]
        kept = ffn.KEPT_8BIT if keep8 else ffn.KEPT_PLAIN
        buffers = lambda cols: ffn.checkpoint_buffers(tokens, cols, device) if keep8 else (empty(tokens, cols), None)  # noqa: E731
        self.gate, self.up = buffers(features), buffers(features)
        self.kept_r, self.kept_n = (buffers(model), buffers(model)) if keep8 else ((None, None), (None, None))
        self.mean, self.rstd = empty(tokens, t=torch.float32), empty(tokens, t=torch.float32)
        self.n, self.h, self.out = empty(tokens, model), empty(tokens, features), empty(tokens, model)
        self.dh, self.dn, self.dr = empty(tokens, features), empty(tokens, model), empty(tokens, model)

        norm = dict(type=typ, weight_type=abi.CUDA_R_32F, rows=tokens, cols=model, x_kept=kept)
        self.norm_forward, self.norm_backward = ffn.NormForward(norm), ffn.NormBackward(norm)
        self.store = ffn.Checkpoint(dict(type=typ, rows=tokens, cols=model))
        gated = dict(type=typ, activation=activation, tokens=tokens, model=model, features=features, kept=kept, x_kept=kept, h=True)
        self.gated_forward, self.gated_backward = ffn.GatedForward(gated), ffn.GatedBackward(gated)
        # row-major matrices are transposed column-major ones
        api = cublaslt.load()
        base = dict(a_type=typ, b_type=typ, c_type=typ, d_type=typ, compute_type=abi.CUBLAS_COMPUTE_32F, scale_type=abi.CUDA_R_32F)
        matmul = lambda **s: cublaslt.MatmulCall(api, dict(base, **s), max_workspace=_WORKSPACE)  # noqa: E731
        self.down = matmul(m=model, n=tokens, k=features, transa=1)               # out^T = down h^T + r^T
        self.down_dh = matmul(m=features, n=tokens, k=model)                      # dh^T = down^T dout^T
        self.down_dw = matmul(m=features, n=model, k=tokens, transb=1)            # ddown^T = h^T dout
        self.workspace = torch.empty(max(_WORKSPACE, self.gated_forward.workspace, self.gated_backward.workspace, self.norm_backward.workspace),
                                     dtype=torch.uint8, device=device)

    def kept_bytes(self):
        """bytes that stay between forward() and backward(), the input r of a block without 8-bit checkpoints among them"""
        t = [self.mean, self.rstd, *self.gate, *self.up] + ([*self.kept_r, *self.kept_n] if self.keep8 else [self.out, self.n])
        return sum(x.numel() * x.element_size() for x in t if x is not None)

    def _matmul(self, call, a, b, beta, c, d):
        one, beta = C.c_float(1.0), C.c_float(beta)
        call.api.check(call.run(one, a.data_ptr(), b.data_ptr(), beta, c.data_ptr(), d.data_ptr(), self.workspace.data_ptr(), _WORKSPACE, _stream()), "cublasLtMatmul")

    def _scratch(self):
        return dict(workspace=self.workspace.data_ptr(), workspace_size=self.workspace.numel(), stream=_stream())

    def forward(self, r):
        p = self.params
        self.r = None if self.keep8 else r
        self.norm_forward.run(x=r.data_ptr(), y=self.n.data_ptr(), weight=p["norm_weight"].data_ptr(), bias=p["norm_bias"].data_ptr(), mean=self.mean.data_ptr(),
                              rstd=self.rstd.data_ptr(), kept=_ptr(self.kept_r[0]), kept_scales=_ptr(self.kept_r[1]), stream=_stream())
        if self.keep8:
            self.store.store(x=self.n.data_ptr(), codes=self.kept_n[0].data_ptr(), scales=self.kept_n[1].data_ptr(), stream=_stream())
        self.gated_forward.run(x=self.n.data_ptr(), w=p["w"].data_ptr(), h=self.h.data_ptr(), gate=_ptr(self.gate[0]), gate_scales=_ptr(self.gate[1]),
                               up=_ptr(self.up[0]), up_scales=_ptr(self.up[1]), **self._scratch())
        self._matmul(self.down, p["down"], self.h, 1.0, r, self.out)
        return self.out

    def backward(self, dout):
        """gradients of sum(dout * out): the parameters' in `grads`, r's is returned"""
        p, g = self.params, self.grads
        n = self.kept_n if self.keep8 else (self.n, None)
        r = self.kept_r if self.keep8 else (self.r, None)
        self._matmul(self.down_dh, p["down"], dout, 0.0, self.dh, self.dh)
        self.gated_backward.run(dh=self.dh.data_ptr(), gate=_ptr(self.gate[0]), gate_scales=_ptr(self.gate[1]), up=_ptr(self.up[0]), up_scales=_ptr(self.up[1]),
                                x=n[0].data_ptr(), x_scales=_ptr(n[1]), w=p["w"].data_ptr(), dx=self.dn.data_ptr(), dw=g["w"].data_ptr(), h=self.h.data_ptr(),
                                **self._scratch())
        self._matmul(self.down_dw, self.h, dout, 0.0, g["down"], g["down"])
        self.norm_backward.run(x=r[0].data_ptr(), x_scales=_ptr(r[1]), dy=self.dn.data_ptr(), mean=self.mean.data_ptr(), rstd=self.rstd.data_ptr(),
                               weight=p["norm_weight"].data_ptr(), add=dout.data_ptr(), dx=self.dr.data_ptr(), dweight=g["norm_weight"].data_ptr(),
                               dbias=g["norm_bias"].data_ptr(), **self._scratch())
        return self.dr

    def close(self):
        for call in (self.down, self.down_dh, self.down_dw):
            call.close()


def descend(block, r, target, steps, rate):
    """gradient descent on mean((out - target)^2) / 2; the losses"""
    losses = []
    for _ in range(steps):
        diff = block.forward(r).float() - target
        losses.append(0.5 * diff.square().mean().item())
        block.backward((diff / block.out.shape[1]).to(r.dtype))
        for k, v in block.params.items():
            v -= (rate / r.shape[0] * block.grads[k].float()).to(v.dtype)
    return losses


if __name__ == "__main__":
    tokens, model, features = 2000, 1024, 2816
    torch.manual_seed(0)
    r = torch.randn(tokens, model, device="cuda:0").to(torch.bfloat16)
    target = r.float() + torch.tanh(r.float() @ torch.randn(model, model, device="cuda:0") / model ** 0.5)
    for keep8 in (False, True):
        block = FeedForwardBlock(tokens, model, features, keep8=keep8)
        losses = descend(block, r, target, 60, 5.0)
        print("%s checkpoints: %.1f MB kept, loss %.4f -> %.4f" % ("8-bit " if keep8 else "16-bit", block.kept_bytes() / 1e6, losses[0], losses[-1]))
        block.close()
