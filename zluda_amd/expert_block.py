"""A feed-forward layer of experts behind an RMS norm on this library's operators, forward and backward, and forward in 8 bits:

    s = x + residual,  n = rms(s),  out = s + sum over a token's experts e of share_e * D_e (act(n G_e^T) * (n U_e^T))

Which experts a token has, and their shares, is the caller's (a router's) choice: `chosen` and `share`, tokens x top.  Rows are sorted by expert and brought back by
torch; norm, products by expert, activation and all their gradients go through zluda_amd.ffn.

    python -m zluda_amd.expert_block      a forward and a backward pass, and how far the 8-bit forward pass is from the 16-bit one
"""
import torch

from . import abi, ffn

_TYPES = {torch.bfloat16: abi.CUDA_R_16BF, torch.float16: abi.CUDA_R_16F}


def _stream():
    return torch.cuda.current_stream().cuda_stream


class ExpertBlock:
    """One layer for a fixed number of tokens.  Parameters: norm_weight (32 bits), w (experts x 2 features x model: G's rows, then U's), down (experts x model x
    features); their gradients after backward(): the same names in `grads`."""

    def __init__(self, tokens, model, features, experts, top=2, dtype=torch.bfloat16, activation=ffn.SILU, device="cuda:0", seed=0):
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)
        rand = lambda *s, std: (torch.randn(s, device=device, generator=gen) * std).to(dtype)  # noqa: E731
        empty = lambda *s, t=dtype: torch.empty(s, dtype=t, device=device)  # noqa: E731
        self.top, self.experts, self.features, self.device, self.shape = top, experts, features, device, (tokens, model)
        rows, typ = tokens * top, _TYPES[dtype]
        self.params = {"norm_weight": torch.ones(model, device=device), "w": rand(experts, 2 * features, model, std=model ** -0.5),
                       "down": rand(experts, model, features, std=features ** -0.5)}
        self.grads = {k: torch.empty_like(v) for k, v in self.params.items()}
        self.s, self.n, self.rstd, self.ds = empty(tokens, model), empty(tokens, model), empty(tokens, t=torch.float32), empty(tokens, model)
        self.z, self.h, self.y = empty(rows, 2 * features), empty(rows, features), empty(rows, model)
        self.dz, self.dh, self.dx = empty(rows, 2 * features), empty(rows, features), empty(rows, model)

        norm = dict(type=typ, weight_type=abi.CUDA_R_32F, rows=tokens, cols=model)
        up = dict(type=typ, rows=rows, experts=experts, features=2 * features, model=model)
        down = dict(type=typ, rows=rows, experts=experts, features=model, model=features)
        halves = dict(type=typ, rows=rows, cols=features, activation=activation, ldgate=2 * features, ldup=2 * features)
        self.norm_forward, self.norm_backward = ffn.RmsForward(norm), ffn.RmsBackward(norm)
        self.activate = ffn.Activate(halves)
        self.activate_backward = ffn.GatedBackward(dict(halves, tokens=rows, features=features, model=model, kept=ffn.KEPT_PLAIN, dx=False, dw=False, dz=True))
        self.up, self.up_backward = ffn.GroupedForward(up), ffn.GroupedBackward(up)
        self.down, self.down_backward = ffn.GroupedForward(down), ffn.GroupedBackward(down)
        self.up8, self.down8 = ffn.GroupedForward(dict(up, packed=True)), ffn.GroupedForward(dict(down, packed=True))
        calls = (self.norm_backward, self.activate_backward, self.up, self.up_backward, self.down, self.down_backward, self.up8, self.down8)
        self.workspace = torch.empty(max(16, *(c.workspace for c in calls)), dtype=torch.uint8, device=device)
        self.codes_n, self.codes_h = ffn.packed_buffers(tokens, model, device), ffn.packed_buffers(rows, features, device)
        self.share = None

    def _check(self, chosen=None, share=None, **matrices):
        """the operators take addresses: what they are not told must be so"""
        for name, t in matrices.items():
            if tuple(t.shape) != self.shape or t.dtype != self.s.dtype or t.device != self.s.device or not t.is_contiguous():
                raise ValueError("%s: a contiguous tensor of %d x %d, %s, on %s" % (name, *self.shape, self.s.dtype, self.s.device))
        for name, t in (("chosen", chosen), ("share", share)):
            if t is not None and tuple(t.shape) != (self.shape[0], self.top):
                raise ValueError("%s: %d x %d" % (name, self.shape[0], self.top))

    def _scratch(self):
        return dict(workspace=self.workspace.data_ptr(), workspace_size=self.workspace.numel(), stream=_stream())

    def _sort(self, chosen):
        """the token of each row, rows sorted by expert, and where the experts' rows start"""
        self.order = torch.argsort(chosen.reshape(-1), stable=True)
        self.token = self.order // self.top
        self.offsets = torch.zeros(self.experts + 1, dtype=torch.int32, device=self.device)
        self.offsets[1:] = torch.cumsum(torch.bincount(chosen.reshape(-1), minlength=self.experts), 0)

    def _bring_back(self, base, rows, share=None):
        """base + the rows of each token, in 32 bits"""
        rows = rows.float() if share is None else rows.float() * share.reshape(-1, 1)[self.order]
        back = torch.empty_like(rows)
        back[self.order] = rows
        return (base.float() + back.reshape(base.shape[0], self.top, base.shape[1]).sum(1)).to(base.dtype)

    def forward(self, x, residual, chosen, share):
        self._check(chosen, share, x=x, residual=residual)
        self._sort(chosen)
        p, offsets = self.params, self.offsets.data_ptr()
        self.norm_forward.run(x=x.data_ptr(), residual=residual.data_ptr(), weight=p["norm_weight"].data_ptr(), sum=self.s.data_ptr(), y=self.n.data_ptr(),
                              rstd=self.rstd.data_ptr(), stream=_stream())
        self.rows = self.n[self.token]
        self.up.run(offsets=offsets, x=self.rows.data_ptr(), w=p["w"].data_ptr(), y=self.z.data_ptr(), **self._scratch())
        self.activate.run(gate=self.z.data_ptr(), up=self.z[:, self.features:].data_ptr(), y=self.h.data_ptr(), stream=_stream())
        self.down.run(offsets=offsets, x=self.h.data_ptr(), w=p["down"].data_ptr(), y=self.y.data_ptr(), **self._scratch())
        self.share = share
        return self._bring_back(self.s, self.y, share)

    def backward(self, dout):
        """gradients of sum(dout * out) of the forward() before it: the parameters' in `grads`; x's (and residual's) and share's are returned"""
        if self.share is None:
            raise RuntimeError("backward() reads what forward() left: there was none, or forward8() has written over it")
        self._check(dout=dout)
        p, g, offsets = self.params, self.grads, self.offsets.data_ptr()
        rows = dout[self.token].float()
        dshare = torch.empty(self.order.numel(), device=self.device)
        dshare[self.order] = (rows * self.y.float()).sum(1)
        dy = (rows * self.share.reshape(-1, 1)[self.order]).to(dout.dtype)
        self.down_backward.run(offsets=offsets, dy=dy.data_ptr(), x=self.h.data_ptr(), w=p["down"].data_ptr(), dx=self.dh.data_ptr(), dw=g["down"].data_ptr(), **self._scratch())
        self.activate_backward.run(dh=self.dh.data_ptr(), gate=self.z.data_ptr(), up=self.z[:, self.features:].data_ptr(), dz=self.dz.data_ptr(), **self._scratch())
        self.up_backward.run(offsets=offsets, dy=self.dz.data_ptr(), x=self.rows.data_ptr(), w=p["w"].data_ptr(), dx=self.dx.data_ptr(), dw=g["w"].data_ptr(), **self._scratch())
        dn = self._bring_back(torch.zeros_like(self.n), self.dx)
        self.norm_backward.run(h=self.s.data_ptr(), dy=dn.data_ptr(), rstd=self.rstd.data_ptr(), weight=p["norm_weight"].data_ptr(), add=dout.data_ptr(), dx=self.ds.data_ptr(),
                               dweight=g["norm_weight"].data_ptr(), **self._scratch())
        return self.ds, dshare.reshape(self.share.shape)

    def pack(self):
        """the experts' matrices in 8 bits, with a scale for each 128 x 128"""
        def packed(w):
            e, f, d = w.shape
            call = ffn.Activate(dict(type=_TYPES[w.dtype], activation=ffn.COPY, rows=f, cols=d, block_rows=ffn.PACK))
            parts = [ffn.packed_buffers(f, d, self.device, ffn.PACK) for _ in range(e)]
            codes, scales = torch.stack([c for c, _ in parts]), torch.stack([s for _, s in parts])
            for i in range(e):
                call.run(gate=w[i].data_ptr(), codes=codes[i].data_ptr(), scales=scales[i].data_ptr(), stream=_stream())
            return codes, scales
        self.w8, self.d8 = packed(self.params["w"]), packed(self.params["down"])

    def forward8(self, x, residual, chosen, share):
        """forward() with both products in 8 bits; pack() first, and again when the parameters have changed"""
        self._check(chosen, share, x=x, residual=residual)
        self.share = None  # (z and y are what backward() would read)
        self._sort(chosen)
        offsets, (nc, ns), (hc, hs) = self.offsets.data_ptr(), self.codes_n, self.codes_h
        self.norm_forward.run(x=x.data_ptr(), residual=residual.data_ptr(), weight=self.params["norm_weight"].data_ptr(), sum=self.s.data_ptr(), codes=nc.data_ptr(),
                              scales=ns.data_ptr(), stream=_stream())
        rows, scales = nc[self.token], ns[:, self.token].contiguous()
        self.up8.run(offsets=offsets, x=rows.data_ptr(), x_scales=scales.data_ptr(), w=self.w8[0].data_ptr(), w_scales=self.w8[1].data_ptr(), y=self.z.data_ptr(), **self._scratch())
        self.activate.run(gate=self.z.data_ptr(), up=self.z[:, self.features:].data_ptr(), codes=hc.data_ptr(), scales=hs.data_ptr(), stream=_stream())
        self.down8.run(offsets=offsets, x=hc.data_ptr(), x_scales=hs.data_ptr(), w=self.d8[0].data_ptr(), w_scales=self.d8[1].data_ptr(), y=self.y.data_ptr(), **self._scratch())
        return self._bring_back(self.s, self.y, share)


def example(tokens, model, features, experts, top, device="cuda:0", dtype=torch.bfloat16):
    """a block, inputs for it, and a router's choice"""
    gen = torch.Generator(device=device)
    gen.manual_seed(tokens + experts)
    block = ExpertBlock(tokens, model, features, experts, top, dtype, device=device)
    block.params["norm_weight"].add_(torch.randn(model, device=device, generator=gen) * 0.2)
    x, residual, dout = ((torch.randn(tokens, model, device=device, generator=gen) * std).to(dtype) for std in (0.5, 1.0, 1.0))
    share, chosen = torch.randn(tokens, experts, device=device, generator=gen).softmax(1).topk(top, 1)
    return block, x, residual, chosen, share, dout


if __name__ == "__main__":
    block, x, residual, chosen, share, dout = example(4096, 1024, 2816, 8, 2)
    out = block.forward(x, residual, chosen, share)
    block.backward(dout)
    block.pack()
    out8 = block.forward8(x, residual, chosen, share)
    print("rows of the experts: %s" % block.offsets.diff().tolist())
    print("8 bits off 16 bits: %.4f of what the experts add" % ((out8.float() - out.float()).norm() / (out.float() - block.s.float()).norm()).item())
