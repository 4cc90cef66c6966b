"""The feed-forward half of a transformer block beyond its plain matmuls, as cases that can be timed: a gated feed-forward layer
(forward, backward, and a training step of both), layer norm (forward, backward, both), and activation checkpoints in 8 bits, alone
and between the forward and the backward pass of the other two.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes what a program holds before the call (device
tensors, and with `own` the configured call objects), `run()` makes one pass: in plain 32-bit torch operations, or with `own` through
zluda_amd.ffn.  `exact()` restates the operators in 64 bits.

Matrices are row-major; a token is a row.  Notation: X tokens x model, W = [Wg; Wu] 2 features x model, G = X Wg^T, U = X Wu^T,
H = act(G) * U.  A checkpoint holds e4m3 codes and, for each 32 neighbours of a row, a power of two.
"""
import math

import torch

own = False
DEV = "cuda:0"
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 32
EPS = 1e-5


def listed():
    return [
        # the smallest call: a few tokens through a little layer (a draft model), where the launch is what counts
        {"name": "gated_small", "kind": "gated", "type": "bf16", "act": "silu", "tokens": 5, "model": 256, "features": 688, "bias": False},
        # one new token of one sequence: the weights are read once
        {"name": "gated_t1", "kind": "gated", "type": "bf16", "act": "silu", "tokens": 1, "model": 4096, "features": 14336, "bias": False},
        # a decode step of 24 sequences, half precision, GELU gate, biases
        {"name": "gated_t24_f16", "kind": "gated", "type": "f16", "act": "gelu", "tokens": 24, "model": 5120, "features": 13824, "bias": True},
        # a prompt whose length no tile divides
        {"name": "gated_t777", "kind": "gated", "type": "bf16", "act": "silu", "tokens": 777, "model": 4096, "features": 14336, "bias": False},
        # the backward pass of a little layer over an odd number of tokens, with bias gradients
        {"name": "gated_bwd_t1001_f16", "kind": "gated_bwd", "type": "f16", "act": "gelu", "tokens": 1001, "model": 1024, "features": 2816, "bias": True},
        # the backward pass of a training step that kept its pre-activations in 16 bits
        {"name": "gated_bwd_t8192", "kind": "gated_bwd", "type": "bf16", "act": "silu", "tokens": 8192, "model": 2048, "features": 8192, "bias": False},
        # forward and backward with everything in between kept in 8 bits: the largest work
        {"name": "gated_step_8bit", "kind": "gated_step", "type": "bf16", "act": "silu", "tokens": 4096, "model": 4096, "features": 14336, "bias": False},
        # the norm of a decode step
        {"name": "norm_t8", "kind": "norm", "type": "bf16", "weights": "bf16", "rows": 8, "cols": 4096},
        # the norm of a long batch of prompts, the widest layers
        {"name": "norm_16384x8192", "kind": "norm", "type": "bf16", "weights": "bf16", "rows": 16384, "cols": 8192},
        # a norm's gradient over rows of an odd length
        {"name": "norm_bwd_777x1001_f16", "kind": "norm_bwd", "type": "f16", "weights": "f16", "rows": 777, "cols": 1001},
        # forward and backward of a norm inside a residual branch, its input kept in 8 bits, weights in single precision
        {"name": "norm_step_8bit", "kind": "norm_step", "type": "bf16", "weights": "f32", "rows": 16384, "cols": 4096},
        # a large activation put away in 8 bits and fetched again
        {"name": "checkpoint_8192x14336", "kind": "checkpoint", "type": "bf16", "rows": 8192, "cols": 14336},
    ]


def _log(rng, lo, hi, multiple=1):
    """a multiple of `multiple` from lo to hi, spread over the logarithm"""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / multiple)) * multiple))


def draw(rng):
    kind = rng.choice(["gated", "gated", "gated", "gated_bwd", "gated_step", "norm", "norm_bwd", "norm_step", "checkpoint"])
    if kind.startswith("gated"):
        model = _log(rng, 256, 5120, 8)
        features = min(14336, int(model * rng.uniform(2.0, 3.6)) // 8 * 8)
        if kind == "gated":
            tokens = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 64, 4096)
        else:
            tokens = _log(rng, 64, 8192)
        times = {"gated": 1, "gated_bwd": 2, "gated_step": 3}[kind]
        tokens = max(1, min(tokens, int(2.5e12 / (4.0 * times * model * features))))
        return {"kind": kind, "type": rng.choice(["bf16", "f16"]), "act": rng.choice(["silu", "gelu", "relu"]), "tokens": tokens, "model": model,
                "features": features, "bias": rng.random() < 0.4}
    typ = rng.choice(["bf16", "f16", "f32"])
    if kind == "checkpoint":
        cols = _log(rng, 64, 14336)
        return {"kind": kind, "type": typ, "rows": _log(rng, 1, min(16384, 8192 * 14336 // cols // 2)), "cols": cols}
    cols = _log(rng, 64, 16384, rng.choice([1, 8]))
    rows = _log(rng, 1, min(16384, 16384 * 4096 // cols))
    return {"kind": kind, "type": typ, "weights": rng.choice([typ, "f32"]), "rows": rows, "cols": cols}


# ---- inputs ---------------------------------------------------------------------------------------------------------------

def _randn(gen, std, *shape):
    return torch.randn(shape, device=DEV, generator=gen).mul_(std)


def _inputs(case, seed):
    """The tensors that a program holds before the call"""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed * 1000003 + 12345)
    typ = TORCH[case["type"]]
    s = {}
    if case["kind"].startswith("gated"):
        t, d, f = case["tokens"], case["model"], case["features"]
        x = _randn(gen, 1.0, t, d)
        x[:, :: max(1, d // 7)] *= 6.0              # the few wide channels that normalised activations have
        s["x"] = x.to(typ)
        s["w"] = _randn(gen, d ** -0.5, 2 * f, d).to(typ)
        s["bias"] = _randn(gen, 0.1, 2 * f).to(typ) if case["bias"] else None
        if case["kind"] != "gated":
            s["dh"] = _randn(gen, 0.05, t, f).to(typ)
        if case["kind"] == "gated_bwd":             # (what the forward pass kept)
            s["gate"] = _randn(gen, 1.3, t, f).to(typ)
            s["up"] = _randn(gen, 1.3, t, f).to(typ)
        return s
    rows, cols = case["rows"], case["cols"]
    x = _randn(gen, 1.0, rows, cols)
    x *= 0.5 + 3.0 * torch.rand((rows, 1), device=DEV, generator=gen)
    x[:, :: max(1, cols // 5)] *= 8.0
    x += 0.3
    s["x"] = x.to(typ)
    if case["kind"] == "checkpoint":
        return s
    wt = TORCH[case["weights"]]
    s["weight"] = (1.0 + _randn(gen, 0.2, cols)).to(wt)
    s["bias"] = _randn(gen, 0.1, cols).to(wt)
    if case["kind"] != "norm":
        s["dy"] = _randn(gen, 0.05, rows, cols).to(typ)
    if case["kind"] == "norm_bwd":                  # (what the forward pass kept)
        xf = s["x"].float()
        s["mean"] = xf.mean(1)
        s["rstd"] = (xf.var(1, unbiased=False) + EPS).rsqrt()
    if case["kind"] == "norm_step":                 # (the gradient that reaches the norm's input past the branch)
        s["add"] = _randn(gen, 0.05, rows, cols).to(typ)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    s["call"] = _calls(case, s) if own else None    # configured calls, output buffers and workspace
    return s


# ---- the framework's operators ----------------------------------------------------------------------------------------------

def _calls(case, s):
    from zluda_amd import abi, ffn
    types = {"bf16": abi.CUDA_R_16BF, "f16": abi.CUDA_R_16F, "f32": abi.CUDA_R_32F}
    typ, kind = TORCH[case["type"]], case["kind"]
    empty = lambda shape, t=typ: torch.empty(shape, dtype=t, device=DEV)  # noqa: E731
    c = {}
    need = 0
    if kind.startswith("gated"):
        t, d, f = case["tokens"], case["model"], case["features"]
        spec = dict(type=types[case["type"]], activation={"silu": ffn.SILU, "gelu": ffn.GELU, "relu": ffn.RELU}[case["act"]], tokens=t, model=d,
                    features=f, bias=case["bias"])
        if kind != "gated_bwd":
            c["h"] = empty((t, f))
            c["forward"] = ffn.GatedForward(dict(spec, kept=ffn.KEPT_8BIT if kind == "gated_step" else ffn.KEPT_NONE))
            need = max(need, c["forward"].workspace)
        if kind != "gated":
            c["dx"], c["dw"], c["dbias"] = empty((t, d)), empty((2 * f, d)), empty((2 * f,)) if case["bias"] else None
            eight = kind == "gated_step"
            c["backward"] = ffn.GatedBackward(dict(spec, kept=ffn.KEPT_8BIT if eight else ffn.KEPT_PLAIN, x_kept=ffn.KEPT_8BIT if eight else ffn.KEPT_PLAIN))
            need = max(need, c["backward"].workspace)
            if eight:
                c["gate"], c["up"], c["x"] = (ffn.checkpoint_buffers(t, n, DEV) for n in (f, f, d))
                c["store"] = ffn.Checkpoint(dict(type=types[case["type"]], rows=t, cols=d))
    elif kind == "checkpoint":
        rows, cols = case["rows"], case["cols"]
        c["checkpoint"] = ffn.Checkpoint(dict(type=types[case["type"]], rows=rows, cols=cols))
        c["x"], c["back"] = ffn.checkpoint_buffers(rows, cols, DEV), empty((rows, cols))
    else:
        rows, cols = case["rows"], case["cols"]
        spec = dict(type=types[case["type"]], weight_type=types[case["weights"]], rows=rows, cols=cols, eps=EPS)
        if kind != "norm_bwd":
            c["y"], c["mean"], c["rstd"] = empty((rows, cols)), empty((rows,), torch.float32), empty((rows,), torch.float32)
            c["forward"] = ffn.NormForward(dict(spec, kept=ffn.KEPT_8BIT if kind == "norm_step" else ffn.KEPT_NONE))
        if kind != "norm":
            wt = TORCH[case["weights"]]
            c["dx"], c["dweight"], c["dbias"] = empty((rows, cols)), empty((cols,), wt), empty((cols,), wt)
            c["backward"] = ffn.NormBackward(dict(spec, x_kept=ffn.KEPT_8BIT if kind == "norm_step" else ffn.KEPT_PLAIN, add=kind == "norm_step"))
            need = c["backward"].workspace
        if kind == "norm_step":
            c["x"] = ffn.checkpoint_buffers(rows, cols, DEV)
    c["workspace"] = torch.empty(need, dtype=torch.uint8, device=DEV) if need else None
    return c


def _run_own(s):
    case, c, kind = s["case"], s["call"], s["case"]["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    ws = dict(workspace=ptr(c["workspace"]), workspace_size=0 if c["workspace"] is None else c["workspace"].numel(), stream=stream)
    if kind == "gated":
        c["forward"].run(x=s["x"].data_ptr(), w=s["w"].data_ptr(), bias=ptr(s["bias"]), h=c["h"].data_ptr(), **ws)
        return c["h"]
    if kind == "gated_bwd":
        c["backward"].run(dh=s["dh"].data_ptr(), gate=s["gate"].data_ptr(), up=s["up"].data_ptr(), x=s["x"].data_ptr(), w=s["w"].data_ptr(),
                          dx=c["dx"].data_ptr(), dw=c["dw"].data_ptr(), dbias=ptr(c["dbias"]), **ws)
        return {"dx": c["dx"], "dw": c["dw"], "dbias": c["dbias"]}
    if kind == "gated_step":
        (g, gs), (u, us), (x, xs) = (tuple(t.data_ptr() for t in c[n]) for n in ("gate", "up", "x"))
        c["store"].store(x=s["x"].data_ptr(), codes=x, scales=xs, stream=stream)
        c["forward"].run(x=s["x"].data_ptr(), w=s["w"].data_ptr(), bias=ptr(s["bias"]), h=c["h"].data_ptr(), gate=g, gate_scales=gs, up=u,
                         up_scales=us, **ws)
        c["backward"].run(dh=s["dh"].data_ptr(), gate=g, gate_scales=gs, up=u, up_scales=us, x=x, x_scales=xs, w=s["w"].data_ptr(),
                          dx=c["dx"].data_ptr(), dw=c["dw"].data_ptr(), dbias=ptr(c["dbias"]), **ws)
        return {"h": c["h"], "dx": c["dx"], "dw": c["dw"], "dbias": c["dbias"]}
    if kind == "checkpoint":
        codes, scales = c["x"]
        c["checkpoint"].store(x=s["x"].data_ptr(), codes=codes.data_ptr(), scales=scales.data_ptr(), stream=stream)
        c["checkpoint"].load(codes=codes.data_ptr(), scales=scales.data_ptr(), x=c["back"].data_ptr(), stream=stream)
        return c["back"]
    out, x, xs = {}, s["x"].data_ptr(), None
    stats = (c if "mean" in c else s)
    if kind != "norm_bwd":
        kept = {} if kind == "norm" else dict(kept=c["x"][0].data_ptr(), kept_scales=c["x"][1].data_ptr())
        c["forward"].run(x=x, weight=s["weight"].data_ptr(), bias=s["bias"].data_ptr(), y=c["y"].data_ptr(), mean=c["mean"].data_ptr(),
                         rstd=c["rstd"].data_ptr(), stream=stream, **kept)
        out.update(y=c["y"], mean=c["mean"], rstd=c["rstd"])
    if kind != "norm":
        if kind == "norm_step":
            x, xs = c["x"][0].data_ptr(), c["x"][1].data_ptr()
        c["backward"].run(x=x, x_scales=xs, dy=s["dy"].data_ptr(), weight=s["weight"].data_ptr(), mean=stats["mean"].data_ptr(),
                          rstd=stats["rstd"].data_ptr(), add=ptr(s.get("add")), dx=c["dx"].data_ptr(), dweight=c["dweight"].data_ptr(),
                          dbias=c["dbias"].data_ptr(), **ws)
        out.update(dx=c["dx"], dweight=c["dweight"], dbias=c["dbias"])
    return out


# ---- plain forms ------------------------------------------------------------------------------------------------------------

_GELU = math.sqrt(2.0 / math.pi)


def _act(act, g):
    """act(g) and its derivative"""
    if act == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if act == "silu":
        sg = 1.0 / (1.0 + torch.exp(-g))
        return g * sg, sg * (1.0 + g * (1.0 - sg))
    th = torch.tanh(_GELU * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * g * (1.0 - th * th) * _GELU * (1.0 + 3 * 0.044715 * g * g)


def _checkpoint(x):
    """the values that a checkpoint of x stands for, in 32 bits"""
    rows, cols = x.shape
    pad = -cols % BLOCK
    v = torch.cat([x, x.new_zeros(rows, pad)], 1) if pad else x
    v = v.reshape(rows, -1, BLOCK)
    a = v.abs()
    top = torch.where(torch.isfinite(a), a, 0.0).amax(2, keepdim=True)
    e = ((top.view(torch.int32) + 0x1FFFFF) >> 23) - 135      # the smallest e with top <= 448 * 2^e
    scale = ((e.clamp_(min=-126) + 127) << 23).view(torch.float32)
    return ((v / scale).to(torch.float8_e4m3fn).float() * scale).reshape(rows, -1)[:, :cols]


def _gated_forward(s):
    f = s["case"]["features"]
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    g, u = z[:, :f], z[:, f:]
    return _act(s["case"]["act"], g)[0] * u, g, u


def _gated_backward(s, g, u, x):
    a, da = _act(s["case"]["act"], g)
    dh = s["dh"].float()
    dz = torch.cat([dh * u * da, dh * a], 1)
    typ = s["x"].dtype
    return {"dx": (dz @ s["w"].float()).to(typ), "dw": (dz.t() @ x).to(typ), "dbias": None if s["bias"] is None else dz.sum(0).to(typ)}


def _norm_backward(s, x, mean, rstd):
    dy = s["dy"].float()
    xh = (x - mean[:, None]) * rstd[:, None]
    dyw = dy * s["weight"].float()
    dx = rstd[:, None] * (dyw - dyw.mean(1, keepdim=True) - xh * (dyw * xh).mean(1, keepdim=True))
    if "add" in s:
        dx = dx + s["add"].float()
    wt = s["weight"].dtype
    return {"dx": dx.to(s["x"].dtype), "dweight": (dy * xh).sum(0).to(wt), "dbias": dy.sum(0).to(wt)}


def _run_plain(s):
    kind, typ = s["case"]["kind"], s["x"].dtype
    if kind == "gated":
        return _gated_forward(s)[0].to(typ)
    if kind == "gated_bwd":
        return _gated_backward(s, s["gate"].float(), s["up"].float(), s["x"].float())
    if kind == "gated_step":
        h, g, u = _gated_forward(s)
        return {"h": h.to(typ), **_gated_backward(s, _checkpoint(g), _checkpoint(u), _checkpoint(s["x"].float()))}
    if kind == "checkpoint":
        return _checkpoint(s["x"].float()).to(typ)
    out = {}
    x = s["x"].float()
    mean, rstd = s.get("mean"), s.get("rstd")
    if kind != "norm_bwd":
        mean = x.mean(1)
        rstd = 1.0 / torch.sqrt((x - mean[:, None]).square().mean(1) + EPS)
        y = (x - mean[:, None]) * rstd[:, None] * s["weight"].float() + s["bias"].float()
        out.update(y=y.to(typ), mean=mean, rstd=rstd)
    if kind != "norm":
        out.update(_norm_backward(s, _checkpoint(x) if kind == "norm_step" else x, mean, rstd))
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def _pow2(e):
    """2^e in 64 bits, exactly"""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_checkpoint(x):
    """each value to the nearest of its block's e4m3 grid (3 bits behind the leading one, steps of 2^-9 at least), ties to even"""
    rows, cols = x.shape
    out = torch.empty_like(x)
    for c0 in range(0, cols, BLOCK * 64):
        v = x[:, c0:c0 + BLOCK * 64]
        n = v.shape[1]
        v = torch.nn.functional.pad(v, (0, -n % BLOCK)).reshape(rows, -1, BLOCK)
        m, e = torch.frexp(v.abs().amax(2, keepdim=True))      # top = m 2^e, m in [0.5, 1)
        e = torch.where(m > 0.875, e - 8, e - 9)
        e = torch.where(m > 0, e, torch.full_like(e, -126)).clamp(min=-126)
        q = v * _pow2(-e)
        step = (torch.frexp(q)[1] - 4).clamp(min=-9)
        q = torch.round(q * _pow2(-step)) * _pow2(step)
        out[:, c0:c0 + n] = (q * _pow2(e)).reshape(rows, -1)[:, :n]
    return out


def _exact_act(act, g):
    if act == "relu":
        return g.clamp(min=0), torch.where(g > 0, 1.0, 0.0).to(g.dtype)
    z = g if act == "silu" else 2 * (2 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)      # both are g * sigmoid(z)
    dz = 1.0 if act == "silu" else 2 * (2 / math.pi) ** 0.5 * (1 + 0.134145 * g ** 2)
    sig = torch.sigmoid(z)
    return g * sig, sig + g * sig * torch.sigmoid(-z) * dz


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    d = {k: v.double() for k, v in s.items() if v is not None}
    if kind == "checkpoint":
        return _exact_checkpoint(d["x"])
    if kind.startswith("gated"):
        f, x = case["features"], d["x"]
        out = {}
        if kind == "gated_bwd":
            g, u = d["gate"], d["up"]
        else:
            g, u = x @ d["w"][:f].t(), x @ d["w"][f:].t()
            if case["bias"]:
                g, u = g + d["bias"][:f], u + d["bias"][f:]
            out["h"] = _exact_act(case["act"], g)[0] * u
            if kind == "gated":
                return out["h"]
            g, u, x = _exact_checkpoint(g), _exact_checkpoint(u), _exact_checkpoint(x)
        a, da = _exact_act(case["act"], g)
        dg, du = d["dh"] * u * da, d["dh"] * a
        out["dx"] = dg @ d["w"][:f] + du @ d["w"][f:]
        out["dw"] = torch.cat([dg.t() @ x, du.t() @ x])
        out["dbias"] = torch.cat([dg.sum(0), du.sum(0)]) if case["bias"] else None
        return out
    x, n, out = d["x"], case["cols"], {}
    if kind == "norm_bwd":
        mean, rstd = d["mean"], d["rstd"]
    else:
        mean = x.sum(1) / n
        rstd = ((x - mean.unsqueeze(1)).pow(2).sum(1) / n + EPS).pow(-0.5)
        out = {"y": torch.addcmul(d["bias"], (x - mean.unsqueeze(1)) * rstd.unsqueeze(1), d["weight"]), "mean": mean, "rstd": rstd}
    if kind == "norm":
        return out
    if kind == "norm_step":
        x = _exact_checkpoint(x)
    xh = (x - mean.unsqueeze(1)) * rstd.unsqueeze(1)
    v = d["dy"] * d["weight"]
    dx = (v - (v.sum(1, keepdim=True) + xh * (v * xh).sum(1, keepdim=True)) / n) * rstd.unsqueeze(1)
    out["dx"] = dx + d["add"] if kind == "norm_step" else dx
    out["dweight"], out["dbias"] = (d["dy"] * xh).sum(0), d["dy"].sum(0)
    return out


# ---- work -------------------------------------------------------------------------------------------------------------------

def work(case):
    kind, e = case["kind"], {"bf16": 2, "f16": 2, "f32": 4}[case["type"]]
    if kind.startswith("gated"):
        t, d, f = case["tokens"], case["model"], case["features"]
        fwd = e * (t * d + 2 * f * d + t * f + (2 * f if case["bias"] else 0))
        bwd = e * (t * f + 2 * (t * d + 2 * f * d) + (2 * f if case["bias"] else 0))
        kept = {"gated": 0, "gated_bwd": 2 * t * f * e, "gated_step": 2 * (1 + 1 / BLOCK) * t * (2 * f + d)}[kind]   # (a step writes and reads it)
        return {"bytes": {"gated": fwd, "gated_bwd": bwd, "gated_step": fwd + bwd - e * t * d}[kind] + kept,
                "flops": 4.0 * t * d * f * {"gated": 1, "gated_bwd": 2, "gated_step": 3}[kind]}
    n = case["rows"] * case["cols"]
    packed = n * (1 + 1 / BLOCK)
    if kind == "checkpoint":
        return {"bytes": 2 * n * e + 2 * packed, "flops": 2.0 * n}
    w = case["cols"] * {"bf16": 2, "f16": 2, "f32": 4}[case["weights"]]
    fwd, bwd = 2 * n * e + 2 * w + 8 * case["rows"], 3 * n * e + 3 * w + 8 * case["rows"]
    if kind == "norm_step":    # (the checkpoint in the place of x, and the gradient that is added)
        return {"bytes": fwd + packed + bwd + packed, "flops": 20.0 * n}
    return {"bytes": fwd if kind == "norm" else bwd, "flops": {"norm": 8.0, "norm_bwd": 12.0}[kind] * n}
