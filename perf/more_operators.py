"""Products of 8-bit operands with a float scale for each 128 of K, what makes such operands, and products grouped by expert, as cases that can be timed:

  scaled    cublasLtMatmul of 8-bit floats whose scales stand for 128 of K (of a row, or of 128 rows), with the epilogues
  grouped   rows sorted by expert times their expert's matrix: forward (16-bit, or 8-bit with scales), backward
  rms       root-mean-square norm with the residual's addition: plain or packed output, forward, forward and backward
  activate  a gated activation packed into 8 bits

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes what a program holds before the call (device tensors, and with
`own` the configured call objects), `run()` makes one pass: in plain 32-bit torch operations, or with `own` through zluda_amd.cublaslt and
zluda_amd.ffn.  `exact()` restates the operators in 64 bits.

Matrices are row-major; a token is a row.  Packed: e4m3 codes and, for each 128 neighbours of a row (or for each 128 x 128 of a weight), a float
scale, the largest magnitude over 448; what is packed is returned as the values it stands for.
"""
import math
import random

import torch

own = False
DEV = "cuda:0"
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
BLOCK = 128
EPS = 1e-5


def listed():
    return [
        # one new token of one sequence through a down projection: the weights are read once
        {"name": "scaled_t1", "kind": "scaled", "tokens": 1, "features": 4096, "model": 14336, "out": "bf16", "weights": "e4m3", "x": "e4m3",
         "w_block": 128, "act": "none", "bias": False},
        # a prompt of an odd length, a last block of K that is not whole, a scale for each row of the weights, bias and GELU
        {"name": "scaled_t333_f16", "kind": "scaled", "tokens": 333, "features": 5632, "model": 2000, "out": "f16", "weights": "e4m3", "x": "e4m3",
         "w_block": 1, "act": "gelu", "bias": True},
        # the largest product: a long batch of prompts
        {"name": "scaled_8192", "kind": "scaled", "tokens": 8192, "features": 8192, "model": 8192, "out": "bf16", "weights": "e4m3", "x": "e4m3",
         "w_block": 128, "act": "none", "bias": False},
        # a decode step of eight sequences, each token with eight of 64 experts: a row or two of an expert, a third of them without any
        {"name": "grouped_t64", "kind": "grouped", "type": "bf16", "rows": 64, "spare": 0, "experts": 64, "empty": 22, "model": 2048, "features": 2816},
        # a prompt over eight experts, an odd number of rows, some behind the last expert's
        {"name": "grouped_t1001_f16", "kind": "grouped", "type": "f16", "rows": 1001, "spare": 37, "experts": 8, "empty": 1, "model": 1024, "features": 2816},
        # a long batch of prompts over 16 experts in 8 bits
        {"name": "grouped_8bit_t16384", "kind": "grouped8", "type": "bf16", "rows": 16384, "spare": 0, "experts": 16, "empty": 0, "model": 4096, "features": 4096},
        # the gradients of a training step's expert layer
        {"name": "grouped_bwd_t8192", "kind": "grouped_bwd", "type": "bf16", "rows": 8192, "spare": 0, "experts": 8, "empty": 0, "model": 4096, "features": 2816},
        # the norm of a decode step of four sequences: the launch is what counts
        {"name": "rms_t4", "kind": "rms", "type": "bf16", "weights": "bf16", "rows": 4, "cols": 4096},
        # a norm whose output is the operand of an 8-bit product
        {"name": "rms_8bit_16384x8192", "kind": "rms8", "type": "bf16", "weights": "bf16", "rows": 16384, "cols": 8192},
        # forward and backward over rows of an odd length
        {"name": "rms_step_777x1001_f16", "kind": "rms_step", "type": "f16", "weights": "f32", "rows": 777, "cols": 1001},
        # the activation between two 8-bit products: a decode step of 24 sequences
        {"name": "activate_t24_f16", "kind": "activate", "type": "f16", "act": "gelu", "rows": 24, "cols": 13824},
        # and a long batch of prompts
        {"name": "activate_8192x14336", "kind": "activate", "type": "bf16", "act": "silu", "rows": 8192, "cols": 14336},
    ]


def _log(rng, lo, hi, multiple=1):
    """a multiple of `multiple` from lo to hi, spread over the logarithm"""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / multiple)) * multiple))


def draw(rng):
    kind = rng.choice(["scaled", "scaled", "scaled", "grouped", "grouped", "grouped8", "grouped_bwd", "rms", "rms8", "rms_step", "activate"])
    if kind == "scaled":
        model, features = _log(rng, 256, 14336, 16), _log(rng, 256, 14336, 8)
        tokens = _log(rng, 1, 64) if rng.random() < 0.4 else _log(rng, 64, 8192)
        tokens = max(1, min(tokens, int(1.0e12 / (2.0 * model * features))))
        return {"kind": kind, "tokens": tokens, "features": features, "model": model, "out": rng.choice(["bf16", "f16", "f32"]), "weights": "e4m3",
                "x": rng.choice(["e4m3", "e4m3", "e5m2"]), "w_block": rng.choice([128, 128, 1]), "act": rng.choice(["none", "none", "relu", "gelu"]),
                "bias": rng.random() < 0.4}
    if kind.startswith("grouped"):
        experts = rng.choice([2, 3, 8, 16, 40, 64])
        model = _log(rng, 256, 4096, 16 if kind == "grouped8" else 8)
        features = min(_log(rng, 256, 5632, 8), int(4.0e8 / (experts * model)) // 8 * 8)
        rows = _log(rng, 1, 64) if kind != "grouped_bwd" and rng.random() < 0.4 else _log(rng, 64, 16384)
        rows = max(1, min(rows, int(5.0e11 / (2.0 * (2 if kind == "grouped_bwd" else 1) * model * features))))
        spare = min(rows // 4, rng.choice([0, 0, 5, 64]))
        empty = max(experts - (rows - spare), rng.choice([0, 0, 1, experts // 3]))
        return {"kind": kind, "type": rng.choice(["bf16", "f16"]), "rows": rows, "spare": spare, "experts": experts, "empty": empty, "model": model, "features": features}
    typ = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "activate":
        cols = _log(rng, 64, 14336)
        return {"kind": kind, "type": rng.choice(["bf16", "f16"]), "act": rng.choice(["silu", "gelu", "relu"]), "rows": _log(rng, 1, min(16384, 8192 * 14336 // cols)),
                "cols": cols}
    cols = _log(rng, 64, 16384, rng.choice([1, 8]))
    if kind == "rms8":
        typ = "bf16" if typ == "f32" else typ
    return {"kind": kind, "type": typ, "weights": rng.choice([typ, "f32"]), "rows": _log(rng, 1, min(16384, 16384 * 4096 // cols)), "cols": cols}


# ---- inputs ---------------------------------------------------------------------------------------------------------------

def _randn(gen, std, *shape):
    return torch.randn(shape, device=DEV, generator=gen).mul_(std)


def _blocks(n):
    return -(-n // BLOCK)


def _quantised(v, typ, block_rows):
    """codes of v (rows x cols, 32 bits) and the scales of blocks of block_rows x 128: [row block][block]"""
    top = {"e4m3": 448.0, "e5m2": 57344.0}[typ]
    rows, cols = v.shape
    rb, cb = -(-rows // block_rows), _blocks(cols)
    scales = torch.empty((rb, cb), device=DEV)
    codes = torch.empty((rows, cols), dtype=TORCH[typ], device=DEV)
    for c0 in range(0, cols, BLOCK * 16):          # (in strips, for the memory that the 32-bit steps take)
        strip = v[:, c0:c0 + BLOCK * 16]
        n = strip.shape[1]
        p = torch.nn.functional.pad(strip, (0, -n % BLOCK, 0, rb * block_rows - rows)).reshape(rb, block_rows, -1, BLOCK)
        s = (p.abs().amax((1, 3)) / top).clamp_(min=2.0 ** -126)
        scales[:, c0 // BLOCK:c0 // BLOCK + s.shape[1]] = s
        codes[:, c0:c0 + n] = (p / s[:, None, :, None]).reshape(rb * block_rows, -1)[:rows, :n].to(TORCH[typ])
    return codes, scales


def _counts(case, seed):
    """rows of each expert: some have none, the others an uneven share"""
    rng = random.Random(seed * 7919 + case["rows"] * 31 + case["experts"])
    live = sorted(rng.sample(range(case["experts"]), case["experts"] - case["empty"]))
    left = case["rows"] - case["spare"] - len(live)
    weight = [0.6 + 0.8 * rng.random() for _ in live]
    counts = [0] * case["experts"]
    share = [int(left * w / sum(weight)) for w in weight]
    for i in range(left - sum(share)):
        share[i % len(share)] += 1
    for e, n in zip(live, share):
        counts[e] = 1 + n
    return counts


def _activations(gen, rows, cols):
    x = _randn(gen, 1.0, rows, cols)
    x[:, :: max(1, cols // 7)] *= 6.0              # the few wide channels that activations have
    return x


def _inputs(case, seed):
    """The tensors that a program holds before the call"""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed * 1000003 + 54321)
    kind = case["kind"]
    s = {}
    if kind == "scaled":
        t, f, d = case["tokens"], case["features"], case["model"]
        s["x"], s["x_scales"] = _quantised(_activations(gen, t, d), case["x"], 1)
        s["w"], s["w_scales"] = _quantised(_randn(gen, d ** -0.5, f, d), case["weights"], case["w_block"])
        s["x_scales"] = s["x_scales"].t().contiguous()                               # [block][token]
        if case["w_block"] == 1:
            s["w_scales"] = s["w_scales"].t().contiguous()
        else:                                                                        # rows of a multiple of four
            s["w_scales"] = torch.nn.functional.pad(s["w_scales"], (0, -s["w_scales"].shape[1] % 4)).contiguous()
        s["bias"] = _randn(gen, 0.1, f).to(TORCH[case["out"]]) if case["bias"] else None
        return s
    typ = TORCH[case["type"]]
    if kind.startswith("grouped"):
        r, e, f, d = case["rows"], case["experts"], case["features"], case["model"]
        counts = _counts(case, seed)
        offsets = [0]
        for n in counts:
            offsets.append(offsets[-1] + n)
        s["offsets"] = torch.tensor(offsets, dtype=torch.int32, device=DEV)
        s["most"] = max(counts)                                                       # (what a plain program pads to)
        if kind == "grouped8":
            s["x"], xs = _quantised(_activations(gen, r, d), "e4m3", 1)
            s["x_scales"] = xs.t().contiguous()
            s["w"] = torch.empty((e, f, d), dtype=TORCH["e4m3"], device=DEV)
            s["w_scales"] = torch.zeros((e, _blocks(f), -(-_blocks(d) // 4) * 4), device=DEV)
            for i in range(e):
                s["w"][i], s["w_scales"][i, :, :_blocks(d)] = _quantised(_randn(gen, d ** -0.5, f, d), "e4m3", BLOCK)
            return s
        s["w"] = torch.empty((e, f, d), dtype=typ, device=DEV)
        for i in range(e):
            s["w"][i] = _randn(gen, d ** -0.5, f, d)
        s["x"] = _activations(gen, r, d).to(typ)
        if kind == "grouped_bwd":
            s["dy"] = _randn(gen, 0.05, r, f).to(typ)
        return s
    rows, cols = case["rows"], case["cols"]
    if kind == "activate":
        s["z"] = _randn(gen, 1.3, rows, 2 * cols).to(typ)                             # [G U], as the product in front leaves them
        return s
    s["x"] = _randn(gen, 0.4, rows, cols).to(typ)                                     # what the branch adds
    res = _activations(gen, rows, cols) * (0.5 + 3.0 * torch.rand((rows, 1), device=DEV, generator=gen))
    s["residual"] = res.to(typ)
    s["weight"] = (1.0 + _randn(gen, 0.2, cols)).to(TORCH[case["weights"]])
    if kind == "rms_step":
        s["dy"] = _randn(gen, 0.05, rows, cols).to(typ)
        s["add"] = _randn(gen, 0.05, rows, cols).to(typ)                              # the gradient that reaches the sum past the norm
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    s["call"] = _calls(case, s) if own else None    # configured calls, output buffers and workspace
    return s


# ---- the framework's operators ----------------------------------------------------------------------------------------------

def _calls(case, s):
    import ctypes
    from zluda_amd import abi, cublaslt, ffn
    types = {"bf16": abi.CUDA_R_16BF, "f16": abi.CUDA_R_16F, "f32": abi.CUDA_R_32F, "e4m3": abi.CUDA_R_8F_E4M3, "e5m2": abi.CUDA_R_8F_E5M2}
    acts = {"silu": ffn.SILU, "gelu": ffn.GELU, "relu": ffn.RELU}
    kind, c, need = case["kind"], {}, 0
    empty = lambda shape, t: torch.empty(shape, dtype=t, device=DEV)  # noqa: E731
    if kind == "scaled":
        t, f, d = case["tokens"], case["features"], case["model"]
        epilogue = {("none", False): abi.CUBLASLT_EPILOGUE_DEFAULT, ("none", True): abi.CUBLASLT_EPILOGUE_BIAS, ("relu", False): abi.CUBLASLT_EPILOGUE_RELU,
                    ("relu", True): abi.CUBLASLT_EPILOGUE_RELU_BIAS, ("gelu", False): abi.CUBLASLT_EPILOGUE_GELU,
                    ("gelu", True): abi.CUBLASLT_EPILOGUE_GELU_BIAS}[case["act"], case["bias"]]
        vec, blk = abi.CUBLASLT_MATMUL_MATRIX_SCALE_VEC128_32F, abi.CUBLASLT_MATMUL_MATRIX_SCALE_BLK128x128_32F
        c["call"] = cublaslt.MatmulCall(cublaslt.load(), dict(
            m=f, n=t, k=d, a_type=types[case["weights"]], b_type=types[case["x"]], d_type=types[case["out"]], compute_type=abi.CUBLAS_COMPUTE_32F,
            scale_type=abi.CUDA_R_32F, transa=abi.CUBLAS_OP_T, a_scale_mode=blk if case["w_block"] == 128 else vec, b_scale_mode=vec, epilogue=epilogue),
            max_workspace=32 << 20)
        c["call"].set_pointers(bias=s["bias"].data_ptr() if case["bias"] else None, a_scale=s["w_scales"].data_ptr(), b_scale=s["x_scales"].data_ptr())
        c["one"], c["zero"] = ctypes.c_float(1.0), ctypes.c_float(0.0)
        c["y"], need = empty((t, f), TORCH[case["out"]]), 32 << 20
    elif kind.startswith("grouped"):
        typ = TORCH[case["type"]]
        spec = dict(type=types[case["type"]], **{k: case[k] for k in ("rows", "experts", "model", "features")})
        if kind == "grouped_bwd":
            c["backward"] = ffn.GroupedBackward(spec)
            c["dx"], c["dw"] = torch.zeros_like(s["x"]), empty(s["w"].shape, typ)
            need = c["backward"].workspace
        else:
            c["forward"] = ffn.GroupedForward(dict(spec, packed=kind == "grouped8"))
            c["y"] = torch.zeros((case["rows"], case["features"]), dtype=typ, device=DEV)   # (the rows behind the last expert's stay as they are)
            need = c["forward"].workspace
    else:
        rows, cols, typ = case["rows"], case["cols"], TORCH[case["type"]]
        spec = dict(type=types[case["type"]], rows=rows, cols=cols)
        c["y"] = empty((rows, cols), typ)
        if kind in ("activate", "rms8"):
            c["packed"] = ffn.packed_buffers(rows, cols, DEV)
            c["unpack"] = ffn.Unpack(spec)
        if kind == "activate":
            c["activate"] = ffn.Activate(dict(spec, activation=acts[case["act"]], ldgate=2 * cols, ldup=2 * cols))
        else:
            c["sum"] = empty((rows, cols), typ)
            c["forward"] = ffn.RmsForward(dict(spec, weight_type=types[case["weights"]], eps=EPS))
        if kind == "rms_step":
            c["rstd"], c["dx"], c["dweight"] = empty((rows,), torch.float32), empty((rows, cols), typ), empty((cols,), TORCH[case["weights"]])
            c["backward"] = ffn.RmsBackward(dict(spec, weight_type=types[case["weights"]]))
            need = c["backward"].workspace
    c["workspace"] = torch.empty(need, dtype=torch.uint8, device=DEV) if need else None
    return c


def _run_own(s):
    case, c, kind = s["case"], s["call"], s["case"]["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    ws = dict(workspace=None if c["workspace"] is None else c["workspace"].data_ptr(), workspace_size=0 if c["workspace"] is None else c["workspace"].numel(),
              stream=stream)
    if kind == "scaled":
        y = c["y"].data_ptr()
        status = c["call"].run(c["one"], s["w"].data_ptr(), s["x"].data_ptr(), c["zero"], y, y, **ws)
        if status:
            raise RuntimeError("cublasLtMatmul: status %d" % status)
        return c["y"]
    if kind == "grouped_bwd":
        c["backward"].run(offsets=s["offsets"].data_ptr(), dy=s["dy"].data_ptr(), x=s["x"].data_ptr(), w=s["w"].data_ptr(), dx=c["dx"].data_ptr(),
                          dw=c["dw"].data_ptr(), **ws)
        return {"dx": c["dx"], "dw": c["dw"]}
    if kind.startswith("grouped"):
        scales = dict(x_scales=s["x_scales"].data_ptr(), w_scales=s["w_scales"].data_ptr()) if kind == "grouped8" else {}
        c["forward"].run(offsets=s["offsets"].data_ptr(), x=s["x"].data_ptr(), w=s["w"].data_ptr(), y=c["y"].data_ptr(), **scales, **ws)
        return c["y"]
    if kind == "activate":
        z, (codes, scales) = s["z"].data_ptr(), (t.data_ptr() for t in c["packed"])
        c["activate"].run(gate=z, up=z + case["cols"] * s["z"].element_size(), codes=codes, scales=scales, stream=stream)
        c["unpack"].run(codes=codes, scales=scales, y=c["y"].data_ptr(), stream=stream)
        return c["y"]
    args = dict(x=s["x"].data_ptr(), residual=s["residual"].data_ptr(), weight=s["weight"].data_ptr(), sum=c["sum"].data_ptr(), stream=stream)
    if kind == "rms8":
        codes, scales = (t.data_ptr() for t in c["packed"])
        c["forward"].run(codes=codes, scales=scales, **args)
        c["unpack"].run(codes=codes, scales=scales, y=c["y"].data_ptr(), stream=stream)
        return {"sum": c["sum"], "y": c["y"]}
    if kind == "rms":
        c["forward"].run(y=c["y"].data_ptr(), **args)
        return {"sum": c["sum"], "y": c["y"]}
    c["forward"].run(y=c["y"].data_ptr(), rstd=c["rstd"].data_ptr(), **args)
    c["backward"].run(h=c["sum"].data_ptr(), dy=s["dy"].data_ptr(), rstd=c["rstd"].data_ptr(), weight=s["weight"].data_ptr(), add=s["add"].data_ptr(),
                      dx=c["dx"].data_ptr(), dweight=c["dweight"].data_ptr(), **ws)
    return {"sum": c["sum"], "y": c["y"], "rstd": c["rstd"], "dx": c["dx"], "dweight": c["dweight"]}


# ---- plain forms ------------------------------------------------------------------------------------------------------------

_GELU = math.sqrt(2.0 / math.pi)


def _act(act, g):
    if act == "none":
        return g
    if act == "relu":
        return g.clamp(min=0)
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(_GELU * (g + 0.044715 * g * g * g)))


def _values(codes, scales, rows_each):
    """the 32-bit values of codes: rows x cols, scales [row block][block]"""
    rows, cols = codes.shape[-2:]
    s = scales.repeat_interleave(rows_each, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :cols]
    return codes.float() * s


def _packed(v):
    """the values that packing v (rows x cols) makes of it, in 32 bits"""
    rows, cols = v.shape
    p = torch.nn.functional.pad(v, (0, -cols % BLOCK)).reshape(rows, -1, BLOCK)
    scale = (p.abs().amax(2, keepdim=True) / 448.0).clamp(min=2.0 ** -126)
    return ((p / scale).to(torch.float8_e4m3fn).float() * scale).reshape(rows, -1)[:, :cols]


def _slots(s):
    """a place for each row in a batch of experts x most rows; rows behind the last expert's go past its end"""
    case, most = s["case"], s["most"]
    r = torch.arange(case["rows"], device=DEV)
    o = s["offsets"].long()
    e = (torch.searchsorted(o, r, right=True) - 1).clamp(max=case["experts"] - 1)
    return torch.where(r < o[-1], e * most + r - o[e], case["experts"] * most)


def _padded(s, slots, v):
    """rows sorted by expert in a batch of experts, in 32 bits"""
    e, most = s["case"]["experts"], s["most"]
    out = torch.zeros((e * most + 1, v.shape[1]), device=DEV)
    out[slots] = v.float()
    return out[:-1].reshape(e, most, -1)


def _rows_of(slots, v):
    """and back; zeros for the rows behind the last expert's"""
    v = v.reshape(-1, v.shape[-1])
    return torch.cat([v, v.new_zeros(1, v.shape[1])])[slots]


def _run_plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "scaled":
        w_scales = s["w_scales"].t() if case["w_block"] == 1 else s["w_scales"]
        y = _values(s["x"], s["x_scales"].t(), 1) @ _values(s["w"], w_scales, case["w_block"]).t()
        if case["bias"]:
            y = y + s["bias"].float()
        return _act(case["act"], y).to(TORCH[case["out"]])
    typ = TORCH[case["type"]]
    if kind == "grouped8":
        slots = _slots(s)
        x = _padded(s, slots, _values(s["x"], s["x_scales"].t(), 1))
        return _rows_of(slots, torch.bmm(x, _values(s["w"], s["w_scales"], BLOCK).transpose(1, 2))).to(typ)
    if kind == "grouped":
        slots = _slots(s)
        return _rows_of(slots, torch.bmm(_padded(s, slots, s["x"]), s["w"].float().transpose(1, 2))).to(typ)
    if kind == "grouped_bwd":
        slots = _slots(s)
        x, dy = _padded(s, slots, s["x"]), _padded(s, slots, s["dy"])
        return {"dx": _rows_of(slots, torch.bmm(dy, s["w"].float())).to(typ), "dw": torch.bmm(dy.transpose(1, 2), x).to(typ)}
    if kind == "activate":
        g, u = s["z"].float().chunk(2, 1)
        return _packed(_act(case["act"], g) * u).to(typ)
    h = (s["x"].float() + s["residual"].float()).to(typ)
    hf, w = h.float(), s["weight"].float()
    rstd = 1.0 / torch.sqrt(hf.square().mean(1) + EPS)
    y = hf * rstd[:, None] * w
    if kind == "rms8":
        return {"sum": h, "y": _packed(y).to(typ)}
    out = {"sum": h, "y": y.to(typ)}
    if kind == "rms_step":
        dy = s["dy"].float()
        xh, v = hf * rstd[:, None], dy * w
        dx = rstd[:, None] * (v - xh * (v * xh).mean(1, keepdim=True)) + s["add"].float()
        out.update(rstd=rstd, dx=dx.to(typ), dweight=(dy * xh).sum(0).to(TORCH[case["weights"]]))
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def _pow2(e):
    """2^e in 64 bits, exactly"""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_packed(x):
    """each value to the nearest of its block's e4m3 grid (3 bits behind the leading one, steps of 2^-9 at least), ties to even"""
    rows, cols = x.shape
    out = torch.empty_like(x)
    for c0 in range(0, cols, BLOCK * 16):
        v = x[:, c0:c0 + BLOCK * 16]
        n = v.shape[1]
        v = torch.nn.functional.pad(v, (0, -n % BLOCK)).reshape(rows, -1, BLOCK)
        scale = (v.abs().amax(2, keepdim=True) / 448).float().double()
        scale = torch.where(scale < 2.0 ** -126, torch.full_like(scale, 2.0 ** -126), scale)
        q = v / scale
        step = _pow2((torch.frexp(q)[1] - 4).clamp(min=-9))
        q = (torch.round(q / step) * step).clamp(-448, 448)
        out[:, c0:c0 + n] = (q * scale).reshape(rows, -1)[:, :n]
    return out


def _exact_act(act, g):
    if act == "none":
        return g
    if act == "relu":
        return torch.where(g > 0, g, torch.zeros_like(g))
    return g * torch.sigmoid(g if act == "silu" else 2 * (2 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3))


def _exact_blocks(x, w, xs, ws):
    """x w^T, one block of K after the other: xs [block][token], ws [block][feature]"""
    y = torch.zeros((x.shape[0], w.shape[0]), dtype=torch.float64, device=x.device)
    for b in range(xs.shape[0]):
        k = slice(b * BLOCK, (b + 1) * BLOCK)
        y.addmm_(x[:, k].double() * xs[b].double()[:, None], (w[:, k].double() * ws[b].double()[:, None]).t())
    return y


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "scaled":
        f = case["features"]
        ws = s["w_scales"] if case["w_block"] == 1 else s["w_scales"].t()[:_blocks(case["model"])].repeat_interleave(BLOCK, 1)[:, :f]
        y = _exact_blocks(s["x"], s["w"], s["x_scales"], ws)
        return _exact_act(case["act"], y + s["bias"].double() if case["bias"] else y)
    if kind.startswith("grouped"):
        o = s["offsets"].tolist()
        f, d = case["features"], case["model"]
        y = torch.zeros((case["rows"], d if kind == "grouped_bwd" else f), dtype=torch.float64, device=DEV)
        dw = torch.zeros(s["w"].shape, dtype=torch.float64, device=DEV) if kind == "grouped_bwd" else None
        for e in range(case["experts"]):
            r = slice(o[e], o[e + 1])
            if kind == "grouped8":
                ws = s["w_scales"][e].t()[:_blocks(d)].repeat_interleave(BLOCK, 1)[:, :f]
                y[r] = _exact_blocks(s["x"][r], s["w"][e], s["x_scales"][:, r], ws)
            elif kind == "grouped":
                y[r] = s["x"][r].double() @ s["w"][e].double().t()
            else:
                dy = s["dy"][r].double()
                y[r] = dy @ s["w"][e].double()
                dw[e] = dy.t() @ s["x"][r].double()
        return {"dx": y, "dw": dw} if kind == "grouped_bwd" else y
    d = {k: v.double() for k, v in s.items() if torch.is_tensor(v)}
    if kind == "activate":
        n = case["cols"]
        return _exact_packed(_exact_act(case["act"], d["z"][:, :n]) * d["z"][:, n:])
    h = (d["x"] + d["residual"]).to(TORCH[case["type"]]).double()
    n = case["cols"]
    rstd = (h.pow(2).sum(1) / n + EPS).pow(-0.5)
    xh = h * rstd.unsqueeze(1)
    y = xh * d["weight"]
    out = {"sum": h, "y": _exact_packed(y) if kind == "rms8" else y}
    if kind == "rms_step":
        v = d["dy"] * d["weight"]
        out["rstd"] = rstd
        out["dx"] = (v - xh * ((v * xh).sum(1, keepdim=True) / n)) * rstd.unsqueeze(1) + d["add"]
        out["dweight"] = (d["dy"] * xh).sum(0)
    return out


# ---- work -------------------------------------------------------------------------------------------------------------------

def work(case):
    kind, size = case["kind"], {"bf16": 2, "f16": 2, "f32": 4}
    if kind == "scaled":
        t, f, d, o = case["tokens"], case["features"], case["model"], size[case["out"]]
        scales = 4 * _blocks(d) * (t + (f if case["w_block"] == 1 else _blocks(f)))
        return {"bytes": t * d + f * d + scales + o * t * f + (o * f if case["bias"] else 0), "flops": 2.0 * t * f * d}
    if kind.startswith("grouped"):
        r, d, f, live = case["rows"] - case["spare"], case["model"], case["features"], case["experts"] - case["empty"]
        if kind == "grouped8":
            return {"bytes": r * d + live * f * d + 4 * _blocks(d) * (r + live * _blocks(f)) + 2 * r * f, "flops": 2.0 * r * d * f}
        if kind == "grouped":
            return {"bytes": 2 * (r * d + live * f * d + r * f), "flops": 2.0 * r * d * f}
        return {"bytes": 2 * (2 * r * d + r * f + live * f * d + case["experts"] * f * d), "flops": 4.0 * r * d * f}
    n, e = case["rows"] * case["cols"], size[case["type"]]
    packed = n * (1 + 4 / BLOCK)
    if kind == "activate":      # (packed, and fetched again)
        return {"bytes": 2 * n * e + 2 * packed + n * e, "flops": 12.0 * n}
    w = case["cols"] * size[case["weights"]]
    if kind == "rms":
        return {"bytes": 4 * n * e + w, "flops": 6.0 * n}
    if kind == "rms8":
        return {"bytes": 3 * n * e + w + 2 * packed + n * e, "flops": 8.0 * n}
    return {"bytes": 4 * n * e + w + 4 * n * e + 2 * w + 8 * case["rows"], "flops": 18.0 * n}
