"""The feed-forward operators of include/zluda_ffn.h restated in 64 bits, with error bounds for kernels that compute in 32.

Every oracle returns (value, bound on the error in front of the last rounding).  The bounds are worst cases of the arithmetic:
a product of two 16-bit numbers is exact in 32 bits, a sum of n terms in any order is off by at most n 2^-24 times the sum of the
terms' magnitudes, v_exp_f32 and v_rcp_f32 are good to one unit in the last place."""
import math

import torch

E32 = 2.0 ** -24
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}     # half a unit in the last place, relative
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half the smallest subnormal
K2 = 2 * math.sqrt(2 / math.pi)
ACTS = ["silu", "gelu", "relu"]


def act(name, g):
    """act(g), act'(g), |z| of the sigmoid's argument, the magnitude of the derivative's terms"""
    if name == "relu":
        on = (g > 0).double()
        return g.clamp(min=0), on, torch.zeros_like(g), on
    z = g if name == "silu" else K2 * (g + 0.044715 * g ** 3)
    dz = torch.ones_like(g) if name == "silu" else K2 * (1 + 3 * 0.044715 * g * g)
    s, ns = torch.sigmoid(z), torch.sigmoid(-z)
    return g * s, s + g * s * ns * dz, z.abs(), s + (g * s * dz).abs()      # (1 - s is rounded at the size of 1)


def checkpoint(x):
    """(the values that a checkpoint of x stands for, codes, scale bytes); what is not finite becomes NaN"""
    x = x.double().cpu()
    rows, cols = x.shape
    v = torch.nn.functional.pad(x, (0, -cols % 32)).reshape(rows, -1, 32)
    a = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v))
    m, e = torch.frexp(a.amax(2, keepdim=True))                 # m 2^e, m in [1/2, 1)
    e = (e - 9 + (m > 0.875)).where(m > 0, torch.full_like(e, -126)).clamp(min=-126).long()
    q = torch.where(torch.isfinite(v), torch.ldexp(v, -e), torch.zeros_like(v))
    step = (torch.frexp(q)[1] - 4).clamp(min=-9)                # e4m3: three bits behind the leading one, 2^-9 at least
    n = torch.round(torch.ldexp(q, -step))                      # ties to even
    val = torch.ldexp(n, step)
    mag = val.abs()
    ex = (torch.frexp(mag)[1] - 1).clamp(min=-6)
    code = torch.where(mag < 2.0 ** -6, torch.ldexp(mag, torch.full_like(ex, 9)), (ex + 7) * 8 + (torch.ldexp(mag, 3 - ex) - 8)).to(torch.int64)
    code = torch.where(torch.isfinite(v), code, torch.full_like(code, 0x7F)) | (torch.signbit(v).long() << 7)
    val = torch.where(torch.isfinite(v), torch.ldexp(val, e), torch.full_like(val, float("nan")))
    return val.reshape(rows, -1)[:, :cols], code.to(torch.uint8).reshape(rows, -1), (e + 127).to(torch.uint8).reshape(rows, -1)


def gated_forward(name, x, w, bias):
    """G, U, H and their bounds: {"g": (value, bound), ...}"""
    x, w = x.double(), w.double()
    f, k = w.shape[0] // 2, x.shape[1]
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    err = (k + 1) * E32 * mag
    if bias is not None:
        z, err = z + bias.double(), err + 2 * E32 * (mag + bias.double().abs())
    g, u, eg, eu = z[:, :f], z[:, f:], err[:, :f], err[:, f:]
    a, _, za, _ = act(name, g)
    ea = 1.13 * eg + (za + 8) * 2 * E32 * a.abs()               # |act'| is below 1.13
    return {"g": (g, eg), "u": (u, eu), "h": (a * u, ea * u.abs() + a.abs() * eu + ea * eu + 2 * E32 * (a * u).abs())}


def gated_backward(name, dh, g, u, x, w):
    """dz = [dG dU], H, dx, dw, dbias from exact dH, G, U, X, W; dz is rounded to dh's type for the products, not for dbias"""
    unit, tiny = UNIT[dh.dtype], TINY[dh.dtype]
    dh, g, u, x, w = (t.double() for t in (dh, g, u, x, w))
    a, da, za, ma = act(name, g)
    rel = (za + 16) * 4 * E32
    dz = torch.cat([dh * u * da, dh * a], 1)
    ez = torch.cat([(dh * u).abs() * ma * rel, (dh * a).abs() * rel], 1)
    er = ez + unit * (dz.abs() + ez) + tiny
    mag = dz.abs() + er
    t, f2 = dz.shape
    out = {"dz": (dz, ez), "h": (a * u, (a * u).abs() * rel)}
    out["dx"] = (dz @ w, er @ w.abs() + (f2 + 1) * E32 * (mag @ w.abs()))
    out["dw"] = (dz.t() @ x, er.t() @ x.abs() + (t + 1) * E32 * (mag.t() @ x.abs()))
    out["dbias"] = (dz.sum(0), ez.sum(0) + (t + 1) * E32 * (dz.abs() + ez).sum(0))
    return out


DEPTH = 40   # additions behind each other in a row's sum: 16 in a thread, 6 in a wave, at most 16 waves


def norm_forward(x, weight, bias, eps):
    x = x.double()
    n = x.shape[1]
    w = torch.ones(n, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros(n, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    em = (DEPTH + 2) * E32 * x.abs().mean(1, keepdim=True)
    var = d.square().mean(1, keepdim=True)
    ev = 2 * em * d.abs().mean(1, keepdim=True) + em * em + (DEPTH + 6) * E32 * var
    rstd = (var + eps).rsqrt()
    er = ev / (2 * (var + eps)) + 4 * E32                       # relative
    er = er + er * er * 2
    y = d * rstd * w + b
    ey = (rstd * em * (1 + er) + d.abs() * rstd * (er + 4 * E32)) * w.abs() + E32 * (y.abs() + b.abs())
    return {"y": (y, ey), "mean": (mean[:, 0], em[:, 0]), "rstd": (rstd[:, 0], (er * rstd)[:, 0])}


def norm_backward(x, dy, weight, mean, rstd, add=None):
    """from exact x, mean and rstd"""
    x, dy, mean, rstd = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
    rows, n = x.shape
    w = torch.ones(n, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    xh = (x - mean) * rstd
    v = dy * w
    m1, m2 = v.mean(1, keepdim=True), (v * xh).mean(1, keepdim=True)
    e1, e2 = (DEPTH + 3) * E32 * v.abs().mean(1, keepdim=True), (DEPTH + 6) * E32 * (v * xh).abs().mean(1, keepdim=True)
    dx = rstd * (v - m1 - xh * m2)
    ex = rstd * (e1 + xh.abs() * e2 + 8 * E32 * (v.abs() + m1.abs() + (xh * m2).abs()))
    if add is not None:
        dx, ex = dx + add.double(), ex + 2 * E32 * (dx.abs() + add.double().abs())
    return {"dx": (dx, ex), "dweight": ((dy * xh).sum(0), (rows + 4) * E32 * (dy * xh).abs().sum(0)),
            "dbias": (dy.sum(0), (rows + 1) * E32 * dy.abs().sum(0))}


def check(got, ref, what=""):
    """got, a tensor of its type, against (value, bound): the bound and one rounding to the type"""
    value, bound = ref
    assert got.shape == value.shape, (what, got.shape, value.shape)
    g = got.double()
    assert torch.isfinite(g).all(), what + ": not finite"
    allowed = bound * 1.01 + UNIT[got.dtype] * (value.abs() + bound) * 1.001 + TINY[got.dtype]
    worst = ((g - value).abs() / allowed).max().item() if g.numel() else 0.0
    assert worst <= 1.0, "%s: %.3g times the bound" % (what, worst)
