"""Plain 64-bit forms and error bounds of the fused linear layer and the layer norm, shared by their tests.

A bound counts the roundings of the operator: half a step of the output type (`finfo(t).eps / 2` relative to the value, or
half of the smallest subnormal), and the float32 arithmetic before it. A float32 sum of R products is at most
(R + 4) * 2^-23 * (sum of the products' sizes) off, whether its additions round to nearest or truncate."""

import math

import torch

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float64: 0.0, torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def act64(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.where(z == z, torch.zeros_like(z), z))
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        s = torch.sigmoid(c * (z + 0.044715 * z ** 3))
        return s + z * s * (1 - s) * c * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    return s + z * s * (1 - s)


def sum_slack(terms):
    return (terms + 4) * 2.0 ** -23


def rounded(want, slack, dtype):
    """The bound of a value known to `slack` before its one rounding to dtype."""
    return slack + half_step(dtype) * (want.abs() + slack) + TINY[dtype]


def linear64(x, w, bias, residual, act):
    """(y, bound of y, z, bound of z) with the bounds of x's dtype."""
    x64, w64 = x.double(), w.double()
    z = x64 @ w64.t()
    size = x64.abs() @ w64.abs().t()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    slack_z = sum_slack(x.shape[1] + 1) * size
    y = act64(z, act)
    # |act'| < 1.13; the function itself: 2^-18 of the value (exponential and quotient by the hardware's approximations, the
    # exponent up to 60), and where 1 + erf cancels a few 2^-24 of |z|
    slack = 1.13 * slack_z + 2.0 ** -18 * y.abs() + 2.0 ** -22 * z.abs() if act not in ("none", "relu") else slack_z
    if residual is not None:
        y = y + residual.double()
        slack = slack + 2.0 ** -24 * (y.abs() + slack)
    return y, rounded(y, slack, x.dtype), z, rounded(z, slack_z, x.dtype)


def linear_backward64(dy, x, w, z, act):
    """{name: (value, bound)} of dx, dw, db; dz is rounded to the type once on its way into the products."""
    dt = x.dtype
    dy64, x64, w64 = dy.double(), x.double(), w.double()
    dz = dy64
    slack_dz = torch.zeros_like(dz)
    if act != "none":
        dz = dy64 * slope64(z.double(), act)
        if act != "relu":
            slack_dz = dy64.abs() * (2.0 ** -18 + 2.0 ** -21 * (1 + z.double().abs()))
    round_dz = slack_dz if act in ("none", "relu") else rounded(dz, slack_dz, dt)
    m, n = dy.shape
    got = {}
    for name, a, ra, b, terms in (("dx", dz, round_dz, w64, n), ("dw", dz.t(), round_dz.t(), x64, m)):
        value = a @ b
        slack = ra @ b.abs() + sum_slack(terms) * ((a.abs() + ra) @ b.abs())
        got[name] = (value, rounded(value, slack, dt))
    value = dz.sum(0)
    got["db"] = (value, rounded(value, slack_dz.sum(0) + sum_slack(m) * (dz.abs() + slack_dz).sum(0), dt))
    return got


def layer_norm64(x, weight, bias, eps):
    """{name: (value, bound)} of y, mean, rstd."""
    d = x.shape[1]
    x64 = x.double()
    mean = x64.mean(1)
    slack_mean = sum_slack(d) * x64.abs().mean(1) + 2.0 ** -24 * mean.abs() if d else mean
    c = x64 - mean[:, None]
    var = c.square().mean(1)
    # the centred values are known to the mean's error and a rounding; the variance about the computed mean is larger by its
    # error squared
    slack_c = slack_mean[:, None] + 2.0 ** -23 * c.abs()
    rstd = 1 / (var + eps).sqrt()
    slack_var = (2 * c.abs() * 2.0 ** -23 * c.abs() + slack_c.square()).mean(1) + sum_slack(d) * (c.abs() + slack_c).square().mean(1)
    rel = 0.5 * slack_var / (var + eps) + 3 * 2.0 ** -23
    slack_rstd = rel * rstd
    g = weight.double() if weight is not None else torch.ones(d, dtype=torch.float64, device=x.device)
    b = bias.double() if bias is not None else torch.zeros(d, dtype=torch.float64, device=x.device)
    h = c * rstd[:, None]
    slack_h = slack_c * rstd[:, None] + h.abs() * rel[:, None] + 2.0 ** -24 * h.abs()
    y = h * g + b
    slack_y = slack_h * g.abs() + 2.0 ** -24 * y.abs()
    return {"y": (y, rounded(y, slack_y, x.dtype)), "mean": (mean, slack_mean), "rstd": (rstd, slack_rstd)}


def layer_norm_backward64(dy, x, mean, rstd, weight):
    """{name: (value, bound)} of dx, dg, db, given the statistics."""
    rows, d = x.shape
    pt = weight.dtype if weight is not None else x.dtype
    x64, dy64, mean, rstd = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
    g = weight.double() if weight is not None else torch.ones(d, dtype=torch.float64, device=x.device)
    h = (x64 - mean) * rstd
    u = dy64 * g
    eh = 2.0 ** -22 * h.abs()          # subtraction and product
    eu = 2.0 ** -24 * u.abs()
    mu, muh = u.mean(1, keepdim=True), (u * h).mean(1, keepdim=True)
    au, auh = u.abs().mean(1, keepdim=True), (u * h).abs().mean(1, keepdim=True)
    emu, emuh = (sum_slack(d) + 2.0 ** -22) * au, (sum_slack(d) + 2.0 ** -21) * auh
    dx = rstd * (u - mu - h * muh)
    slack = rstd * (eu + emu + eh * muh.abs() + h.abs() * emuh + 2.0 ** -22 * (u.abs() + mu.abs() + (h * muh).abs()))
    dg, db = (dy64 * h).sum(0), dy64.sum(0)
    size_dg, size_db = (dy64 * h).abs().sum(0), dy64.abs().sum(0)
    return {"dx": (dx, rounded(dx, slack, x.dtype)), "dg": (dg, rounded(dg, (sum_slack(rows) + 2.0 ** -21) * size_dg, pt)),
            "db": (db, rounded(db, sum_slack(rows) * size_db, pt))}


def check(name, got, want, bound):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = (got.double().cpu() - want.cpu()).abs()
    bound = bound.cpu()
    bad = ~(off <= bound)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} values beyond the bound, worst {float((off / bound).max()):.3g} times it"
