"""What the fused linear layer and the layer norm cost: the cases, their inputs, their plain forms and their 64-bit values.

Four operators, two of them the backward passes of the other two:

  linear            y = act(x w^T + b) + r, and for training z = x w^T + b beside it
  linear_backward   dz = dy * act'(z);  dx = dz w;  dw = dz^T x;  db = sum of dz over the rows
  layer_norm        y = (x - mean) * rstd * g + b, with mean and rstd of every row beside it
  layer_norm_backward   dx, dg, db

With `own` false `run` computes them from elementary torch operations in 32 bits, rounded once at the end; with `own` true it
calls the package's entry points on the same tensors.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5


def _linear(name, m, k, n, dtype, act, bias=True, residual=False, save=False):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias, "residual": residual,
            "save": save}


def _linear_backward(name, m, k, n, dtype, act):
    return {"name": name, "op": "linear_backward", "m": m, "k": k, "n": n, "dtype": dtype, "act": act}


def _norm(name, op, rows, d, dtype):
    return {"name": name, "op": op, "rows": rows, "d": d, "dtype": dtype}


def listed():
    return [
        # one token through the wide projection of a decoder's feed-forward block: all of it is reading the weights
        _linear("linear 1 token up", 1, 4096, 14336, "bf16", "gelu_tanh"),
        # sixteen sequences decoded together, the narrow projection of that block, added to the residual stream
        _linear("linear 16 tokens down", 16, 14336, 4096, "f16", "none", residual=True),
        # a short prompt or a batch of drafted tokens, no bias: between reading weights and multiplying
        _linear("linear 200 tokens", 200, 4096, 6144, "bf16", "silu", bias=False),
        # nothing is a multiple of anything: rows that do not begin on 16 bytes
        _linear("linear ragged", 77, 1003, 517, "f16", "relu", residual=True),
        # the forward pass of a training step (or of a prompt), which keeps what the backward pass needs
        _linear("linear train up", 2048, 4096, 14336, "bf16", "gelu", save=True),
        # the backward pass of a small head on a small batch: latency
        _linear_backward("linear backward small", 24, 512, 2048, "bf16", "relu"),
        # sizes that fill neither the tiles nor the GPU
        _linear_backward("linear backward ragged", 1000, 1024, 1000, "f16", "silu"),
        # the backward pass of the training step above
        _linear_backward("linear backward train up", 2048, 4096, 14336, "bf16", "gelu"),
        # the norm before a decoded token's projections
        _norm("norm 1 token", "layer_norm", 1, 4096, "bf16"),
        # the norm over a training batch or a long prompt
        _norm("norm 16384 tokens", "layer_norm", 16384, 4096, "bf16"),
        # odd rows in 32 bits
        _norm("norm backward ragged", "layer_norm_backward", 333, 1003, "f32"),
        # the backward pass of a wide model's norm over a training batch
        _norm("norm backward 8192 tokens", "layer_norm_backward", 8192, 8192, "bf16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A width: two in three a multiple of 64, as most models have them, the others as they come."""
    v = _spread(rng, low, high)
    return v if rng.random() < 1 / 3 else max(64, v // 64 * 64)


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_backward", "layer_norm", "layer_norm_backward"])
    dtype = rng.choice(["bf16", "f16"]) if op.startswith("linear") else rng.choice(["bf16", "f16", "f32"])
    if op.startswith("linear"):
        while True:
            m, k, n = _spread(rng, 1, 4096), _width(rng, 64, 14336), _width(rng, 64, 14336)
            if m * k * n <= 2048 * 4096 * 14336:
                break
        act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
        if op == "linear_backward":
            return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "act": act}
        return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": rng.random() < 0.7,
                "residual": rng.random() < 0.4, "save": act != "none" and rng.random() < 0.4}
    while True:
        rows, d = _spread(rng, 1, 16384), _width(rng, 16, 16384)
        if rows * d <= (1 << 26 if dtype != "f32" else 1 << 25):
            break
    return {"op": op, "rows": rows, "d": d, "dtype": dtype}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale)

    s = dict(case)
    if case["op"].startswith("linear"):
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = randn(m, k).to(dt)
        s["w"] = randn(n, k, scale=k ** -0.5).to(dt)
        bias = randn(n, scale=0.1).to(dt)
        if case["op"] == "linear":
            s["bias"] = bias if case["bias"] else None
            s["r"] = randn(m, n).to(dt) if case["residual"] else None
        else:
            # what the forward pass kept: the products before the activation, in the activations' type
            s["z"] = (s["x"].float() @ s["w"].float().t() + bias.float()).to(dt) if case["act"] != "none" else None
            s["dy"] = randn(m, n, scale=0.1).to(dt)
        return s
    rows, d = case["rows"], case["d"]
    # rows of different size and offset, and a few channels far larger than the others, as residual streams have
    x = randn(rows, d) * (0.5 + 2 * torch.rand(rows, 1, generator=g, device="cuda")) + randn(rows, 1, scale=0.5)
    x[:, :: max(1, d // 7)] *= 8
    s["x"] = x.to(dt)
    s["g"] = (1 + randn(d, scale=0.2)).to(dt)
    s["b"] = randn(d, scale=0.2).to(dt)
    if case["op"] == "layer_norm_backward":
        s["dy"] = randn(rows, d, scale=0.1).to(dt)
        x64 = s["x"].double()
        mean = x64.mean(1)
        s["mean"] = mean.float()
        s["rstd"] = (1 / torch.sqrt((x64 - mean[:, None]).square().mean(1) + EPS)).float()
    return s


# ---------------------------------------------------------------- the plain forms

_C = math.sqrt(2 / math.pi)


def _act(z, act):
    if act == "relu":
        return torch.clamp_min(z, 0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(_C * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        t = torch.tanh(_C * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * _C * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain(s):
    op, dt = s["op"], s["x"].dtype
    x = s["x"].float()
    if op == "linear":
        z = x @ s["w"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = _act(z, s["act"])
        if s["r"] is not None:
            y = y + s["r"].float()
        return {"y": y.to(dt), "z": z.to(dt)} if s["save"] else {"y": y.to(dt)}
    if op == "linear_backward":
        dz = s["dy"].float()
        if s["act"] != "none":
            dz = dz * _act_slope(s["z"].float(), s["act"])
        return {"dx": (dz @ s["w"].float()).to(dt), "dw": (dz.t() @ x).to(dt), "db": dz.sum(0).to(dt)}
    if op == "layer_norm":
        mean = x.mean(1)
        c = x - mean[:, None]
        rstd = 1 / torch.sqrt((c * c).mean(1) + EPS)
        return {"y": (c * rstd[:, None] * s["g"].float() + s["b"].float()).to(dt), "mean": mean, "rstd": rstd}
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    h = (x - s["mean"][:, None]) * rstd
    a = dy * s["g"].float()
    dx = rstd * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True))
    return {"dx": dx.to(dt), "dg": (dy * h).sum(0).to(dt), "db": dy.sum(0).to(dt)}


# ---------------------------------------------------------------- the package's operators

def _own(s):
    from torch_vulkan_b200 import cabi

    op = s["op"]
    if op == "linear":
        got = cabi.linear(s["x"], s["w"], s["bias"], residual=s["r"], activation=s["act"], save_preactivation=s["save"])
        return {"y": got[0], "z": got[1]} if s["save"] else {"y": got}
    if op == "linear_backward":
        dx, dw, db = cabi.linear_backward(s["dy"], s["x"], s["w"], s["z"], activation=s["act"])
        return {"dx": dx, "dw": dw, "db": db}
    if op == "layer_norm":
        y, mean, rstd = cabi.layer_norm(s["x"], s["g"], s["b"], EPS)
        return {"y": y, "mean": mean, "rstd": rstd}
    dx, dg, db = cabi.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["g"])
    return {"dx": dx, "dg": dg, "db": db}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"].startswith("linear"):
        m, k, n = case["m"], case["k"], case["n"]
        if case["op"] == "linear":
            outs = m * n * (1 + bool(case["save"]))
            return {"bytes": size * (m * k + n * k + n * bool(case["bias"]) + m * n * bool(case["residual"]) + outs), "flops": 2 * m * n * k}
        saved = m * n * (case["act"] != "none")
        return {"bytes": size * (m * n + saved + 2 * m * k + 2 * n * k + n), "flops": 4 * m * n * k}
    rows, d = case["rows"], case["d"]
    if case["op"] == "layer_norm":
        return {"bytes": size * (2 * rows * d + 2 * d) + 8 * rows, "flops": 8 * rows * d}
    return {"bytes": size * (3 * rows * d + 3 * d) + 8 * rows, "flops": 14 * rows * d}


# ---------------------------------------------------------------- the same values from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "linear":
        z = torch.einsum("mk,nk->mn", x, s["w"].double())
        if case["bias"]:
            z += s["bias"].double()
        y = _phi(z, case["act"])[0]
        if case["residual"]:
            y = y + s["r"].double()
        return {"y": y, "z": z} if case["save"] else {"y": y}
    if case["op"] == "linear_backward":
        delta = s["dy"].double()
        if case["act"] != "none":
            delta = delta * _phi(s["z"].double(), case["act"])[1]
        return {"dx": torch.einsum("mn,nk->mk", delta, s["w"].double()), "dw": torch.einsum("mn,mk->nk", delta, x),
                "db": torch.einsum("mn->n", delta)}
    g = s["g"].double()
    d = x.shape[1]
    if case["op"] == "layer_norm":
        var, mean = torch.var_mean(x, dim=1, correction=0)
        sd = (var + EPS).sqrt()
        return {"y": torch.addcmul(s["b"].double().expand_as(x), (x - mean[:, None]) / sd[:, None], g), "mean": mean, "rstd": sd.reciprocal()}
    dy, mean, rstd = s["dy"].double(), s["mean"].double(), s["rstd"].double()
    # y = g h + b with h = (x - mean) rstd:  dL/dx_j = rstd (u_j - <u> - h_j <u h>),  u = g dy,  <.> the mean over the row
    h = torch.einsum("rd,r->rd", x - mean[:, None], rstd)
    u = torch.einsum("rd,d->rd", dy, g)
    first, second = torch.einsum("rd->r", u) / d, torch.einsum("rd,rd->r", u, h) / d
    return {"dx": torch.einsum("rd,r->rd", u - first[:, None] - torch.einsum("rd,r->rd", h, second), rstd),
            "dg": torch.einsum("rd,rd->d", dy, h), "db": torch.einsum("rd->d", dy)}


def _phi(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        on = z > 0
        return torch.where(on, z, torch.zeros_like(z)), on.double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    # 0.5 (1 + tanh(u)) = sigmoid(2 u)
    v = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z.pow(3))
    s = torch.sigmoid(v)
    slope = 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z.square())
    return z * s, s + z * s * torch.sigmoid(-v) * slope
