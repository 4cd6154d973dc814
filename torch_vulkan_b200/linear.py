"""Linear layers over the quantised matrix products: the caller's side of the path.

The reference stops at the three aten ops (crates/pyvk/csrc/quant.cpp:315-322); what calls them in a model is a
Linear whose weight was quantised ahead of time ("as LLaMA's LM head passes it", tests/python/test_quant.py:34).
These modules hold the weights in the form the ops take, so that a forward is one product (plus the bias):

* Int8Linear      aten::_weight_int8pack_mm: int8 weights [N, K], one scale per output feature.
* DynInt4Linear   aten::_dyn_quant_pack_4bit_weight once, aten::_dyn_quant_matmul_4bit per forward: int4 weights in
                  blocks of `block_size` along K (or one block per row), activations quantised per row on the fly.

Both work on whatever device their tensors live on ("vk": the B200 kernels; CPU: PyTorch's own kernels for the same ops,
which is how the logic is tested without a GPU) and both can hold one rank's slice of the output features of a Linear
sharded over the GPUs of a node (`shard(rank, world)`): the forward then assembles the full output on every rank.
`swap_linears` replaces the nn.Linear modules of a model in place; `save` / `load` keep the quantised form on disk so
that a restart skips the quantisation.

The layers that stay in 16 or 32 bits have a form of their own: `linear_act` (and the module LinearAct) is a Linear with its
activation and the residual stream it joins in one call, act(x @ weight.T + bias) + residual, with gradients; `fuse_linears`
puts it in place of the Linear / activation pairs of a model.
"""

import math

import torch
import torch.nn.functional as F
from torch import nn
from torch.autograd.function import once_differentiable

from . import shard as _shard


def quantize_int8_per_channel(weight):
    """float [N, K] -> (int8 [N, K], float32 scales [N]) with weight ~= q * scale: symmetric, absmax / 127 per row."""
    w = weight.detach().to(torch.float32).cpu()
    scales = w.abs().amax(dim=1).clamp_min(1e-12) / 127.0
    q = torch.round(w / scales[:, None]).clamp_(-127, 127).to(torch.int8)
    return q, scales


def quantize_int4_groupwise(weight, block_size):
    """float [N, K] -> (uint8 [N, K/2] nibble pairs, float32 scales [N, K/block_size]) in the layout
    aten::_dyn_quant_pack_4bit_weight takes: value = (nibble - 8) * scale, the even k in the low nibble, the odd k in
    the high one (as ATen/native/cpu/int4mm_kernel.cpp's ref_dyn_quant_matmul_4bit_* and the reference's shader read them)."""
    w = weight.detach().to(torch.float32).cpu()
    n, k = w.shape
    if k % 2 or k % block_size:
        raise ValueError(f"in_features={k} must be even and a multiple of block_size={block_size}")
    blocks = w.reshape(n, k // block_size, block_size)
    scales = blocks.abs().amax(dim=2).clamp_min(1e-12) / 7.0
    q = torch.round(blocks / scales[:, :, None]).clamp_(-8, 7).to(torch.int16).reshape(n, k) + 8
    packed = ((q[:, 1::2] << 4) | q[:, 0::2]).to(torch.uint8)
    return packed, scales


class _ShardedMixin:
    rank, world = 0, 1
    _group = None

    def _gather(self, y_local):
        if self.world == 1:
            return y_local
        return _shard.all_gather_columns(y_local, self._group)

    def _finish(self, y_local, lead, residual):
        """The full output in the caller's shape, with the residual stream (a tensor of that shape) added in place."""
        y = self._gather(y_local).reshape(*lead, self.full_out_features)
        if residual is not None:
            if residual.shape != y.shape:
                raise ValueError(f"residual of shape {tuple(residual.shape)} for an output of shape {tuple(y.shape)}")
            y += residual.contiguous()
        return y


class Int8Linear(nn.Module, _ShardedMixin):
    """y = x @ (weight_int8 * scales[:, None]).T + bias through aten::_weight_int8pack_mm.

    `scales` are kept in the activations' dtype (the op requires it); pass `dtype` to choose it."""

    def __init__(self, weight_int8, scales, bias=None, dtype=torch.bfloat16):
        super().__init__()
        if weight_int8.dtype != torch.int8 or weight_int8.dim() != 2:
            raise ValueError("weight_int8 must be an int8 matrix [out_features, in_features]")
        if scales.shape != (weight_int8.shape[0],):
            raise ValueError("scales must have one entry per output feature")
        self.out_features, self.in_features = weight_int8.shape
        self.register_buffer("weight", weight_int8.contiguous())
        self.register_buffer("scales", scales.to(dtype).contiguous())
        self.register_buffer("bias", None if bias is None else bias.detach().to(dtype).contiguous())
        self.full_out_features = self.out_features

    @classmethod
    def from_float(cls, linear, dtype=torch.bfloat16):
        q, s = quantize_int8_per_channel(linear.weight)
        return cls(q, s, None if linear.bias is None else linear.bias.detach().cpu(), dtype=dtype)

    def shard(self, rank, world, group=None):
        """Keeps only `rank`'s rows (output features); the forward gathers the full output (NCCL on "vk", gloo on CPU)."""
        out = Int8Linear(_shard.shard_rows(self.weight, rank, world), _shard.shard_rows(self.scales, rank, world),
                         None if self.bias is None else _shard.shard_rows(self.bias, rank, world), dtype=self.scales.dtype)
        out.rank, out.world, out._group, out.full_out_features = rank, world, group, self.out_features
        return out

    def forward(self, x, residual=None):
        """`residual`: a tensor of the output's shape added to it (x + proj(h) of a decoder block in one call)."""
        lead = x.shape[:-1]
        x2 = x.reshape(-1, self.in_features)
        if x2.dtype != self.scales.dtype:
            raise TypeError(f"Int8Linear holds {self.scales.dtype} scales; got {x2.dtype} activations")
        if x2.device.type == "vk" and self.world == 1 and (self.bias is not None or residual is not None):
            # one call for product, bias and residual (one launch when at most 32 rows are decoded); same roundings
            if residual is not None and residual.shape != (*lead, self.out_features):
                raise ValueError(f"residual of shape {tuple(residual.shape)} for an output of shape {(*lead, self.out_features)}")
            from . import _native
            r2 = None if residual is None else residual.reshape(-1, self.out_features)
            return _native.int8_linear(x2, self.weight, self.scales, self.bias, r2).reshape(*lead, self.out_features)
        y = torch._weight_int8pack_mm(x2, self.weight, self.scales)
        if self.bias is not None:
            y += self.bias
        return self._finish(y, lead, residual)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.full_out_features}, bias={self.bias is not None}, "
                f"dtype={self.scales.dtype}" + (f", rows {self.rank}/{self.world}" if self.world > 1 else ""))


class DynInt4Linear(nn.Module, _ShardedMixin):
    """y = dynamically quantised x @ int4 weights + bias through aten::_dyn_quant_matmul_4bit (float32 or bfloat16 x).

    Holds the tensor aten::_dyn_quant_pack_4bit_weight returns; on "vk" the tensor-core form of the weights is derived
    from it once and cached by the backend for as long as this tensor lives."""

    def __init__(self, packed, block_size, in_features, out_features):
        super().__init__()
        self.block_size, self.in_features, self.out_features = block_size, in_features, out_features
        self.full_out_features = out_features
        self.register_buffer("packed", packed)

    @classmethod
    def from_quantized(cls, nibbles, scales, bias, block_size, device=None):
        """nibbles uint8 [N, K/2], scales [N, K/block_size] (bfloat16 for blocks, float32 for one block per row),
        bias float32 [N] or None: the arguments of aten::_dyn_quant_pack_4bit_weight."""
        n, k = nibbles.shape[0], nibbles.shape[1] * 2
        if device is not None:
            nibbles, scales = nibbles.to(device), scales.to(device)
            bias = None if bias is None else bias.to(device)
        packed = torch._dyn_quant_pack_4bit_weight(nibbles, scales, bias, block_size, k, n)
        return cls(packed, block_size, k, n)

    @classmethod
    def from_float(cls, linear, block_size=32, device=None):
        k = linear.in_features
        nibbles, scales = quantize_int4_groupwise(linear.weight, block_size)
        scales = scales.to(torch.bfloat16) if block_size < k else scales.to(torch.float32)
        bias = None if linear.bias is None else linear.bias.detach().to(torch.float32).cpu()
        return cls.from_quantized(nibbles, scales, bias, block_size, device)

    def shard(self, rank, world, group=None):
        lo, hi = _shard.shard_bounds(self.out_features, rank, world)
        part = _shard.shard_packed_4bit(self.packed, self.block_size, self.in_features, self.out_features, rank, world)
        out = DynInt4Linear(part, self.block_size, self.in_features, hi - lo)
        out.rank, out.world, out._group, out.full_out_features = rank, world, group, self.out_features
        return out

    def forward(self, x, residual=None):
        lead = x.shape[:-1]
        x2 = x.reshape(-1, self.in_features)
        y = torch._dyn_quant_matmul_4bit(x2, self.packed, self.block_size, self.in_features, self.out_features)
        return self._finish(y, lead, residual)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.full_out_features}, block_size={self.block_size}"
                + (f", rows {self.rank}/{self.world}" if self.world > 1 else ""))


def _rows(t, cols):
    """A [rows, cols] form of t that the kernels can read: contiguous columns, rows that do not overlap (a copy where there is
    none, for instance of an expanded gradient)."""
    t = t.reshape(math.prod(t.shape[:-1]), cols)
    if (cols > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t


def _apply(x, w, bias, residual, activation, keep):
    """The kernel on matrices: (y, the values before the activation or None)."""
    from . import cabi

    r = None if residual is None else _rows(residual, w.shape[0])
    y = cabi.linear(x, w, bias, residual=r, activation=activation, save_preactivation=keep)
    return y if keep else (y, None)


def _shaped(y, lead):
    """y [rows, n] in the caller's shape, as a tensor of its own: a view (of a custom function's output, or made while gradients
    are off) could not be written to in place afterwards, as an nn.Linear's output can."""
    return y if len(lead) == 1 else torch.ops.aten._unsafe_view(y, (*lead, y.shape[1]))


class _LinearAct(torch.autograd.Function):
    """cabi.linear and cabi.linear_backward as one differentiable operation. Keeps x, the weight and, with an activation, the
    values before it."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        x2, w2 = _rows(x, weight.shape[1]), _rows(weight, weight.shape[1])
        ctx.on_vk = x.device.type == "vk"
        y, z = _apply(x2, w2, bias, residual, activation, ctx.on_vk and activation != "none" and any(ctx.needs_input_grad[:3]))
        if ctx.on_vk:
            ctx.save_for_backward(x2, w2, z)
        ctx.activation, ctx.x_shape = activation, x.shape
        return _shaped(y, x.shape[:-1])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        from . import cabi

        if not ctx.on_vk:
            raise NotImplementedError("no gradients through CUDA tensors (PyTorch's autograd engine serves device \"vk\" in this "
                                      "process): call cabi.linear_backward")
        x2, w2, z = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        dx = dw = db = None
        if any(need):
            dx, dw, db = cabi.linear_backward(_rows(dy, w2.shape[0]), x2, w2, z, activation=ctx.activation, need=need)
        # (contiguous, so that it can be added to other gradients of the same tensor: x may be its own residual)
        return (None if dx is None else dx.view(ctx.x_shape)), dw, db, (dy.contiguous() if ctx.needs_input_grad[3] else None), None


def _has_kernel(x):
    """Whether the fused kernel serves x: on "vk" always (it refuses what it cannot do), of CUDA tensors those of its types where
    autocast asks for no other."""
    return x.device.type == "vk" or (x.device.type == "cuda" and x.dtype in (torch.float32, torch.float16, torch.bfloat16)
                                     and not torch.is_autocast_enabled("cuda"))


def linear_act(x, weight, bias=None, activation="none", residual=None):
    """act(x @ weight.T + bias) + residual: x [..., in], weight [out, in], bias [out], residual [..., out], all of one dtype
    (float32, float16 or bfloat16). activation: "none", "relu", "gelu" (by erf), "gelu_tanh" or "silu". Differentiable (once)
    in every operand. On "vk" one kernel computes it (tvb_linear; the gradients: tvb_linear_backward). CUDA tensors of those types
    take the kernel too, without gradients: PyTorch's autograd engine serves one accelerator per process, and here that is
    "vk" (a backward pass through them raises, as through any CUDA tensor; cabi.linear_backward computes them when called).
    Anything else that an nn.Linear runs on (the CPU, the meta device, float64, autocast on CUDA) takes PyTorch's own operations."""
    from . import cabi

    if activation not in cabi.ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(cabi.ACTIVATIONS)}, got {activation!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x of shape {tuple(x.shape)} does not go with a weight of shape {tuple(weight.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], weight.shape[0]):
        raise ValueError(f"residual of shape {tuple(residual.shape)} for an output of shape {(*x.shape[:-1], weight.shape[0])}")
    if not _has_kernel(x):
        y = F.linear(x, weight, bias)
        y = {"none": lambda t: t, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"),
             "silu": F.silu}[activation](y)
        return y if residual is None else y + residual
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _LinearAct.apply(x, weight, bias, residual, activation)
    k = weight.shape[1]
    return _shaped(_apply(_rows(x, k), _rows(weight, k), bias, residual, activation, False)[0], x.shape[:-1])


class LinearAct(nn.Linear):
    """nn.Linear (its parameters, its state dict) with an activation and, in the call, a residual: `linear_act` as a module."""

    def __init__(self, in_features, out_features, bias=True, activation="none", device=None, dtype=None):
        from . import cabi

        if activation not in cabi.ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(cabi.ACTIVATIONS)}, got {activation!r}")
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.activation = activation

    @classmethod
    def from_float(cls, linear, activation="none"):
        """The same layer (it shares `linear`'s parameters) followed by `activation`."""
        out = cls(linear.in_features, linear.out_features, bias=linear.bias is not None, activation=activation, device="meta")
        out.weight, out.bias = linear.weight, linear.bias
        return out.train(linear.training)

    def forward(self, x, residual=None):
        return linear_act(x, self.weight, self.bias, self.activation, residual)

    def extra_repr(self):
        return super().extra_repr() + f", activation={self.activation}"


def _activation_name(module):
    """What LinearAct calls an activation module, or None."""
    if type(module) is nn.ReLU:
        return "relu"
    if type(module) is nn.GELU:
        return "gelu" if module.approximate == "none" else "gelu_tanh"
    return "silu" if type(module) is nn.SiLU else None


def _hooked(module):
    return any(getattr(module, kind) for kind in ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks"))


def fuse_linears(model, plain=False):
    """Replaces, in every nn.Sequential under `model` (in place), an nn.Linear that is followed by ReLU, GELU or SiLU with one
    LinearAct that shares its parameters, and the activation with nn.Identity (so that the other layers keep their names).
    plain: every other nn.Linear under `model`, whatever it stands in, becomes a LinearAct without an activation too. A model that
    trains on "vk" needs that: an nn.Linear's own backward pass asks for the sum of its bias's gradient, which has no kernel there.
    Left as they are: layers with hooks (a fused one would not run them), and containers with a forward pass of their own (but for
    `plain`). Returns the names of the layers it replaced."""
    replaced = []
    for name, module in list(model.named_modules()):
        if not isinstance(module, nn.Sequential) or type(module).forward is not nn.Sequential.forward:
            continue
        children = list(module._modules.items())  # (named_children leaves out a module's second place in the container)
        for (first, linear), (second, act) in zip(children, children[1:]):
            activation = _activation_name(act)
            if type(linear) is not nn.Linear or activation is None or _hooked(linear) or _hooked(act):
                continue
            setattr(module, first, LinearAct.from_float(linear, activation))
            setattr(module, second, nn.Identity())
            replaced.append(f"{name}.{first}" if name else first)
    made = {}  # (a layer that stands in two places stays one)
    for name, module in list(model.named_modules()) if plain else []:
        for key, child in list(module._modules.items()):
            if type(child) is not nn.Linear or _hooked(child):
                continue
            if child not in made:
                made[child] = LinearAct.from_float(child)
            setattr(module, key, made[child])
            replaced.append(f"{name}.{key}" if name else key)
    return replaced


def swap_linears(model, kind="int8", dtype=torch.bfloat16, block_size=32, device=None, skip=None):
    """Replaces every nn.Linear under `model` (in place) with its quantised counterpart, quantising on the CPU and moving
    the result to `device`. kind: "int8" (Int8Linear) or "dyn4" (DynInt4Linear). `skip(name, module)` keeps a layer as is; a
    LinearAct with an activation is kept too (the quantised layers have none). Returns the names of the layers it replaced."""
    if kind not in ("int8", "dyn4"):
        raise ValueError("kind must be 'int8' or 'dyn4'")
    replaced = []
    for name, module in list(model.named_modules()):
        for child_name, child in list(module.named_children()):
            full = f"{name}.{child_name}" if name else child_name
            if not isinstance(child, nn.Linear) or (skip is not None and skip(full, child)):
                continue
            if isinstance(child, LinearAct) and child.activation != "none":
                continue
            if kind == "int8":
                new = Int8Linear.from_float(child, dtype=dtype)
                if device is not None:
                    new = new.to(device)
            else:
                new = DynInt4Linear.from_float(child, block_size=block_size, device=device)
            setattr(module, child_name, new)
            replaced.append(full)
    return replaced


def save(module, path):
    """Writes the quantised form of an Int8Linear / DynInt4Linear (CPU copies of its tensors and its geometry)."""
    if isinstance(module, Int8Linear):
        blob = {"kind": "int8", "weight": module.weight.cpu(), "scales": module.scales.cpu(),
                "bias": None if module.bias is None else module.bias.cpu()}
    elif isinstance(module, DynInt4Linear):
        blob = {"kind": "dyn4", "packed": module.packed.cpu(), "block_size": module.block_size,
                "in_features": module.in_features, "out_features": module.out_features}
    else:
        raise TypeError("save() takes an Int8Linear or a DynInt4Linear")
    torch.save(blob, path)


def load(path, device=None):
    """The module `save` wrote, on `device` (no quantisation and, for int4, no packing is repeated)."""
    blob = torch.load(path, map_location="cpu", weights_only=True)
    if blob["kind"] == "int8":
        out = Int8Linear(blob["weight"], blob["scales"], blob["bias"], dtype=blob["scales"].dtype)
    else:
        out = DynInt4Linear(blob["packed"], blob["block_size"], blob["in_features"], blob["out_features"])
    return out if device is None else out.to(device)
