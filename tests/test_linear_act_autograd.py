"""linear_act, LinearAct and fuse_linears as parts of other people's models: outputs written in place, inputs used twice, training of
a fused model, the devices and types that an nn.Linear runs on."""

import pytest
import torch
import torch.nn.functional as F
from torch import nn

import _dense as D
from torch_vulkan_b200 import linear as L

gpu = pytest.mark.gpu


def near(got, want, rel):
    off = float((got.detach().cpu().double() - want.double()).norm() / want.double().norm())
    assert off <= rel, off


@gpu
@pytest.mark.parametrize("shape", [(40,), (7, 40), (3, 5, 40), (2, 3, 4, 40)])
@pytest.mark.parametrize("mode", ["grad", "no_grad", "plain"])
def test_outputs_may_be_written_in_place(shape, mode):
    x = torch.randn(shape, generator=D.gen(1))
    w = torch.randn(24, 40, generator=D.gen(2)) / 6
    other = torch.randn(*shape[:-1], 24, generator=D.gen(3))
    vx, vw = x.to("vk"), w.to("vk").requires_grad_(mode == "grad")
    with torch.set_grad_enabled(mode != "no_grad"):
        y = L.linear_act(vx, vw, None, "silu")
    vo = other.to("vk").requires_grad_(mode != "grad")
    y += vo  # (with gradients on)
    want = F.silu(x.double() @ w.double().t()) + other.double()
    near(y, want, 2.0 ** -18)
    dy = torch.randn(y.shape, generator=D.gen(4))
    y.backward(dy.to("vk"))
    if mode == "grad":
        cw = w.double().requires_grad_(True)
        F.silu(x.double() @ cw.t()).backward(dy.double())
        near(vw.grad, cw.grad, 2.0 ** -18)
    else:
        assert torch.equal(vo.grad.cpu(), dy)


@gpu
@pytest.mark.parametrize("how", ["contiguous", "expanded", "transposed"])
@pytest.mark.parametrize("dtype,rel", [(torch.float32, 2.0 ** -18), (torch.bfloat16, 2.0 ** -6)])
def test_an_input_that_is_its_own_residual(how, dtype, rel):
    """x + act(x w^T): both gradients of x are added, whatever the layout of the one that comes in. (16 bits: dz, dx and the sum
    are rounded once each.)"""
    x = torch.randn(24, 24, generator=D.gen(1)).to(dtype)
    w = (torch.randn(24, 24, generator=D.gen(2)) / 5).to(dtype)
    dy = {"contiguous": torch.randn(24, 24, generator=D.gen(3)).to(dtype), "expanded": torch.full((1, 1), 0.5, dtype=dtype).expand(24, 24),
          "transposed": torch.randn(24, 24, generator=D.gen(3)).to(dtype).t()}[how]
    given = {"contiguous": lambda t: t.to("vk"), "expanded": lambda t: t[:1, :1].contiguous().to("vk").expand(24, 24),
             "transposed": lambda t: t.t().contiguous().to("vk").t()}[how](dy)
    vx, vw = x.to("vk").requires_grad_(True), w.to("vk").requires_grad_(True)
    y = L.linear_act(vx, vw, None, "gelu", vx)
    y.backward(given)
    cx, cw = x.double().requires_grad_(True), w.double().requires_grad_(True)
    (F.gelu(cx @ cw.t()) + cx).backward(dy.double())
    near(vx.grad, cx.grad, rel)
    near(vw.grad, cw.grad, rel)


@pytest.mark.parametrize("act", D.ACTS)
def test_a_fused_model_on_the_meta_device(act):
    layer = L.LinearAct(12, 20, activation=act, device="meta")
    x = torch.empty(3, 5, 12, device="meta", requires_grad=True)
    y = layer(x, residual=torch.empty(3, 5, 20, device="meta"))
    assert y.device.type == "meta" and y.shape == (3, 5, 20)
    y.backward(torch.empty_like(y))
    assert x.grad.shape == x.shape and layer.weight.grad.shape == (20, 12)


@gpu
@pytest.mark.parametrize("act", D.ACTS)
def test_cuda_tensors_in_float64_and_under_autocast(act):
    torch.manual_seed(1)
    layer = L.LinearAct(40, 24, activation=act)
    x = torch.randn(7, 40)
    want = layer.double()(x.double())
    layer = layer.cuda()
    with torch.no_grad():
        got = layer(x.double().cuda())
        assert got.dtype == torch.float64
        near(got, want.detach(), 2.0 ** -45)
        layer = layer.float()
        with torch.autocast("cuda", torch.bfloat16):
            got, plain = layer(x.cuda()), F.linear(x.cuda(), layer.weight, layer.bias)
        assert plain.dtype == torch.bfloat16 and got.dtype in (torch.bfloat16, torch.float32)
        near(got, want.detach(), 2.0 ** -6)


@gpu
def test_cuda_tensors_that_require_gradients_run_forward_and_refuse_backward():
    x = torch.randn(7, 40, generator=D.gen(1)).cuda().requires_grad_(True)
    w = torch.randn(24, 40, generator=D.gen(2)).cuda().requires_grad_(True)
    y = L.linear_act(x, w, None, "gelu")
    with torch.no_grad():
        assert torch.equal(y, L.linear_act(x, w, None, "gelu"))
    assert y.requires_grad and y.grad_fn.saved_tensors == ()  # (nothing is kept for a pass that cannot be run)
    with pytest.raises(RuntimeError):
        y.backward(torch.ones_like(y))
    assert x.grad is None and w.grad is None
    vx = x.detach().cpu().to("vk").requires_grad_(True)  # the device's own gradients go on
    L.linear_act(vx, w.detach().cpu().to("vk"), None, "gelu").backward(torch.ones(7, 24).to("vk"))
    assert vx.grad.shape == vx.shape


class TwoBlocks(nn.Module):
    """Linears in every place that fuse_linears has to find: before an activation, alone, in a ModuleDict, one in two places."""

    def __init__(self, d=64, h=160, seed=3):
        super().__init__()
        torch.manual_seed(seed)
        self.ffn = nn.Sequential(nn.LayerNorm(d), nn.Linear(d, h), nn.GELU(), nn.Linear(h, d))
        self.rest = nn.ModuleDict({"gate": nn.Linear(d, h, bias=False), "down": nn.Linear(h, d)})
        self.tied = self.rest["down"]

    def forward(self, x):
        h = self.rest["gate"](self.ffn(x))
        return self.rest["down"](h) + self.tied(h)


def test_fuse_linears_with_the_plain_ones():
    a, b = TwoBlocks(), TwoBlocks()
    kept = b.rest["gate"].register_forward_hook(lambda module, args, out: out)
    assert L.fuse_linears(b, plain=True) == ["ffn.1", "tied", "ffn.3", "rest.down"]
    assert type(b.rest["gate"]) is nn.Linear  # (hooked)
    kept.remove()
    assert L.fuse_linears(b, plain=True) == ["rest.gate"]
    assert all(type(m) is L.LinearAct for m in b.modules() if isinstance(m, nn.Linear)) and b.tied is b.rest["down"]
    assert b.ffn[1].activation == "gelu" and b.ffn[3].activation == "none"
    assert list(a.state_dict()) == list(b.state_dict())
    x = torch.randn(5, 64, generator=D.gen(1))
    assert torch.equal(a(x), b(x))
    assert L.fuse_linears(TwoBlocks()) == ["ffn.1"]


@gpu
@pytest.mark.parametrize("dtype,rel", [(torch.float32, 2.0 ** -17), (torch.bfloat16, 2.0 ** -5)])
def test_a_fused_model_trains_on_vk(dtype, rel):
    """One step's gradients of every parameter against 64 bits (16 bits: some ten roundings between the output and the first
    layer, half a step each)."""
    model, twin = TwoBlocks().to(dtype), TwoBlocks().to(dtype).double()
    L.fuse_linears(model, plain=True)
    model = model.to("vk")
    x, dy = (torch.randn(3, 17, 64, generator=D.gen(i)).to(dtype) for i in (1, 2))
    vx, cx = x.to("vk").requires_grad_(True), x.double().requires_grad_(True)
    y = model(vx)
    y.backward(dy.to("vk"))
    want = twin(cx)
    want.backward(dy.double())
    near(y, want.detach(), rel)
    near(vx.grad, cx.grad, rel)
    names = dict(twin.named_parameters())
    for name, p in model.named_parameters():
        near(p.grad, names[name].grad, rel)
