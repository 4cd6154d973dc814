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
