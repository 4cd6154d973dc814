"""More of the layer norm on the GPU: parameters of their own type without a weight, sums over more rows than 31 bits of values."""

import pytest
import torch
import torch.nn.functional as F

import _dense as D
from torch_vulkan_b200 import cabi

pytestmark = pytest.mark.gpu


def run(fn, *args, **kw):
    torch.cuda.synchronize()
    got = fn(*args, **kw)
    cabi.synchronize()
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [40, 1003, 2048])
def test_a_float32_bias_without_a_weight_keeps_a_float32_gradient(dtype, d):
    rows = 300
    x, dy = torch.randn(rows, d, generator=D.gen(1)).to(dtype), torch.randn(rows, d, generator=D.gen(2)).to(dtype)
    bias = torch.randn(d, generator=D.gen(3)).to("vk").requires_grad_(True)
    vx = x.to("vk").requires_grad_(True)
    F.layer_norm(vx, (d,), None, bias).backward(dy.to("vk"))
    assert bias.grad.dtype == torch.float32
    size = dy.double().abs().sum(0)
    want = dy.double().sum(0)
    D.check("db", bias.grad.cpu(), want, D.rounded(want, D.sum_slack(rows) * size, torch.float32))
    mean, rstd = cabi.layer_norm(x.cuda())[1:]
    got = run(cabi.layer_norm_backward, dy.cuda(), x.cuda(), mean, rstd, param_dtype=torch.float32)
    assert got[1].dtype == got[2].dtype == torch.float32
    D.check("db", got[2], want, D.rounded(want, D.sum_slack(rows) * size, torch.float32))
    grads = D.layer_norm_backward64(dy, x, mean.cpu(), rstd.cpu(), torch.ones(d))
    D.check("dg", got[1], *grads["dg"])
    with pytest.raises(ValueError, match="parameters"):
        cabi.layer_norm_backward(dy.cuda(), x.cuda(), mean, rstd, param_dtype=torch.float64)
