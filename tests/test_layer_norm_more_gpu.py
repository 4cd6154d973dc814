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


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 4096), (torch.bfloat16, 1000), (torch.float16, 16384), (torch.bfloat16, 1003), (torch.float32, 8192)])
def test_sums_over_rows_beyond_31_bits(dtype, d):
    """dweight and dbias of more than 2^31 values of dy, which is 0 but in some rows at the beginning, where the offsets pass
    2^31, and at the end: the sums are those of these rows, and bounded by them."""
    rows = 2 ** 31 // d + 300
    x = torch.randn(rows, d, device="cuda", dtype=dtype)
    g, b = (1 + 0.3 * torch.randn(d, generator=D.gen(1))).to(dtype).cuda(), torch.randn(d, generator=D.gen(2)).to(dtype).cuda()
    some = torch.cat([torch.arange(0, 40), torch.arange(2 ** 31 // d - 100, 2 ** 31 // d + 100), torch.arange(rows - 60, rows)]).cuda()
    dy = torch.zeros_like(x)
    dy[some] = torch.randn(len(some), d, generator=D.gen(3)).to(dtype).cuda()
    _, mean, rstd = run(cabi.layer_norm, x, g, b)
    dx, dg, db = run(cabi.layer_norm_backward, dy, x, mean, rstd, g)
    want = D.layer_norm_backward64(dy[some], x[some], mean[some], rstd[some], g)
    for name, got in (("dg", dg), ("db", db)):
        value, bound = want[name]
        assert bound.abs().median() < 0.02 * value.abs().median()  # (sums of nothing, or without some rows, are beyond it)
        D.check(name, got, value, bound)
    D.check("dx", dx[some], *want["dx"])
    assert int(torch.count_nonzero(dx.count_nonzero(1))) <= len(some)
