"""The fused linear layer at the ends of its ranges: values far into the activations' tails and infinite ones, sums of thousands of
values on the kernel of CTA pairs, offsets beyond 31 bits with results that show every row, the longest sum."""

import pytest
import torch

import _dense as D
from torch_vulkan_b200 import cabi

pytestmark = pytest.mark.gpu


def run(fn, *args, **kw):
    torch.cuda.synchronize()
    got = fn(*args, **kw)
    cabi.synchronize()
    return got


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("act", D.ACTS)
@pytest.mark.parametrize("cols", [64, 67])
def test_slopes_far_out_and_at_infinity(dtype, act, cols):
    """act' of a z whose square or cube is beyond float32, or that is infinite (a float16 z beyond 65504), is at its limit."""
    inf = float("inf")
    far = torch.tensor([0.5, -0.5, 6, -6, 13, -13, 29, -29, 31, -31, 90, -90, 127, -127, 129, -129, 1e3, -1e3, 6e4, -6e4, 1e12, -1e12, 2e13, -2e13,
                        1e19, -1e19, 2e19, -2e19, 3e38, -3e38, inf, -inf, 0.0, -0.0]).to(dtype)
    z = torch.zeros(3, cols, dtype=dtype)
    z[1, :len(far)] = far
    dy = torch.randn(3, cols, generator=D.gen(1)).to(dtype)
    w = torch.eye(cols).to(dtype)
    dx, _, db = run(cabi.linear_backward, dy.cuda(), torch.zeros(3, cols, dtype=dtype, device="cuda"), w.cuda(), z.cuda(), activation=act)
    # (in 64 bits the formulas hold up to 1e6, where every slope is at its limit to the last bit)
    want = D.linear_backward64(dy, torch.zeros(3, cols, dtype=dtype), w, z.double().clamp(-1e6, 1e6), act)
    D.check("dx", dx, *want["dx"])
    D.check("db", db, *want["db"])
    if act not in ("none", "relu"):
        z[2, 5] = float("nan")
        dx = run(cabi.linear_backward, dy.cuda(), torch.zeros(3, cols, dtype=dtype, device="cuda"), w.cuda(), z.cuda(), activation=act,
                 need=(True, False, False))[0]
        assert torch.isnan(dx[2]).all() and torch.isfinite(dx[:2]).all()
