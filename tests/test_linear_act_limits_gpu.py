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


def test_the_longest_sum():
    """The weight gradient of 2^31 - 1024 rows (34 GB each of x and dy): one cluster's work, and more of it than its other waits
    are allowed to last. Rows are zero but for some at the beginning, around 2^30 and at the end, whose products are exact."""
    m, k, n = 2 ** 31 - 1024, 8, 8
    x, dy = (torch.zeros(m, c, dtype=torch.bfloat16, device="cuda") for c in (k, n))
    want = torch.zeros(n, k, dtype=torch.float64)
    for seed, first in enumerate((0, 2 ** 30 - 40, m - 77)):
        a, b = (torch.randint(-4, 5, (77, c), generator=D.gen(2 * seed + i)).float() for i, c in enumerate((k, n)))
        x[first:first + 77], dy[first:first + 77] = a.to(torch.bfloat16).cuda(), b.to(torch.bfloat16).cuda()
        want += b.double().t() @ a.double()
    w = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
    dw = run(cabi.linear_backward, dy, x, w, need=(False, True, False))[1]
    assert torch.equal(dw.cpu(), want.to(torch.bfloat16))  # (whole numbers below 2^24, rounded once)
