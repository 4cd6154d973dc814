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


def operands(m, k, n, dtype, seed):
    def rand(*shape, at, scale=1.0):
        return (torch.randn(*shape, generator=D.gen(seed + at)) * scale).to(dtype).cuda()

    return rand(m, k, at=1), rand(n, k, at=2, scale=k ** -0.5), rand(n, at=3, scale=0.3), rand(m, n, at=4)


# Outputs of at least 74 tiles of 256 x 256 whose sums have 8192 values or more: one product on tiles of 512 rows. Whole and ragged
# edges, a last tile row of one half (2100, 1900), rows that do not begin on 16 bytes (2603), the last tiles cut to 256 x 128
# (2100 x 4096: 80 tiles of 512 rows for 74 pairs) and to 256 x 256 (4000 x 3300: 104).
TALL = [(2048, 8200, 2600), (1900, 8192, 2603), (2100, 8192, 4096), (4000, 8264, 3300)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", TALL)
def test_long_sums_forward(dtype, m, k, n):
    x, w, b, r = operands(m, k, n, dtype, seed=100)
    for act, bias, res in (("gelu", b, r), ("none", None, None)):
        want, tol, z64, ztol = D.linear64(x, w, bias, res, act)
        y, z = run(cabi.linear, x, w, bias, residual=res, activation=act, save_preactivation=True)
        D.check("y", y, want, tol)
        D.check("z", z, z64, ztol)
        again = run(cabi.linear, x, w, bias, residual=res, activation=act)
        assert torch.equal(again, y)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,r,cols", TALL)
def test_long_sums_in_one_gradient(dtype, rows, r, cols):
    """dx alone, whose sums run over the outputs, and dw alone, whose sums run over the rows: both operands' other orders."""
    x, w, _, dy = operands(rows, cols, r, dtype, seed=110)
    want = D.linear_backward64(dy, x, w, None, "none")["dx"]
    dx = run(cabi.linear_backward, dy, x, w, need=(True, False, False))[0]
    D.check("dx", dx, *want)
    assert torch.equal(run(cabi.linear_backward, dy, x, w, need=(True, False, False))[0], dx)
    x, w, _, dy = operands(r, cols, rows, dtype, seed=120)
    want = D.linear_backward64(dy, x, w, None, "none")["dw"]
    dw = run(cabi.linear_backward, dy, x, w, need=(False, True, False))[1]
    D.check("dw", dw, *want)
    assert torch.equal(run(cabi.linear_backward, dy, x, w, need=(False, True, False))[1], dw)


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 36000), (torch.float16, 36001), (torch.float32, 36000)])
def test_sums_over_rows_beyond_31_bits(dtype, n):
    """dw and db of more than 2^31 values of dy, which is 0 but in some rows at the beginning, where the offsets pass 2^31, and at
    the end: the sums are those of these rows, and bounded by them."""
    m, k = 66000, 24
    x, w = operands(m, k, 8, dtype, seed=130)[0], operands(8, k, n, dtype, seed=131)[1]
    at = 2 ** 31 // n
    rows = torch.cat([torch.arange(0, 40), torch.arange(at - 100, at + 100), torch.arange(m - 60, m)]).cuda()
    dy = torch.zeros(m, n, dtype=dtype, device="cuda")
    dy[rows] = torch.randn(len(rows), n, generator=D.gen(132)).to(dtype).cuda()
    z = run(cabi.linear, x, w, save_preactivation=True)[1]
    _, dw, db = run(cabi.linear_backward, dy, x, w, z, activation="silu", need=(False, True, True))
    want = D.linear_backward64(dy[rows], x[rows], w, z[rows], "silu")
    for name, got in (("dw", dw), ("db", db)):
        value, bound = want[name]
        # 300 roundings of dz to bfloat16 are bounded by 2^-8 sqrt(300) = 0.07 of a sum of 300 values of either sign; without any 40
        # of the rows it would be sqrt(40 / 300) = 0.37 off
        assert bound.abs().median() < 0.125 * value.abs().median()
        D.check(name, got, value, bound)
