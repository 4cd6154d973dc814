"""Layer norm, forward and backward (tvb_layer_norm, tvb_layer_norm_backward), against plain 64-bit forms: types of values and
parameters, rows from one value to longer than the registers hold, ragged lengths, strides, offsets, constant rows."""

import pytest
import torch

import _dense as D
from torch_vulkan_b200 import cabi

pytestmark = pytest.mark.gpu

SIZES = [(1, 1), (3, 2), (5, 7), (1, 64), (33, 128), (1000, 16), (7, 255), (129, 256), (2, 512), (65, 520), (300, 1003), (40, 1024),
         (17, 2048), (9, 2056), (2000, 768), (5, 4096), (6, 4097), (4, 8192), (3, 8200), (2, 16384), (3, 16392), (2, 32768), (2, 33000),
         (1300, 1032), (700, 2048), (2500, 1032), (3000, 4096), (400, 8192), (333, 8200), (500, 4104),
         (1301, 500), (2001, 384), (303, 5120), (200, 6001), (1500, 8704), (1400, 12296), (1000, 16376)]


def run(fn, *args, **kw):
    torch.cuda.synchronize()
    got = fn(*args, **kw)
    cabi.synchronize()
    return got


def values(rows, d, dtype, seed=0, ld=None, off=0):
    x = torch.randn(rows, (ld or d) + off, generator=D.gen(seed)) * (0.5 + torch.rand(rows, 1, generator=D.gen(seed + 1)))
    x = x + torch.randn(rows, 1, generator=D.gen(seed + 2))
    return x.to(dtype).cuda()[:, off:off + d]


def params(d, dtype, seed=5):
    return ((1 + 0.3 * torch.randn(d, generator=D.gen(seed))).to(dtype).cuda(), (0.3 * torch.randn(d, generator=D.gen(seed + 1))).to(dtype).cuda())


def check_all(x, g, b, dy, eps=1e-5):
    want = D.layer_norm64(x, g, b, eps)
    y, mean, rstd = run(cabi.layer_norm, x, g, b, eps)
    for name, got in (("y", y), ("mean", mean), ("rstd", rstd)):
        D.check(name, got, *want[name])
    grads = D.layer_norm_backward64(dy, x, mean, rstd, g)
    for name, got in zip(("dx", "dg", "db"), run(cabi.layer_norm_backward, dy, x, mean, rstd, g)):
        D.check(name, got, *grads[name])


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("rows,d", SIZES)
def test_sizes(dtype, rows, d):
    g, b = params(d, dtype)
    check_all(values(rows, d, dtype), g, b, values(rows, d, dtype, seed=7))


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("d", [24, 768, 5000, 12000, 20000])
def test_parameters_of_either_type_or_none(dtype, d):
    x, dy = values(37, d, dtype), values(37, d, dtype, seed=7)
    g, b = params(d, torch.float32)
    for weight, bias in ((g, b), (None, None), (g, None), (None, b)):
        check_all(x, weight, bias, dy)


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("d", [64, 1000, 4096, 17000])
def test_strides_and_alignment(dtype, d):
    g, b = params(d + 1, dtype)
    for ld, off in ((d + 8, 0), (d + 16, 8), (d + 3, 1)):
        check_all(values(11, d, dtype, ld=ld, off=off), g[1:], b[1:], values(11, d, dtype, seed=9, ld=ld, off=off))


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("d", [1, 8, 300, 4096])
def test_constant_rows_and_far_means(dtype, d):
    """A row of one value has no variance: y is the bias, rstd 1 / sqrt(eps). A mean far above the spread keeps its digits."""
    x = torch.full((3, d), 3.25, dtype=dtype, device="cuda")
    x[1] = 0
    g, b = params(d, dtype)
    y, mean, rstd = run(cabi.layer_norm, x, g, b, 1e-5)
    assert torch.equal(y, b.expand(3, d)) and torch.equal(mean.cpu(), torch.tensor([3.25, 0.0, 3.25]))
    assert ((rstd.double() - 1e-5 ** -0.5).abs() <= 1e-5 ** -0.5 * 2.0 ** -21).all()
    if d > 1 and dtype == torch.float32:
        far = (1000 + torch.randn(5, d, generator=D.gen(3))).cuda()
        check_all(far, g, b, values(5, d, dtype, seed=4))


def test_infinities_and_nans_stay_in_their_rows():
    x = values(9, 1000, torch.bfloat16)
    g, b = params(1000, torch.bfloat16)
    clean = run(cabi.layer_norm, x, g, b)[0]
    x[2, 5], x[6, 7] = float("nan"), float("inf")
    y = run(cabi.layer_norm, x, g, b)[0]
    rest = [0, 1, 3, 4, 5, 7, 8]
    assert torch.isnan(y[[2, 6]]).all() and torch.equal(y[rest], clean[rest])


@pytest.mark.parametrize("rows,d", [(0, 8), (0, 20000), (3, 0), (0, 0)])
def test_empty_sizes(rows, d):
    x = torch.zeros(rows, d, device="cuda")
    g, b = torch.ones(d, device="cuda"), torch.zeros(d, device="cuda")
    y, mean, rstd = run(cabi.layer_norm, x, g, b)
    assert y.shape == (rows, d) and mean.shape == rstd.shape == (rows,)
    dx, dg, db = run(cabi.layer_norm_backward, x, x.clone(), mean, rstd, g)
    assert dx.shape == (rows, d) and torch.equal(dg, torch.zeros(d, device="cuda")) and torch.equal(db, torch.zeros(d, device="cuda"))


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("d", [40, 1000, 17000])
def test_backward_parts_and_repeats(dtype, d):
    """Any subset of the gradients; the same bits every time."""
    rows = 700
    x, dy = values(rows, d, dtype), values(rows, d, dtype, seed=7)
    g, b = params(d, dtype)
    _, mean, rstd = run(cabi.layer_norm, x, g, b)
    full = run(cabi.layer_norm_backward, dy, x, mean, rstd, g)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, True, True)):
        got = run(cabi.layer_norm_backward, dy, x, mean, rstd, g, need=need)
        for a, f, asked in zip(got, full, need):
            assert (a is not None) == asked and (a is None or torch.equal(a, f))


@pytest.mark.parametrize("d", [4096, 1000, 16384])
def test_offsets_beyond_31_bits(d):
    rows = 2 ** 31 // d + 300
    x, dy = (torch.randn(rows, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    g, b = params(d, torch.bfloat16)
    y, mean, rstd = run(cabi.layer_norm, x, g, b)
    dx, dg, db = run(cabi.layer_norm_backward, dy, x, mean, rstd, g)
    for part in (slice(0, 50), slice(rows - 400, rows)):
        want = D.layer_norm64(x[part], g, b, 1e-5)
        for name, got in (("y", y), ("mean", mean), ("rstd", rstd)):
            D.check((name, part), got[part], *want[name])
        D.check(("dx", part), dx[part], *D.layer_norm_backward64(dy[part], x[part], mean[part], rstd[part], g)["dx"])
    cols = slice(d - 16, d)  # (the sums over the rows, of some columns)
    dy64, h = dy[:, cols].double(), (x[:, cols].double() - mean.double()[:, None]) * rstd.double()[:, None]
    slack = D.sum_slack(rows) * (1 + dy64.abs() * (1 + h.abs())).sum(0)
    D.check("dg", dg[cols], (dy64 * h).sum(0), D.rounded((dy64 * h).sum(0), slack, torch.bfloat16))
    D.check("db", db[cols], dy64.sum(0), D.rounded(dy64.sum(0), slack, torch.bfloat16))


def test_gradients_against_differences():
    rows, d, eps = 5, 24, 1e-5
    x, dy = values(rows, d, torch.float32), values(rows, d, torch.float32, seed=7)
    g, b = params(d, torch.float32)
    _, mean, rstd = run(cabi.layer_norm, x, g, b, eps)
    got = run(cabi.layer_norm_backward, dy, x, mean, rstd, g)
    for at, (t, grad) in enumerate(zip((x, g, b), got)):
        v = torch.randn(t.shape, generator=D.gen(11), dtype=torch.float64).cuda()
        h = 1e-6

        def loss(s):
            ops = [x.double(), g.double(), b.double()]
            ops[at] = ops[at] + s * v
            return float((dy.double() * D.layer_norm64(ops[0], ops[1], ops[2], eps)["y"][0]).sum())

        diff = (loss(h) - loss(-h)) / (2 * h)
        size = float((grad.double().abs() * v.abs()).sum())
        assert abs(diff - float((grad.double() * v).sum())) <= 1e-4 * size + 1e-7 * abs(loss(0)), at
