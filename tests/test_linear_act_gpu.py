"""The fused linear layer (tvb_linear, tvb_linear_backward) against plain 64-bit forms: types, activations, sizes from one row
and one value to several tiles, ragged sizes, strides and alignments, empty sizes, in-place residuals, repeated results."""

import pytest
import torch

import _dense as D
from torch_vulkan_b200 import cabi

pytestmark = pytest.mark.gpu

# (m, k, n): one value; odd everything; edges of the tiles in every direction; few rows; tall and wide
SIZES = [(1, 1, 1), (1, 8, 3), (3, 5, 7), (1, 64, 128), (2, 200, 129), (16, 128, 256), (17, 64, 130), (33, 72, 264), (64, 512, 128),
         (77, 1003, 517), (130, 328, 72), (200, 512, 300), (256, 64, 256), (257, 136, 520), (700, 96, 640), (5, 4104, 24)]


# outputs large enough for the kernel of CTA pairs: whole tiles, ragged edges in both directions, widths of tile below 256
LARGE = [(2048, 128, 2048), (1900, 200, 2600), (1024, 1032, 5000), (2001, 77, 1999), (4096, 64, 1024), (300, 520, 14336)]


def cuda(*shape, seed, dtype, scale=1.0):
    return (torch.randn(*shape, generator=D.gen(seed)) * scale).to(dtype).cuda()


def operands(m, k, n, dtype, seed=0):
    return (cuda(m, k, seed=seed + 1, dtype=dtype), cuda(n, k, seed=seed + 2, dtype=dtype, scale=max(k, 1) ** -0.5),
            cuda(n, seed=seed + 3, dtype=dtype, scale=0.3), cuda(m, n, seed=seed + 4, dtype=dtype))


def run(fn, *args, **kw):
    torch.cuda.synchronize()
    got = fn(*args, **kw)
    cabi.synchronize()
    return got


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_forward_sizes(dtype, m, k, n):
    x, w, b, r = operands(m, k, n, dtype)
    want, tol, z, ztol = D.linear64(x, w, b, r, "silu")
    y, pre = run(cabi.linear, x, w, b, residual=r, activation="silu", save_preactivation=True)
    D.check("y", y, want, tol)
    D.check("z", pre, z, ztol)
    want, tol, _, _ = D.linear64(x, w, None, None, "none")
    D.check("product", run(cabi.linear, x, w), want, tol)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", LARGE)
def test_large_outputs(dtype, m, k, n):
    x, w, b, r = operands(m, k, n, dtype, seed=15)
    for act, bias, res in (("gelu_tanh", b, r), ("none", None, None)):
        want, tol, z, ztol = D.linear64(x, w, bias, res, act)
        y, pre = run(cabi.linear, x, w, bias, residual=res, activation=act, save_preactivation=True)
        D.check("y", y, want, tol)
        D.check("z", pre, z, ztol)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [(2048, 2048, 2048), (1900, 2600, 2000), (2048, 4096, 1024), (4100, 1800, 1900), (2001, 1999, 2003)])
def test_large_gradients(dtype, m, k, n):
    """Both products of the backward pass in one launch, and each alone."""
    x, w, b, dy = operands(m, k, n, dtype, seed=16)
    z = (x.double() @ w.double().t() + b.double()).to(dtype)
    want = D.linear_backward64(dy, x, w, z, "silu")
    for need in ((True, True, True), (True, False, False), (False, True, False)):
        got = run(cabi.linear_backward, dy, x, w, z, activation="silu", need=need)
        for name, g, asked in zip(("dx", "dw", "db"), got, need):
            if asked:
                D.check((need, name), g, *want[name])


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("act", D.ACTS)
@pytest.mark.parametrize("m", [4, 150, 600])
def test_forward_activations(dtype, act, m):
    k, n = 192, 272
    x, w, b, r = operands(m, k, n, dtype, seed=10)
    x = x * 4  # (values far into the activations' tails)
    for bias, res in ((None, None), (b, None), (None, r), (b, r)):
        want, tol, z, ztol = D.linear64(x, w, bias, res, act)
        y, pre = run(cabi.linear, x, w, bias, residual=res, activation=act, save_preactivation=True)
        D.check("y", y, want, tol)
        D.check("z", pre, z, ztol)


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("m", [3, 100, 300])
def test_forward_strides_and_alignment(dtype, m):
    """Slices of wider matrices: rows further apart than they are long, beginning anywhere, aligned or not."""
    k, n = 136, 200
    for off, pad in ((0, 8), (8, 24), (1, 3), (3, 13)):
        x, w, r = (cuda(rows, cols + pad + off, seed=21 + rows, dtype=dtype, scale=0.3)[:, off:off + cols]
                   for rows, cols in ((m, k), (n, k), (m, n)))
        b = cuda(n + 1, seed=22, dtype=dtype)[1:]
        want, tol, _, _ = D.linear64(x, w, b, r, "gelu")
        D.check((off, pad), run(cabi.linear, x, w, b, residual=r, activation="gelu"), want, tol)


@pytest.mark.parametrize("dtype", D.DTYPES)
def test_forward_empty_sizes(dtype):
    for m, k, n in ((0, 8, 8), (4, 8, 0), (4, 0, 24), (300, 0, 300), (0, 0, 0)):
        x, w, b, r = operands(m, k, n, dtype)
        want, tol, z, ztol = D.linear64(x, w, b, r, "gelu")
        y, pre = run(cabi.linear, x, w, b, residual=r, activation="gelu", save_preactivation=True)
        D.check("y", y, want, tol)
        D.check("z", pre, z, ztol)


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("m", [2, 40, 700])
def test_forward_written_over_the_residual(dtype, m):
    k, n = 128, 392
    x, w, b, r = operands(m, k, n, dtype, seed=30)
    want, tol, _, _ = D.linear64(x, w, b, r, "relu")
    code = cabi._dtype_code(dtype)
    torch.cuda.synchronize()
    cabi.check(cabi.lib().tvb_linear(0, x.data_ptr(), code, k, w.data_ptr(), k, b.data_ptr(), cabi.ACTIVATIONS["relu"], r.data_ptr(), n,
                                     r.data_ptr(), None, m, n, k, None, 0, None))
    cabi.synchronize()
    D.check("y", r, want, tol)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [3, 300])
def test_forward_infinities_and_nans_stay_in_their_rows_and_columns(dtype, m):
    k, n = 200, 264
    x, w, b, r = operands(m, k, n, dtype, seed=40)
    clean = run(cabi.linear, x, w, b, residual=r, activation="silu")
    x[1, 5] = float("nan")
    w[7, 3] = float("inf")
    got = run(cabi.linear, x, w, b, residual=r, activation="silu")
    assert torch.isnan(got[1]).all()
    rest = [i for i in range(m) if i != 1]
    assert not torch.isfinite(got[rest, 7]).any() or (got[rest, 7] == r[rest, 7]).any()  # silu(-inf) is nan, silu(inf) inf
    cols = [j for j in range(n) if j != 7]
    assert torch.equal(got[rest][:, cols], clean[rest][:, cols])


def test_large_values_saturate_to_infinity_in_float16():
    x = torch.full((2, 64), 200.0, dtype=torch.float16, device="cuda")
    w = torch.full((8, 64), 200.0, dtype=torch.float16, device="cuda")
    got = run(cabi.linear, x, w)  # 64 * 40000 is beyond float16: the float32 sum is finite, its rounding is not
    assert torch.isinf(got).all() and (got > 0).all()


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_backward_sizes(dtype, m, k, n):
    x, w, b, dy = operands(m, k, n, dtype, seed=50)
    z = (x.double() @ w.double().t() + b.double()).to(dtype)
    for act in ("gelu", "none"):
        want = D.linear_backward64(dy, x, w, z, act)
        got = run(cabi.linear_backward, dy, x, w, z if act != "none" else None, activation=act)
        for name, g in zip(("dx", "dw", "db"), got):
            D.check((act, name), g, *want[name])


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("act", D.ACTS)
@pytest.mark.parametrize("m", [4, 150, 600])
def test_backward_activations(dtype, act, m):
    k, n = 200, 272
    x, w, b, dy = operands(m, k, n, dtype, seed=60)
    z = (x.double() @ w.double().t() * 4).to(dtype)
    z[:, ::9] = 0
    want = D.linear_backward64(dy, x, w, z, act)
    for need in ((True, True, True), (True, False, False), (False, True, False), (False, False, True), (True, False, True)):
        got = run(cabi.linear_backward, dy, x, w, z, activation=act, need=need)
        for name, g, asked in zip(("dx", "dw", "db"), got, need):
            assert (g is not None) == asked
            if asked:
                D.check((need, name), g, *want[name])


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("m", [3, 100, 300])
def test_backward_strides_and_alignment(dtype, m):
    k, n = 136, 200
    for off, pad in ((0, 8), (8, 24), (1, 3), (3, 13)):
        x, w, dy = (cuda(rows, cols + pad + off, seed=71 + rows, dtype=dtype, scale=0.3)[:, off:off + cols]
                    for rows, cols in ((m, k), (n, k), (m, n)))
        z = cuda(m, n, seed=72, dtype=dtype)
        for act in ("none", "silu"):
            want = D.linear_backward64(dy, x, w, z, act)
            got = run(cabi.linear_backward, dy, x, w, z, activation=act)
            for name, g in zip(("dx", "dw", "db"), got):
                D.check((off, pad, act, name), g, *want[name])


@pytest.mark.parametrize("dtype", D.DTYPES)
def test_backward_empty_sizes(dtype):
    for m, k, n in ((0, 8, 16), (4, 8, 0), (4, 0, 24), (0, 0, 0)):
        x, w, b, dy = operands(m, k, n, dtype)
        z = torch.zeros_like(dy)
        got = run(cabi.linear_backward, dy, x, w, z, activation="gelu")
        want = D.linear_backward64(dy, x, w, z, "gelu")
        for name, g in zip(("dx", "dw", "db"), got):
            D.check((m, k, n, name), g, *want[name])


@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("m,k,n", [(2, 4096, 256), (300, 640, 512), (2000, 72, 136)])
def test_results_repeat_bit_for_bit(dtype, m, k, n):
    x, w, b, dy = operands(m, k, n, dtype, seed=80)
    z = (x.double() @ w.double().t()).to(dtype)
    first = [run(cabi.linear, x, w, b, activation="gelu")] + list(run(cabi.linear_backward, dy, x, w, z, activation="gelu"))
    for _ in range(3):
        again = [run(cabi.linear, x, w, b, activation="gelu")] + list(run(cabi.linear_backward, dy, x, w, z, activation="gelu"))
        assert all(torch.equal(a, c) for a, c in zip(first, again))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [(200, 8192, 2048), (100, 4096, 1000), (40, 6000, 520), (4, 8000, 1024), (500, 1024, 2048), (1000, 1024, 1000),
                                   (24, 512, 2048), (130, 4104, 264)])
def test_products_cut_along_their_sums(dtype, m, k, n):
    """Clusters of two to eight CTAs per tile, ragged last parts, both gradients in one launch and alone."""
    x, w, b, dy = operands(m, k, n, dtype, seed=33)
    want, tol, z64, ztol = D.linear64(x, w, b, dy, "relu")
    y, z = run(cabi.linear, x, w, b, residual=dy, activation="relu", save_preactivation=True)
    D.check("y", y, want, tol)
    D.check("z", z, z64, ztol)
    want = D.linear_backward64(dy, x, w, z, "relu")
    for need in ((True, True, True), (True, False, False), (False, True, True)):
        for name, g, asked in zip(("dx", "dw", "db"), run(cabi.linear_backward, dy, x, w, z, activation="relu", need=need), need):
            if asked:
                D.check((need, name), g, *want[name])


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 36000), (torch.float16, 36001), (torch.float32, 36000)])
def test_offsets_beyond_31_bits(dtype, n):
    """Outputs and gradients of more than 2^31 values, checked where the offsets pass 2^31 and at the end."""
    m, k = 66000, 24
    x, w, b, _ = operands(m, k, n, dtype, seed=30)[:3] + (None,)
    r = torch.randn(m, n, device="cuda", dtype=dtype)
    y, z = run(cabi.linear, x, w, b, residual=r, activation="silu", save_preactivation=True)
    at = 2 ** 31 // n
    for rows in (slice(0, 100), slice(at - 100, at + 300), slice(m - 100, m)):
        want, tol, z64, ztol = D.linear64(x[rows], w, b, r[rows], "silu")
        D.check(("y", rows), y[rows], want, tol)
        D.check(("z", rows), z[rows], z64, ztol)
    dx, dw, db = run(cabi.linear_backward, r, x, w, z, activation="silu")
    for rows in (slice(0, 100), slice(at - 100, at + 300), slice(m - 100, m)):
        D.check(("dx", rows), dx[rows], *D.linear_backward64(r[rows], x[rows], w, z[rows], "silu")["dx"])
    cols = slice(n - 70, n)
    want = D.linear_backward64(r[:, cols], x, w[cols], z[:, cols], "silu")
    D.check("dw", dw[cols], *want["dw"])
    D.check("db", db[cols], *want["db"])


def test_more_rows_than_a_grids_second_dimension():
    x, w, b, _ = operands(4_300_000, 4, 9, torch.float32, seed=31)
    want, tol, _, _ = D.linear64(x, w, b, None, "relu")
    D.check("y", run(cabi.linear, x, w, b, activation="relu"), want, tol)


@pytest.mark.parametrize("m,k,n", [(1, 1000, 4099), (1, 4096, 256), (3, 4095, 1024), (8, 700, 512), (9, 512, 512), (32, 4096, 128), (33, 2000, 300),
                                   (500, 4096, 64), (64, 64, 4096)])
def test_float32_shapes(m, k, n):
    """Tiles of 8, 32 and 64 rows, r cut in one to eight parts, operands on and off 16 bytes."""
    x, w, b, dy = operands(m, k, n, torch.float32, seed=32)
    want, tol, z64, ztol = D.linear64(x, w, b, dy, "gelu")
    y, z = run(cabi.linear, x, w, b, residual=dy, activation="gelu", save_preactivation=True)
    D.check("y", y, want, tol)
    D.check("z", z, z64, ztol)
    want = D.linear_backward64(dy, x, w, z, "gelu")
    for name, g in zip(("dx", "dw", "db"), run(cabi.linear_backward, dy, x, w, z, activation="gelu")):
        D.check(name, g, *want[name])


def test_gradients_against_differences():
    """d/dt L(x + t v) for L = sum(dy * y), by central differences of the 64-bit form, against the returned gradients in
    float32: the formula is the derivative of the forward pass, in every operand."""
    m, k, n = 6, 20, 12
    for act in D.ACTS:
        x, w, b, dy = operands(m, k, n, torch.float32, seed=90)
        z = run(cabi.linear, x, w, b, activation=act, save_preactivation=True)[1]
        got = run(cabi.linear_backward, dy, x, w, z, activation=act)
        for at, (t, g) in enumerate(zip((x, w, b), got)):
            v = torch.randn(t.shape, generator=D.gen(91), dtype=torch.float64).cuda()
            h = 1e-6

            def loss(s):
                ops = [x.double(), w.double(), b.double()]
                ops[at] = ops[at] + s * v
                return float((dy.double() * D.act64(ops[0] @ ops[1].t() + ops[2], act)).sum())

            diff = (loss(h) - loss(-h)) / (2 * h)
            # differences: h^2 of the third derivative and 2^-52 |L| / h; the gradient: its float32 roundings
            size = float((g.double().abs() * v.abs()).sum())
            assert abs(diff - float((g.double() * v).sum())) <= 1e-4 * size + 1e-7 * abs(loss(0)), (act, at)
