"""What the fused linear layer and the layer norm refuse, before they touch a device (no GPU needed)."""

import pytest
import torch

from torch_vulkan_b200 import cabi

A, B, C, E, F, G = (0x100000000 * i for i in range(1, 7))  # addresses that nothing reads: every call here is refused


def refused(rc, *words):
    text = cabi.lib().tvb_last_error().decode()
    assert rc == -1 and all(w in text for w in words), (rc, text)


def linear(x=A, dtype=cabi.BF16, x_sm=64, w=B, w_sn=64, bias=None, act=0, res=None, res_sm=0, y=C, z=None, m=4, n=32, k=64, ws=None, nb=0):
    return cabi.lib().tvb_linear(0, x, dtype, x_sm, w, w_sn, bias, act, res, res_sm, y, z, m, n, k, ws, nb, None)


def backward(dy=A, dtype=cabi.BF16, dy_sm=32, z=None, x=B, x_sm=64, w=C, w_sn=64, act=0, dx=E, dw=F, db=G, m=4, n=32, k=64, ws=None, nb=0):
    return cabi.lib().tvb_linear_backward(0, dy, dtype, dy_sm, z, x, x_sm, w, w_sn, act, dx, dw, db, m, n, k, ws, nb, None)


def test_linear_refusals():
    refused(linear(dtype=cabi.E4M3), "float32, float16 or bfloat16")
    refused(linear(act=5), "unknown activation")
    refused(linear(act=-1), "unknown activation")
    refused(linear(m=-1), "negative size")
    refused(linear(n=1 << 31), "2^31 - 1")
    refused(linear(x_sm=63), "at least k apart")
    refused(linear(w_sn=0), "at least k apart")
    refused(linear(res=E, res_sm=31), "at least n apart")
    refused(linear(x=None), "NULL pointer")
    refused(linear(w=None), "NULL pointer")
    refused(linear(y=None), "NULL pointer")
    refused(linear(y=A + 2), "overlaps")             # over x
    refused(linear(y=B + 32 * 64 * 2 - 2), "overlaps")  # over the end of w
    refused(linear(bias=C + 10), "overlaps")
    refused(linear(res=C + 2, res_sm=32), "overlaps")  # over the residual, but not the residual itself
    refused(linear(res=C, res_sm=40), "overlaps")      # the residual's address with other rows
    refused(linear(z=C), "overlap")
    refused(linear(z=E, res=E, res_sm=32), "overlaps")


def test_linear_backward_refusals():
    refused(backward(dtype=cabi.I8), "float32, float16 or bfloat16")
    refused(backward(act=9), "unknown activation")
    refused(backward(k=-2), "negative size")
    refused(backward(dy_sm=31), "at least n")
    refused(backward(x_sm=60), "at least k apart")
    refused(backward(act=1), "needs the values before it")
    refused(backward(dy=None), "NULL pointer")
    refused(backward(x=None), "NULL pointer")
    refused(backward(w=None), "NULL pointer")
    refused(backward(act=1, z=G + 4096), "workspace")   # dz needs a workspace
    refused(backward(act=1, z=G + 4096, ws=G + 8192 + 1, nb=1 << 20), "workspace")
    refused(backward(dx=A), "overlaps")
    refused(backward(dw=B), "overlaps")
    refused(backward(db=C), "overlaps")
    refused(backward(dx=E, dw=E), "two outputs overlap")


def test_layer_norm_refusals():
    so = cabi.lib()

    def fwd(x=A, dtype=cabi.BF16, x_sm=64, w=B, b=None, pdt=cabi.BF16, eps=1e-5, y=C, mean=E, rstd=F, rows=4, d=64):
        return so.tvb_layer_norm(0, x, dtype, x_sm, w, b, pdt, eps, y, mean, rstd, rows, d, None)

    def bwd(dy=A, dtype=cabi.BF16, dy_sm=64, x=B, x_sm=64, mean=C, rstd=C + 4096, w=None, pdt=cabi.BF16, dx=E, dw=F, db=F + 4096, rows=4, d=64,
            ws=G, nb=1 << 20):
        return so.tvb_layer_norm_backward(0, dy, dtype, dy_sm, x, x_sm, mean, rstd, w, pdt, dx, dw, db, rows, d, ws, nb, None)

    refused(fwd(dtype=cabi.F64), "float32, float16 or bfloat16")
    refused(fwd(pdt=cabi.F16), "x's dtype or float32")
    refused(fwd(rows=-1), "negative size")
    refused(fwd(eps=-1.0), "eps")
    refused(fwd(x_sm=63), "at least d apart")
    refused(fwd(x=None), "NULL pointer")
    refused(fwd(y=None), "NULL pointer")
    refused(fwd(y=A), "overlaps")
    refused(fwd(mean=C), "overlaps")
    refused(fwd(mean=F), "overlaps")
    refused(fwd(rstd=A), "overlaps")
    refused(fwd(b=C + 2), "overlaps")
    refused(bwd(dtype=cabi.I32), "float32, float16 or bfloat16")
    refused(bwd(pdt=cabi.E5M2), "x's dtype or float32")
    refused(bwd(dy_sm=1), "at least d apart")
    refused(bwd(mean=None), "NULL pointer")
    refused(bwd(ws=None), "workspace")
    refused(bwd(nb=16), "workspace")
    refused(bwd(ws=G + 4), "workspace")
    refused(bwd(dx=A), "overlaps")
    refused(bwd(dw=E), "two outputs overlap")
    refused(bwd(ws=A), "overlaps")


def test_wrappers_refuse_what_they_cannot_pass_on():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    for bad in (lambda: cabi.linear(x, w.t()), lambda: cabi.linear(x, w.half()), lambda: cabi.linear(x[0], w),
                lambda: cabi.linear(x, w, torch.zeros(5)), lambda: cabi.linear(x, w, residual=torch.zeros(4, 5)),
                lambda: cabi.linear(x, w, activation="swish"), lambda: cabi.linear(x.t().contiguous().t(), w),
                lambda: cabi.linear(x[:1].expand(4, 8), w), lambda: cabi.linear_backward(torch.zeros(4, 6), x, w, activation="gelu"),
                lambda: cabi.linear_backward(torch.zeros(4, 5), x, w), lambda: cabi.layer_norm(x, torch.ones(7)),
                lambda: cabi.layer_norm(x, torch.ones(8, dtype=torch.float64)), lambda: cabi.layer_norm(x, torch.ones(8), torch.ones(8).half()),
                lambda: cabi.layer_norm(torch.zeros(2, 3, 4)),
                lambda: cabi.layer_norm_backward(x, x, torch.zeros(3), torch.zeros(4)),
                lambda: cabi.layer_norm_backward(x, x, torch.zeros(4).double(), torch.zeros(4))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cabi.linear(x.double(), w.double()), lambda: cabi.layer_norm(x.to(torch.int32))):
        with pytest.raises(TypeError):
            bad()


@pytest.mark.parametrize("sizes,blocks,pairs", [(((2048, 4096), (14336, 4096)), (224, 32), 74), (((0, 0), (2048, 14336)), (0, 64), 74),
                                                (((300, 600), (5000, 1100)), (100, 7), 74), (((1000, 1000), (1000, 1024)), (16, 16), 74),
                                                (((513, 257), (511, 255)), (3, 2), 2), (((9000, 900), (700, 9000)), (9, 9), 74),
                                                (((0, 0), (257, 300)), (0, 5), 74), (((2049, 2049), (8200, 2100)), (33, 32), 74)])
def test_the_schedule_of_two_products_covers_every_output_once(sizes, blocks, pairs):
    """The same formulas as PairSchedule and pair_run (csrc/kernels/linear_pair.cu): tiles of 512 rows x 256 columns, the last
    ones cut; every 256 x 128 piece of both outputs belongs to one pair."""
    def up(a, b):
        return -(-a // b)

    tj, ti = [up(j, 512) for j, _ in sizes], [up(i, 256) for _, i in sizes]
    tiles = [a * b for a, b in zip(tj, ti)]
    a, b = blocks
    extra = light_first = light = 0
    if tiles[0] % pairs:
        light = pairs - tiles[0] % pairs
        extra = (2 * a + b) // (2 * b)
        light_first = extra * b < a
    early = min(light * extra, tiles[1])
    rest = (tiles[1] - early) % pairs
    half, quarter = up(2 * rest, pairs) * 32, up(4 * rest, pairs) * 24
    cut, whole = 256, tiles[1]
    if rest and min(half, quarter) < 48:
        whole -= rest
        cut = 256 if half <= quarter else 128
    pairs = min(pairs, tiles[0] + whole + (tiles[1] - whole) * (512 // cut))

    def place(product, index):
        band, r = divmod(index, 8 * ti[product])
        rows = min(8, tj[product] - band * 8)
        row, col = (band * 8 + r % rows) * 512, r // rows * 256
        return row, col, 256, 2 if row + 256 < sizes[product][0] else 1

    heavy = tiles[0] % pairs
    light = pairs - heavy if heavy else 0
    early = light * extra
    seen = set()
    for pair in range(pairs):
        is_light = heavy != 0 and pair >= heavy
        rank = pair - heavy if is_light else pair
        order = (rank if is_light else pairs - heavy + pair) if heavy and light_first else pair
        mine = [(0, *place(0, t)) for t in range(pair, tiles[0], pairs)]
        if is_light:
            mine += [(1, *place(1, t)) for t in range(rank, min(early, whole), light)]
        mine += [(1, *place(1, t)) for t in range(early + order, whole, pairs)]
        per_half = 256 // cut
        for at in range(order, (tiles[1] - whole) * 2 * per_half, pairs):
            row, col, _, _ = place(1, whole + at // (2 * per_half))
            sub = at % (2 * per_half)
            row, col = row + sub // per_half * 256, col + sub % per_half * cut
            if row < sizes[1][0] and col < sizes[1][1]:
                mine.append((1, row, col, cut, 1))
        for product, row, col, cols, halves in mine:
            for r in range(row, row + 256 * halves, 256):
                for c in range(col, col + cols, 128):
                    assert (product, r, c) not in seen
                    seen.add((product, r, c))
    for product, (j, i) in enumerate(sizes):
        for r in range(0, j, 256):
            for c in range(0, i, 128):
                assert (product, r, c) in seen, (product, r, c)
