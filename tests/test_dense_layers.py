"""The unquantised layers around the quantised ones, as a model has them: linear_act / LinearAct / fuse_linears and nn.LayerNorm on
the CPU (host logic), and on device "vk" with their gradients, together in a pre-norm feed-forward block, recorded and
replayed, on CUDA tensors and streams."""

import threading

import pytest
import torch
import torch.nn.functional as F
from torch import nn

import _dense as D
import torch_vulkan_b200 as tv
from torch_vulkan_b200 import cabi
from torch_vulkan_b200 import linear as L


def same_model(d=64, h=160, seed=0):
    torch.manual_seed(seed)
    return nn.Sequential(nn.LayerNorm(d), nn.Linear(d, h), nn.GELU(approximate="tanh"), nn.Linear(h, d), nn.Linear(d, h, bias=False), nn.SiLU(),
                         nn.Sequential(nn.Linear(h, d), nn.ReLU()), nn.Linear(d, d), nn.Tanh())


def test_fuse_linears_keeps_the_function_and_the_parameters():
    a, b = same_model(), same_model()
    names = L.fuse_linears(b)
    assert names == ["1", "4", "6.0"]
    assert [type(m) for m in b] == [nn.LayerNorm, L.LinearAct, nn.Identity, nn.Linear, L.LinearAct, nn.Identity, nn.Sequential, nn.Linear, nn.Tanh]
    assert list(a.state_dict()) == list(b.state_dict())
    x = torch.randn(3, 5, 64, generator=D.gen(1))
    assert torch.equal(a(x), b(x))
    a(x).square().sum().backward()
    b(x).square().sum().backward()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p.grad, q.grad)
    # quantising afterwards leaves the layers that carry an activation
    assert L.swap_linears(b) == ["3", "7"] and isinstance(b[1], L.LinearAct)


def test_fuse_linears_with_shared_modules_hooks_and_own_forward_passes():
    torch.manual_seed(3)
    relu, lin = nn.ReLU(), nn.Linear(16, 16)

    class Twice(nn.Sequential):
        def forward(self, x):
            return super().forward(x) + self[0](x)

    hooked = nn.Linear(16, 16)
    hooked.register_forward_hook(lambda module, args, out: out + 1)
    model = nn.Sequential(lin, relu, nn.Linear(16, 16), relu, nn.GELU(), lin, nn.Tanh(), lin, nn.SiLU(), hooked, nn.ReLU(),
                          Twice(nn.Linear(16, 16), nn.ReLU()))
    x = torch.randn(4, 16, generator=D.gen(2))
    want = model(x)
    assert L.fuse_linears(model) == ["0", "2", "7"]
    assert torch.equal(model(x), want)


def test_linear_act_on_the_cpu_and_what_it_refuses():
    lin = nn.Linear(8, 6)
    x, r = torch.randn(2, 3, 8), torch.randn(2, 3, 6)
    assert torch.equal(L.linear_act(x, lin.weight, lin.bias, "silu", r), F.silu(lin(x)) + r)
    assert torch.equal(L.LinearAct.from_float(lin, "gelu")(x), F.gelu(lin(x)))
    for bad in (lambda: L.linear_act(x, lin.weight, activation="tanh"), lambda: L.linear_act(x[..., :7], lin.weight),
                lambda: L.linear_act(x, lin.weight, residual=r[0]), lambda: L.LinearAct(4, 4, activation="swish")):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------- on the GPU

gpu = pytest.mark.gpu


def vk_leaf(t):
    return t.to("vk").requires_grad_(True)


@gpu
@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("act", D.ACTS)
def test_linear_act_gradients_on_vk(dtype, act):
    x = torch.randn(4, 25, 72, generator=D.gen(1)).to(dtype)
    w = (torch.randn(136, 72, generator=D.gen(2)) / 8).to(dtype)
    b = torch.randn(136, generator=D.gen(3)).to(dtype)
    r = torch.randn(4, 25, 136, generator=D.gen(4)).to(dtype)
    dy = torch.randn(4, 25, 136, generator=D.gen(5)).to(dtype)
    vx, vw, vb, vr = map(vk_leaf, (x, w, b, r))
    y = L.linear_act(vx, vw, vb, act, vr)
    want, tol, z64, _ = D.linear64(x.reshape(100, 72), w, b, r.reshape(100, 136), act)
    D.check("y", y.detach().cpu().reshape(100, 136), want, tol)
    y.backward(dy.to("vk"))
    z = cabi.linear(vx.detach().view(100, 72), vw.detach(), vb.detach(), activation=act, save_preactivation=True)[1].cpu()
    want = D.linear_backward64(dy.reshape(100, 136), x.reshape(100, 72), w, z, act)
    D.check("dx", vx.grad.cpu().reshape(100, 72), *want["dx"])
    D.check("dw", vw.grad.cpu(), *want["dw"])
    D.check("db", vb.grad.cpu(), *want["db"])
    assert torch.equal(vr.grad.cpu(), dy)


@gpu
def test_expanded_inputs_and_gradients():
    """Rows that are one row in memory (an expanded input, the gradient of a sum) are copied, not misread. (The gradient of the
    expanded input itself is a sum that autograd asks of the device, which has no kernel for it.)"""
    w = torch.randn(24, 40, generator=D.gen(2)) / 6
    x = torch.randn(1, 40, generator=D.gen(1))
    cx, cw = x.double(), w.double().requires_grad_(True)
    F.silu(cx.expand(7, 40) @ cw.t()).sum().backward()
    vw = vk_leaf(w)
    L.linear_act(x.to("vk").expand(7, 40), vw, None, "silu").backward(torch.ones(1, 1).to("vk").expand(7, 24))
    # seven products of a float32 sum's size; silu' and its product with 1 are 2^-18 off at most
    assert ((vw.grad.cpu().double() - cw.grad).abs() <= 2.0 ** -17 * 7 * x.double().abs().max() * 1.1).all()


@gpu
@pytest.mark.parametrize("dtype", D.DTYPES)
@pytest.mark.parametrize("shape,normalized", [((5, 64), (64,)), ((2, 3, 40, 768), (768,)), ((7, 6, 10), (6, 10)), ((33,), (33,)), ((4, 0, 16), (16,))])
def test_aten_layer_norm(dtype, shape, normalized):
    x = (torch.randn(shape, generator=D.gen(1)) * 2 + 1).to(dtype)
    d = 1
    for s in normalized:
        d *= s
    ln = nn.LayerNorm(normalized, dtype=dtype)
    with torch.no_grad():
        ln.weight.copy_(1 + 0.3 * torch.randn(normalized, generator=D.gen(2)))
        ln.bias.copy_(torch.randn(normalized, generator=D.gen(3)))
    want = D.layer_norm64(x.reshape(-1, d), ln.weight.detach().reshape(-1), ln.bias.detach().reshape(-1), 1e-5)
    g, b = ln.weight.detach().reshape(-1), ln.bias.detach().reshape(-1)
    vln = nn.LayerNorm(normalized, dtype=dtype)
    vln.load_state_dict(ln.state_dict())
    vln = vln.to("vk")
    vx = vk_leaf(x)
    y = vln(vx)
    assert y.shape == x.shape and y.dtype == dtype
    D.check("y", y.detach().cpu().reshape(-1, d), *want["y"])
    dy = torch.randn(shape, generator=D.gen(4)).to(dtype)
    y.backward(dy.to("vk"))
    _, mean, rstd = torch.native_layer_norm(vx.detach(), normalized, vln.weight.detach(), vln.bias.detach(), 1e-5)
    assert mean.shape == rstd.shape == torch.Size(list(shape[:len(shape) - len(normalized)]) + [1] * len(normalized))
    grads = D.layer_norm_backward64(dy.reshape(-1, d), x.reshape(-1, d), mean.cpu().reshape(-1), rstd.cpu().reshape(-1), g)
    D.check("dx", vx.grad.cpu().reshape(-1, d), *grads["dx"])
    D.check("dg", vln.weight.grad.cpu().reshape(-1), *grads["dg"])
    D.check("db", vln.bias.grad.cpu().reshape(-1), *grads["db"])
    assert not b.requires_grad
    # without parameters, and of a transposed (not contiguous) input
    if len(shape) == 2:
        xt = x.t().contiguous().to("vk").t()
        assert torch.equal(F.layer_norm(xt, normalized).cpu(), F.layer_norm(vx.detach(), normalized).cpu())


@gpu
def test_aten_layer_norm_errors():
    x = torch.randn(4, 8).to("vk")
    with pytest.raises(RuntimeError, match="normalized_shape"):
        F.layer_norm(x, (7,))
    with pytest.raises(NotImplementedError):
        torch.native_layer_norm(x, (8,), torch.ones(8), None, 1e-5)
    with pytest.raises(TypeError):
        F.layer_norm(torch.zeros(4, 8, dtype=torch.int32).to("vk"), (8,))
    with pytest.raises(ValueError):
        L.linear_act(x, torch.zeros(3, 8))
    with pytest.raises(TypeError):
        L.linear_act(x.to(torch.float64), torch.zeros(3, 8, dtype=torch.float64).to("vk"))


class Block(nn.Module):
    """x + down(act(up(norm(x)))), the residual added in the last product's epilogue."""

    def __init__(self, d, h, activation):
        super().__init__()
        self.norm = nn.LayerNorm(d)
        self.up = L.LinearAct(d, h, activation=activation)
        self.down = L.LinearAct(h, d)

    def forward(self, x):
        return self.down(self.up(self.norm(x)), residual=x)


def block_and_twin(dtype, d, h, activation, seed=0):
    torch.manual_seed(seed)
    block = Block(d, h, activation).to(dtype)
    twin = Block(d, h, activation)
    twin.load_state_dict(block.state_dict())
    return block.to("vk"), twin.double()


@gpu
@pytest.mark.parametrize("dtype,rel", [(torch.float32, 2.0 ** -18), (torch.float16, 2.0 ** -8), (torch.bfloat16, 2.0 ** -5)])
@pytest.mark.parametrize("rows", [1, 37, 700])
def test_feed_forward_block_forward_and_backward(dtype, rel, rows):
    """Two blocks in a row against the same model in 64 bits. Each of the eight tensors between input and output (and back) is
    rounded once to the type, half a step relative: in the 2-norm the result and the gradients are off by at most some ten
    times that (float32: the sums' own roundings)."""
    d, h = 96, 392
    pairs = [block_and_twin(dtype, d, h, "gelu", 1), block_and_twin(dtype, d, h, "silu", 2)]
    x = torch.randn(rows, d, generator=D.gen(7)).to(dtype)
    dy = torch.randn(rows, d, generator=D.gen(8)).to(dtype)
    vx, cx = vk_leaf(x), x.double().requires_grad_(True)
    vy, cy = vx, cx
    for vb, cb in pairs:
        vy, cy = vb(vy), cb(cy)
    vy.backward(dy.to("vk"))
    cy.backward(dy.double())

    def near(name, got, want):
        off = float((got.cpu().double() - want).norm() / want.norm())
        assert off <= rel, (name, off)

    near("y", vy.detach(), cy.detach())
    near("dx", vx.grad, cx.grad)
    for vb, cb in pairs:
        for (name, p), q in zip(vb.named_parameters(), cb.parameters()):
            near(name, p.grad, q.grad)
    # a second backward pass adds to the gradients
    before = [p.grad.cpu() for vb, _ in pairs for p in vb.parameters()]
    for vb, _ in pairs:
        vx = vb(vx)
    vx.backward(dy.to("vk"))
    for p, old in zip([p for vb, _ in pairs for p in vb.parameters()], before):
        assert torch.equal(p.grad.cpu(), old + old)


@gpu
@pytest.mark.parametrize("shape,n", [((3, 0), 8), ((2, 0, 16), 8), ((2, 5, 16), 0), ((16,), 8), ((1, 1, 16), 8)])
def test_linear_act_odd_shapes(shape, n):
    x = torch.randn(shape, generator=D.gen(1)).to(torch.bfloat16)
    w = torch.randn(n, shape[-1], generator=D.gen(2)).to(torch.bfloat16)
    b = torch.randn(n, generator=D.gen(3)).to(torch.bfloat16)
    vx, vw, vb = vk_leaf(x), vk_leaf(w), vk_leaf(b)
    y = L.linear_act(vx, vw, vb, "silu")
    assert y.shape == (*shape[:-1], n)
    want = F.silu(F.linear(x.double(), w.double(), b.double()))
    assert ((y.detach().cpu().double() - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -9).all()
    y.backward(torch.ones(y.shape, dtype=torch.bfloat16).to("vk"))
    assert vx.grad.shape == x.shape and vw.grad.shape == w.shape and vb.grad.shape == b.shape


@gpu
def test_nothing_is_kept_where_no_gradient_is_asked_for(monkeypatch):
    kept = []
    plain = cabi.linear
    monkeypatch.setattr(cabi, "linear", lambda *a, **kw: kept.append(kw["save_preactivation"]) or plain(*a, **kw))
    layer = L.LinearAct(64, 32, activation="gelu").to(torch.bfloat16).to("vk")
    x = torch.randn(4, 64, generator=D.gen(1)).to(torch.bfloat16).to("vk")
    y = layer(x)
    with torch.no_grad():
        assert torch.equal(layer(x).cpu(), y.detach().cpu())
    assert kept == [True, False]


@gpu
def test_a_quantised_model_with_its_norms_runs_on_the_device():
    torch.manual_seed(3)
    model = nn.Sequential(nn.LayerNorm(256), nn.Linear(256, 512), nn.SiLU(), nn.Linear(512, 256)).to(torch.bfloat16).requires_grad_(False)
    L.fuse_linears(model)
    twin = nn.Sequential(nn.LayerNorm(256), nn.Linear(256, 512), nn.SiLU(), nn.Linear(512, 256)).requires_grad_(False)
    twin.load_state_dict(model.state_dict())
    L.swap_linears(model, kind="int8")
    model = model.to("vk")
    x = torch.randn(5, 256, generator=D.gen(1)).to(torch.bfloat16)
    want = twin(x.float())
    got = model(x.to("vk")).cpu().float()
    assert (got - want).norm() <= 0.02 * want.norm()  # int8 weights: half a step of 1 / 127 of a row's largest


@gpu
def test_recorded_steps_keep_their_temporaries():
    """A recorded forward and backward pass, replayed while other tensors come and go: the recording's temporaries (z, dz, the
    workspaces) are nobody else's memory, and two recordings share nothing."""
    from torch_vulkan_b200.shard import StepGraph

    d, h, rows = 128, 512, 160
    block, _ = block_and_twin(torch.bfloat16, d, h, "gelu", 5)
    xs = [torch.randn(rows, d, generator=D.gen(20 + i)).to(torch.bfloat16) for i in range(4)]
    dy = torch.randn(rows, d, generator=D.gen(30)).to(torch.bfloat16).to("vk")

    def eager(x):
        leaf = vk_leaf(x)
        y = block(leaf)
        return [t.cpu() for t in (y.detach(), *torch.autograd.grad(y, [leaf, *block.parameters()], dy))]

    want = [eager(x) for x in xs]
    graphs = []
    for _ in range(2):
        x_in = xs[0].to("vk").requires_grad_(True)

        def step(x_in=x_in):
            y = block(x_in)
            return [y.detach(), *torch.autograd.grad(y, [x_in, *block.parameters()], dy)]

        live = block(x_in)  # (an eager graph of the same leaves is alive meanwhile)
        graphs.append((x_in, StepGraph(step)))
        del live
    hold = []
    for turn, x in enumerate(xs):
        hold.append([torch.full((rows, h), float(turn), dtype=torch.bfloat16).to("vk") for _ in range(6)])
        for x_in, graph in graphs:
            with torch.no_grad():
                x_in.copy_(x.to("vk"))
        outs = [graph.replay() for _, graph in graphs]
        tv.synchronize()
        for out in outs:
            for a, b in zip(out, want[turn]):
                assert torch.equal(a.cpu(), b)
        for kept, tensors in enumerate(hold):
            assert all((t.cpu() == float(kept)).all() for t in tensors)
    reserved = tv.memory_stats()["reserved_bytes"]
    del graphs, outs, graph, x_in
    import gc

    gc.collect()
    again = [torch.empty(rows, h, dtype=torch.bfloat16, device="vk") for _ in range(4)]  # the recordings' memory is used again
    assert tv.memory_stats()["reserved_bytes"] == reserved
    del again


@gpu
def test_cuda_tensors_run_on_torchs_stream_and_in_its_graphs():
    x = torch.randn(64, 256, generator=D.gen(1)).to(torch.bfloat16).cuda()
    w = (torch.randn(384, 256, generator=D.gen(2)) / 16).to(torch.bfloat16).cuda()
    dy = torch.randn(64, 384, generator=D.gen(3)).to(torch.bfloat16).cuda()
    torch.cuda.synchronize()
    y, z = cabi.linear(x, w, activation="silu", save_preactivation=True)
    want = [y, *cabi.linear_backward(dy, x, w, z, activation="silu"), cabi.layer_norm(x)[0]]
    torch.cuda.synchronize()

    def step(x):
        y, z = cabi.linear(x, w, activation="silu", save_preactivation=True)
        return [y, *cabi.linear_backward(dy, x, w, z, activation="silu"), cabi.layer_norm(x)[0]]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # queued behind work of the same stream, with no synchronisation in between
        late = torch.zeros_like(x)
        for _ in range(20):
            late.copy_(late + 1)
        late.copy_(x)
        got = step(late)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    buf = torch.zeros_like(x)
    with torch.cuda.stream(side):
        step(buf)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        outs = step(buf)
    buf.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@gpu
def test_two_streams_and_two_graphs_at_once():
    """Calls on two streams share nothing: the same bits as one after the other, queued directly and as graphs."""
    def case(seed):
        x, w, dy = (torch.randn(*shape, generator=D.gen(seed + i)).to(torch.bfloat16).cuda()
                    for i, shape in enumerate([(300, 1100), (1300, 1100), (300, 1300)]))
        return x[:, :1003], w[:, :1003], dy

    def step(x, w, dy):
        y, z = cabi.linear(x, w, activation="gelu", save_preactivation=True)
        h, mean, rstd = cabi.layer_norm(y)
        return [y, h, *cabi.linear_backward(dy, x, w, z, activation="gelu"), *cabi.layer_norm_backward(dy, y, mean, rstd)]

    cases = [case(1), case(50)]
    torch.cuda.synchronize()
    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(outs, want[i]))
    graphs, outs = [], []
    for c in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*c))
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(outs[i], want[i]))


@gpu
def test_two_threads_at_once():
    x = torch.randn(200, 512, generator=D.gen(1)).to(torch.float16)
    w = (torch.randn(640, 512, generator=D.gen(2)) / 20).to(torch.float16)
    vx, vw = x.to("vk"), w.to("vk")
    want = cabi.linear(vx, vw, activation="gelu").cpu()
    wrong = []

    def work():
        for _ in range(50):
            if not torch.equal(cabi.linear(vx, vw, activation="gelu").cpu(), want):
                wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


FIRST_CALLS = """
import torch
import torch_vulkan_b200
from torch_vulkan_b200 import cabi
x, w = torch.randn(40, 256, device="cuda").bfloat16(), torch.randn(512, 256, device="cuda").bfloat16()
long = torch.randn(3, 12000, device="cuda").bfloat16()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, z = cabi.linear(x, w, activation="gelu", save_preactivation=True)
    grads = cabi.linear_backward(y, x, w, z, activation="gelu")
    norm = cabi.layer_norm(long)
graph.replay()
torch.cuda.synchronize()
y2, z2 = cabi.linear(x, w, activation="gelu", save_preactivation=True)
again = [y2, z2, *cabi.linear_backward(y2, x, w, z2, activation="gelu"), *cabi.layer_norm(long)]
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip([y, z, *grads, *norm], again))
print("the same")
"""


@gpu
def test_the_first_calls_of_a_process_may_be_captured():
    import subprocess
    import sys

    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stderr[-2000:]
