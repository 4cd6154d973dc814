"""Recorded steps and the memory pool: a block that a recording may touch is nobody else's for as long as it can be replayed."""

import gc

import pytest
import torch

import torch_vulkan_b200 as tv
from torch_vulkan_b200 import linear as L
from torch_vulkan_b200 import shard


def occupy(shape, count=8):
    """Tensors that take whatever blocks of this size the pool has to give."""
    return [torch.full(shape, 7.0).to("vk") for _ in range(count)]


@pytest.mark.gpu
@pytest.mark.parametrize("first_to_go", ["maker", "user"])
def test_a_block_of_one_recording_given_back_during_another(first_to_go):
    """Recording A makes a tensor, recording B reads it and drops it: A and B both hold its memory, whichever goes first."""
    shape = (256, 384)
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1))
    w = torch.eye(384)
    vx, vw = x.to("vk"), w.to("vk")
    maker = shard.StepGraph(lambda: [L.linear_act(vx, vw, None, "relu")])
    hold = [maker.replay()[0]]
    maker.outputs = None
    tv.synchronize()

    def use():
        y = L.linear_act(hold.pop(), vw, residual=vx)
        return [y]

    user = shard.StepGraph(use, warm=False)
    want = x.clamp_min(0) + x
    if first_to_go == "maker":
        del maker
        gc.collect()
        others = occupy(shape)
        assert torch.equal(user.replay()[0].cpu(), want)
    else:
        del user
        gc.collect()
        others = occupy(shape)
        maker.replay()
    tv.synchronize()
    assert all((t.cpu() == 7).all() for t in others)
    # with both gone the memory is the pool's again
    reserved = tv.memory_stats()["reserved_bytes"]
    maker = user = None
    gc.collect()
    again = torch.empty(shape, device="vk")
    assert tv.memory_stats()["reserved_bytes"] == reserved
    del again


class FakeLibrary:
    """The calls of a recording, without a device."""

    def __init__(self, end_rc=0):
        self.calls, self.end_rc = [], end_rc

    def tvb_synchronize(self, device):
        return 0

    def tvb_graph_begin(self, device):
        self.calls.append("begin")
        return 0

    def tvb_graph_end(self, device, out):
        self.calls.append("end")
        if self.end_rc == 0:
            out._obj.value = 1234
        return self.end_rc

    def tvb_graph_destroy(self, graph):
        self.calls.append(("destroy", graph.value))

    def tvb_last_error(self):
        return b"the capture was lost"


@pytest.mark.parametrize("end_rc,calls", [(0, ["begin", "end", ("destroy", 1234)]), (-1, ["begin", "end"])])
def test_a_step_that_raises_leaves_no_recording(monkeypatch, end_rc, calls):
    from torch_vulkan_b200 import cabi

    fake = FakeLibrary(end_rc)
    monkeypatch.setattr(cabi, "lib", lambda: fake)

    def step():
        raise KeyError("in the step")

    with pytest.raises(KeyError, match="in the step"):
        shard.StepGraph(step, warm=False)
    gc.collect()
    assert fake.calls == calls


def test_a_recording_that_cannot_end_is_an_error(monkeypatch):
    from torch_vulkan_b200 import cabi

    fake = FakeLibrary(-1)
    monkeypatch.setattr(cabi, "lib", lambda: fake)
    with pytest.raises(RuntimeError):
        shard.StepGraph(lambda: [], warm=False)
    assert fake.calls == ["begin", "end"]


@pytest.mark.gpu
def test_a_failed_step_gives_its_memory_back():
    tv.synchronize()
    made = []

    def step():
        made.append(torch.empty(333, 4096, device="vk"))  # a size that nothing else here has
        made.clear()
        raise KeyError("in the step")

    with pytest.raises(KeyError):
        shard.StepGraph(step, warm=False)
    reserved = tv.memory_stats()["reserved_bytes"]
    again = torch.empty(333, 4096, device="vk")
    assert tv.memory_stats()["reserved_bytes"] == reserved
    # the stream runs again
    x = torch.arange(8.0)
    assert torch.equal((x.to("vk") + x.to("vk")).cpu(), x + x)
    del again
