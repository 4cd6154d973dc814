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
