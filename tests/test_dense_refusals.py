"""Calls of the layer norm and the fused linear layer that are refused before they touch a device (no GPU needed)."""

import pytest

from torch_vulkan_b200 import cabi

X, W, B, Y, MEAN, RSTD = (0x100000000 * i for i in range(1, 7))  # addresses that nothing reads: every call here is refused


@pytest.mark.parametrize("place", [{"mean": W}, {"rstd": W + 64 * 2 - 4}, {"mean": B}, {"rstd": B + 124}, {"mean": W - 12}, {"y": W - 2}, {"y": B},
                                   {"mean": X + 4}, {"rstd": Y + 8}, {"mean": RSTD + 12}])
@pytest.mark.parametrize("param", [cabi.BF16, cabi.F32])
def test_layer_norm_refuses_statistics_over_its_parameters(place, param):
    at = {"y": Y, "mean": MEAN, "rstd": RSTD, **place}
    rc = cabi.lib().tvb_layer_norm(0, X, cabi.BF16, 64, W, B, param, 1e-5, at["y"], at["mean"], at["rstd"], 4, 64, None)
    assert rc == -1 and "overlaps" in cabi.lib().tvb_last_error().decode()


def test_the_extension_does_not_need_a_cuda_build_of_pytorch():
    """The backend has a runtime of its own: none of PyTorch's CUDA libraries is among those that its extension asks for."""
    import subprocess

    from torch_vulkan_b200 import _build

    table = subprocess.run(["readelf", "-d", _build.native_path()], capture_output=True, text=True)
    if table.returncode != 0:
        pytest.skip("no readelf here")
    needed = [line for line in table.stdout.splitlines() if "NEEDED" in line]
    assert any("libtorch_cpu" in line for line in needed) and not any("cuda" in line for line in needed), needed
