"""Tensors without dimensions are refused by the block operators with a ValueError, without a GPU."""
import pytest
import torch

from dig_amd import ops, train


def test_no_dimensions():
    class OnDevice(torch.Tensor):
        def get_device(self):
            return 0

    f = lambda *shape: torch.zeros(shape).as_subclass(OnDevice)  # noqa: E731
    with pytest.raises(ValueError, match="must be \\[B"):
        ops.group_norm_act(f(), f(16), f(16), groups=4)
    with pytest.raises(ValueError, match="mean_rstd must be"):
        train.group_norm_act_bwd(f(), f(2, 4, 2), f(16), f(16), f())
    with pytest.raises(ValueError, match="do not fit"):
        ops.linear_act(f(), f(8, 16))
    with pytest.raises(ValueError, match="do not fit"):
        train.linear_act_bwd(f(), f(8, 16), f())
