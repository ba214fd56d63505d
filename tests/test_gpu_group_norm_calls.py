"""Calls of group_norm_act whose plan must not be another call's."""
import pytest
import torch

from rdna4_conv3d.group_norm import group_norm_act

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [False, True])
def test_numbers_held_in_tensors_are_read_at_each_call(cuda_ready, grad):
    """Plans are kept by their numbers, not by an object that may change."""
    x = torch.randn(2, 8, 4, 4, 4, device="cuda").contiguous(memory_format=torch.channels_last_3d).requires_grad_(grad)
    eps, slope = torch.tensor(1e-5), torch.tensor(0.25)
    for e, s in ((1e-5, 0.25), (3.0, 0.25), (3.0, 0.75)):
        eps.fill_(e)
        slope.fill_(s)
        y = group_norm_act(x, 2, eps=eps, activation="leaky_relu", negative_slope=slope)
        want = group_norm_act(x, 2, eps=float(eps), activation="leaky_relu", negative_slope=s)
        assert torch.equal(y, want)
