"""What fuse_group_norm may change about a model, and what it may not."""
import pytest
import torch
import torch.nn as nn

from rdna4_conv3d.group_norm import GroupNormAct3d, fuse_group_norm


class _PlusFive(nn.ReLU):
    def forward(self, x):
        return super().forward(x) + 5


class _OwnLeaky(nn.LeakyReLU):
    pass


class _OwnSiLU(nn.SiLU):
    pass


class _OwnGELU(nn.GELU):
    pass


def _x(c=8, seed=1):
    return torch.randn(2, c, 3, 4, 5, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("act", [_PlusFive(), _OwnLeaky(0.2), _OwnSiLU(), _OwnGELU()])
def test_activations_of_another_class_stay(act):
    """A subclass may have a forward of its own."""
    seq = nn.Sequential(nn.GroupNorm(2, 8), act)
    want = seq(_x())
    assert fuse_group_norm(seq) == 0 and type(seq[0]) is nn.GroupNorm and seq[1] is act
    assert torch.equal(seq(_x()), want)
