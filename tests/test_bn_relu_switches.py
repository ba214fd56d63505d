"""What fuse_bn_relu may change about a model, and what it may not."""
import pytest
import torch
import torch.nn as nn

from rdna4_conv3d.bn_relu import BatchNormReLU3d, fuse_bn_relu


class _PlusFive(nn.ReLU):
    def forward(self, x):
        return super().forward(x) + 5


def _x(c=8):
    return torch.randn(2, c, 3, 4, 5, generator=torch.Generator().manual_seed(1))


def test_an_activation_of_another_class_stays():
    """A subclass may have a forward of its own."""
    act = _PlusFive()
    seq = nn.Sequential(nn.BatchNorm3d(8), act)
    assert fuse_bn_relu(seq) == 0 and type(seq[0]) is nn.BatchNorm3d and seq[1] is act
