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


def test_parameters_and_statistics_are_the_models_own():
    """Frozen ones stay frozen, an optimizer's stay its own, a norm used twice keeps one set of statistics."""
    norm = nn.BatchNorm3d(8)
    seq = nn.Sequential(nn.BatchNorm3d(8), nn.ReLU(), norm, nn.ReLU(), norm, nn.BatchNorm3d(8, affine=False), nn.ReLU(),
                        nn.BatchNorm3d(8, track_running_stats=False), nn.ReLU())
    seq[0].requires_grad_(False)
    params, buffers = (dict(f(remove_duplicate=False)) for f in (seq.named_parameters, seq.named_buffers))
    twin = nn.Sequential(*[m for m in seq])
    assert fuse_bn_relu(seq) == 4 and isinstance(seq[0], BatchNormReLU3d)
    for was, now in ((params, seq.named_parameters), (buffers, seq.named_buffers)):
        now = dict(now(remove_duplicate=False))
        assert list(now) == list(was) and all(now[k] is was[k] for k in was)
    assert not seq[0].weight.requires_grad and seq[2].weight is seq[4].weight
    seq(_x())
    assert int(seq[2].num_batches_tracked) == 2 and int(twin[2].num_batches_tracked) == 2


@pytest.mark.parametrize("which", [0, 1])
def test_modules_with_hooks_stay(which):
    """A hook sees the norm's output before the activation, which a fused pair does not have."""
    seq = nn.Sequential(nn.BatchNorm3d(8), nn.ReLU(), nn.BatchNorm3d(8), nn.ReLU())
    seen = []
    seq[which].register_forward_hook(lambda *a: seen.append(1))
    assert fuse_bn_relu(seq) == 1 and type(seq[0]) is nn.BatchNorm3d and isinstance(seq[2], BatchNormReLU3d)
    seq(_x())
    assert seen == [1]
