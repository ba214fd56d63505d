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


def test_parameters_are_the_models_own():
    """Frozen ones stay frozen, an optimizer's stay its own, tied ones stay tied."""
    seq = nn.Sequential(nn.GroupNorm(2, 8), nn.ReLU(), nn.GroupNorm(2, 8), nn.SiLU())
    seq[2].weight = seq[0].weight
    seq[0].requires_grad_(False)
    before = dict(seq.named_parameters(remove_duplicate=False))
    assert fuse_group_norm(seq) == 2
    after = dict(seq.named_parameters(remove_duplicate=False))
    assert list(after) == list(before) and all(after[k] is before[k] for k in before)
    assert not seq[0].weight.requires_grad and not seq[2].weight.requires_grad and seq[2].bias.requires_grad


def test_a_norm_used_twice_stays_one():
    norm = nn.GroupNorm(2, 8)
    seq = nn.Sequential(norm, nn.ReLU(), nn.Sequential(norm, nn.SiLU()), norm)
    want = seq(_x())
    assert fuse_group_norm(seq) == 2
    torch.testing.assert_close(seq(_x()), want, rtol=1e-4, atol=1e-4)
    assert len(list(seq.parameters())) == 2 and seq[0].weight is seq[2][0].weight is norm.weight


def test_without_parameters_and_without_a_bias():
    plain, biased = nn.GroupNorm(2, 8, affine=False), nn.GroupNorm(2, 8)
    biased.bias = None
    nn.init.normal_(biased.weight)
    seq = nn.Sequential(plain, nn.ReLU(), biased, nn.LeakyReLU(0.1))
    want = seq(_x())
    keys = list(seq.state_dict())
    assert fuse_group_norm(seq) == 2 and list(seq.state_dict()) == keys
    torch.testing.assert_close(seq(_x()), want, rtol=1e-4, atol=1e-4)


HOOKS = {"forward": lambda m, seen: m.register_forward_hook(lambda *a: seen.append(1)),
         "forward_pre": lambda m, seen: m.register_forward_pre_hook(lambda *a: seen.append(1)),
         "backward": lambda m, seen: m.register_full_backward_hook(lambda *a: seen.append(1)),
         "backward_pre": lambda m, seen: m.register_full_backward_pre_hook(lambda *a: seen.append(1))}


@pytest.mark.parametrize("kind", sorted(HOOKS))
@pytest.mark.parametrize("which", [0, 1])
def test_modules_with_hooks_stay(kind, which):
    """A hook sees the norm's output before the activation, which a fused pair does not have."""
    seq = nn.Sequential(nn.GroupNorm(2, 8), nn.SiLU(), nn.GroupNorm(2, 8), nn.SiLU())
    seen = []
    HOOKS[kind](seq[which], seen)
    assert fuse_group_norm(seq) == 1 and type(seq[0]) is nn.GroupNorm and isinstance(seq[2], GroupNormAct3d)
    seq(_x().requires_grad_(True)).sum().backward()
    assert seen == [1]
