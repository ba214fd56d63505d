"""group_norm_act on the CPU where |mean| is far above the spread (u: half a step of fp32)."""
import pytest
import torch

from rdna4_conv3d.group_norm import group_norm_act

U = 2.0 ** -24


@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("value,step", [(30000.0, 0.0), (30000.0, 0.25), (0.1, 0.0), (-1e6, 0.0)])
@pytest.mark.parametrize("shape,groups", [((2, 24, 9, 20, 21), 1), ((2, 24, 9, 20, 21), 3), ((1, 6, 3, 5, 7), 3)])
def test_one_value_far_from_zero(shape, groups, value, step, fmt):
    """y against 64 bits: the mean's rounding moves x - mean by u |mean|, x - mean itself is exact; 16 u for the rest."""
    x = torch.full(shape, value)
    x[0, 0, 1, 2, 3] += step
    x.requires_grad_(True)
    dy = torch.randn(shape, generator=torch.Generator().manual_seed(4))
    y = group_norm_act(x, groups, checkpoint=fmt)
    dx, = torch.autograd.grad(y, x, dy)
    n = shape[0]
    xd, g = (t.detach().double().reshape(n, groups, -1) for t in (x, dy))
    mean = xd.mean(-1, keepdim=True)
    rstd = (((xd - mean) ** 2).mean(-1, keepdim=True) + 1e-5) ** -0.5
    xh = (xd - mean) * rstd
    assert bool(((y.detach().double().reshape(xh.shape) - xh).abs() <= U * (abs(value) * rstd + 16 * xh.abs())).all())
    if step == 0.0 and fmt is None:
        # xh is 0; the mean of dy: torch adds in blocks, 64 u of the magnitudes is far above what those are off by
        want = rstd * (g - g.mean(-1, keepdim=True))
        bound = rstd * U * (16 * g.abs() + 64 * g.abs().mean(-1, keepdim=True))
        # and the mean's rounding, where the value is no mean of fp32 sums: xh = u |value| rstd instead of 0
        e = U * abs(value) * rstd
        bound = bound + rstd * 2 * e * (e * g.abs().mean(-1, keepdim=True))
        assert bool(((dx.double().reshape(want.shape) - want).abs() <= bound).all())


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("shape", [(2, 24, 3, 4, 5), (2, 24, 7), (2, 24)])
def test_an_in_place_activation_may_follow(shape, fmt):
    """As on a CUDA device: the result is no view of something inside."""
    x = torch.randn(shape, generator=torch.Generator().manual_seed(5)).requires_grad_(True)
    y = group_norm_act(x, 3, checkpoint=fmt)
    want = torch.relu(y)
    gx, = torch.autograd.grad((want ** 2).sum(), x)
    y = torch.relu_(group_norm_act(x, 3, checkpoint=fmt))
    assert torch.equal(y, want) and y.movedim(1, -1).is_contiguous()
    assert torch.equal(torch.autograd.grad((y ** 2).sum(), x)[0], gx)
