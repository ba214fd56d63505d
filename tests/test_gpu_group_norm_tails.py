"""The activations' far sides, each value against 64 bits relative to itself (a weight of 0 makes z the bias exactly)."""
import math

import pytest
import torch

from gn_refs import half_step
from rdna4_conv3d.group_norm import group_norm_act

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _tails(dtype, act, low):
    """(y, act'(z), z) on a grid of z from low to 9."""
    z = torch.linspace(low, 9.0, 2000, device="cuda")
    c = z.numel()
    x = torch.randn(2, c, 8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    x = x.movedim(1, -1).contiguous().movedim(-1, 1)
    w = torch.zeros(c, device="cuda")
    z.requires_grad_(True)
    y = group_norm_act(x, c // 8, w, z, activation=act)
    dy = torch.zeros_like(y)
    dy[0, :, 0] = 1.0
    return y.detach()[0, :, 0], torch.autograd.grad(y, z, dy)[0].double(), z.detach().double()


@pytest.mark.parametrize("dtype,low", [(BF, -13.0), (HF, -7.0), (FP, -13.0)])
def test_gelu_far_sides(cuda_ready, dtype, low):
    """gelu(z) = z Phi(z), relative to itself down to where the type ends.

    e^(-z^2/2): its argument is off by at most 3 u of z^2/2 (square, product, constant), so the exponential by 1.5 u z^2,
    and by 8 u of its own; 16 u for the few products and sums. 16-bit results: e^(u^2) erfc(u) by an approximation good
    to 2^-16 of itself. fp32 results: CUDA's erfc is good to 4 units in the last place, its argument z / sqrt(2) to 2 u,
    which moves erfc(v) by at most (2 v^2 + 2) 2 u of itself."""
    y, grad, z = _tails(dtype, "gelu", low)
    phi = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    dens = torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    rel = U * (24 + 4 * z * z) + (2.0 ** -16 if dtype != FP else 0.0)
    want = z * phi
    tiny = 2.0 ** -126 * 16                              # (an exponential below the normal numbers is 0)
    d = (y.double() - want).abs()
    bound = half_step(want, dtype) + rel * want.abs() + tiny
    assert bool((d <= bound).all()), ((d - bound).max().item(), z[(d - bound).argmax()].item())
    want = phi + z * dens
    d = (grad - want).abs()
    bound = rel * (phi + (z * dens).abs()) + tiny
    assert bool((d <= bound).all()), ((d - bound).max().item(), z[(d - bound).argmax()].item())


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_silu_far_sides(cuda_ready, dtype):
    """silu(z) = z / (1 + e^-z): the exponential's argument is off by 2 u of |z|, itself and the reciprocal by 8 u."""
    y, grad, z = _tails(dtype, "silu", -60.0)
    s = 1.0 / (1.0 + torch.exp(-z))
    rel = U * (32 + 4 * z.abs())
    d = (y.double() - z * s).abs()
    assert bool((d <= half_step(z * s, dtype) + rel * (z * s).abs()).all())
    d = (grad - s * (1 + z * (1 - s))).abs()
    assert bool((d <= rel * s * (1 + (z * (1 - s)).abs())).all())


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_infinite_activations(cuda_ready, dtype, act):
    """z of an infinite bias: as in torch's own, f(inf) = inf, and NaN stays NaN."""
    z = torch.tensor([float("inf"), float("nan"), 1.0, -1.0] * 2, device="cuda")
    x = torch.randn(2, 4, 8, device="cuda").to(dtype).movedim(-1, 1)
    y = group_norm_act(x, 1, torch.zeros(8, device="cuda"), z, activation=act).float()
    want = {"gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[act](z)
    assert bool((y[:, 0] == float("inf")).all()) and bool(y[:, 1].isnan().all())
    torch.testing.assert_close(y[:, 2:4], want[2:4].reshape(1, 2, 1).expand(2, 2, 4), rtol=2.0 ** -7, atol=0)
