"""Gradients under hooks on saved tensors (offloading, packing) that give the same values back in other strides."""
from contextlib import nullcontext

import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

pytestmark = pytest.mark.gpu

CL = torch.channels_last_3d


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _reversed(t):
    back = tuple(reversed(range(t.dim())))
    return t.clone().permute(back).contiguous().permute(back)


def _padded(t):
    """Inside something wider, off any alignment."""
    if t.dim() == 0:
        return t.clone()
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    wide[..., 1:-2] = t
    return wide[..., 1:-2]


HOOKS = {"cpu": save_on_cpu, "pinned": lambda: save_on_cpu(pin_memory=True),
         "reversed": lambda: saved_tensors_hooks(_reversed, lambda t: t),
         "padded": lambda: saved_tensors_hooks(_padded, lambda t: t)}
hooks = pytest.mark.parametrize("hook", sorted(HOOKS))


def _grads(forward, inputs, hook):
    with hook():
        y = forward()
    up = torch.randn(y.shape, device="cuda", generator=_gen(3)).to(y.dtype)
    return torch.autograd.grad(y, inputs, up)


@hooks
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_cross_entropy(cuda_ready, dtype, hook):
    from rdna4_conv3d import _native
    from rdna4_conv3d.losses import cross_entropy
    z = torch.randn(2, 4, 6, 8, 10, device="cuda", generator=_gen(1)).to(dtype).contiguous(memory_format=CL).requires_grad_(True)
    t = torch.randint(0, 4, (2, 6, 8, 10), device="cuda", generator=_gen(2))
    t[0, 0] = -100
    n0 = _native.launch_count()
    want, = _grads(lambda: cross_entropy(z, t), (z,), nullcontext)
    assert _native.launch_count() > n0
    got, = _grads(lambda: cross_entropy(z, t), (z,), HOOKS[hook])
    assert torch.equal(got, want)


@hooks
@pytest.mark.parametrize("pool", [False, True])
def test_bn_relu(cuda_ready, pool, hook):
    from rdna4_conv3d import _native
    from rdna4_conv3d.bn_relu import BNReLUFn, BNReLUPoolFn
    x = torch.randn(2, 24, 6, 8, 10, device="cuda", generator=_gen(1)).bfloat16().contiguous(memory_format=CL).requires_grad_(True)
    w = (1 + 0.1 * torch.randn(24, device="cuda", generator=_gen(2))).requires_grad_(True)
    b = (0.1 * torch.randn(24, device="cuda", generator=_gen(4))).requires_grad_(True)

    def forward():
        if pool:
            buf, p = BNReLUPoolFn.apply(x, w, b, None, None, 0.1, 1e-5, 24)
            return torch.cat([buf[:, 24:].reshape(-1), p.reshape(-1)])
        return BNReLUFn.apply(x, w, b, None, None, 0.1, 1e-5, True, None)

    n0 = _native.launch_count()
    want = _grads(forward, (x, w, b), nullcontext)
    assert _native.launch_count() > n0
    for a, e in zip(_grads(forward, (x, w, b), HOOKS[hook]), want):
        assert torch.equal(a, e)


@hooks
@pytest.mark.parametrize("transposed", [False, True])
def test_convolutions(cuda_ready, transposed, hook):
    """(These already read what they are given.)"""
    from rdna4_conv3d.conv3d_wmma import Conv3dWmma, ConvTranspose3dWmma
    x = torch.randn(1, 24, 6, 8, 10, device="cuda", generator=_gen(1)).bfloat16().contiguous(memory_format=CL).requires_grad_(True)
    torch.manual_seed(0)
    m = (ConvTranspose3dWmma(24, 16, 2, stride=2) if transposed else Conv3dWmma(24, 32, 3, padding=1)).cuda().bfloat16()
    inputs = (x, *m.parameters())
    want = _grads(lambda: m(x), inputs, nullcontext)
    for a, e in zip(_grads(lambda: m(x), inputs, HOOKS[hook]), want):
        assert torch.equal(a, e)
