"""Group normalisation with an activation, channels last.

``group_norm_act(x, groups, weight, bias, activation=...)`` is
act(F.group_norm(x, ...)) for (N, C, ...) activations whose channels lie
innermost, as every convolution of this package writes them: two native
passes forward and two backward (r4c_gn_*; one launch each way for small
activations), where stock PyTorch copies them to channels first, normalises,
copies back and applies the activation on its own. bf16, fp16 or fp32 in and
out, fp32 arithmetic on x - mean; a thread's sums in fp32, all others in fp64
and in a fixed order (same bits on every run).

``checkpoint='int8'`` or ``'e4m3'`` keeps x for the backward pass in 8 bits
(``checkpoint8``): the forward writes them beside y, the backward kernels read
them as they are. y does not change; the gradients are those at the values
that the 8 bits hold, with the mean and variance of x itself.

``GroupNormAct3d`` is an ``nn.GroupNorm`` (same parameters and state_dict) on
these kernels, ``fuse_group_norm(model)`` swaps every (GroupNorm, activation)
pair of a model's ``nn.Sequential``s for (GroupNormAct3d, Identity). CPU
tensors take the same formulas in torch operations. No reference counterpart:
the reference's blocks normalise over the batch (benches/unet_e2e.py:13-20).
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn

from . import _native
from .bn_relu import has_hooks
from .checkpoint8 import _pack_torch, _unpack_torch, check_format
from .logprobs import refuse_blind, refuse_twice

_FLOATS = frozenset((torch.bfloat16, torch.float16, torch.float32))
ACTIVATIONS = tuple(_native.ACTIVATIONS)


def _channels_last(t: torch.Tensor) -> torch.Tensor:
    """t with its channels innermost, dense and on 16 bytes (differentiable)."""
    if t.dim() == 5:
        if not t.is_contiguous(memory_format=torch.channels_last_3d):
            t = t.contiguous(memory_format=torch.channels_last_3d)
    else:
        last = t.movedim(1, -1)
        if not last.is_contiguous():
            t = last.contiguous().movedim(-1, 1)
    if t.data_ptr() & 15:
        t = t.clone()
    return t


def _params(weight: Optional[torch.Tensor], bias: Optional[torch.Tensor]):
    """(weight, bias, their type) as the kernels read them."""
    if weight is not None and bias is not None and weight.dtype is bias.dtype and weight.dtype in _FLOATS:
        if weight.is_contiguous() and bias.is_contiguous():
            return weight, bias, weight.dtype
        dtype = weight.dtype
    else:
        given = weight if bias is None else bias if weight is None else None
        dtype = torch.float32 if given is None or given.dtype not in _FLOATS else given.dtype
    return tuple(None if t is None else t.detach().to(dtype).contiguous() for t in (weight, bias)) + (dtype,)


def _as_saved(t: torch.Tensor, count: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A saved vector (hooks may give back another one with the same values), dense and on 16 bytes."""
    if t.shape != (count,) or t.dtype is not dtype or t.device != device:
        _native._not_as_saved(t, (count,), dtype, device)
    if t.data_ptr() & 15 or not t.is_contiguous():
        t = t.clone(memory_format=torch.contiguous_format)
    return t


class GroupNormActFn(torch.autograd.Function):
    """``args``: (groups, eps, activation, slope, format or None)."""

    @staticmethod
    def forward(ctx, x, weight, bias, args):
        groups, eps, activation, slope, fmt = args
        w, b, pdtype = _params(weight, bias)
        key = x.shape, groups, x.dtype, pdtype, eps, activation, slope
        plan = _native.gn_plan(*key)
        y, stats, q8 = _native.gn_forward(x, plan, w, b, fmt)
        ctx.save_for_backward(x if fmt is None else q8, stats, weight, bias)
        ctx.key, ctx.plan, ctx.fmt, ctx.device = key, plan, fmt, x.device
        return y

    @staticmethod
    def backward(ctx, gy):
        refuse_twice()
        x, stats, weight, bias = ctx.saved_tensors
        key, plan, fmt, device = ctx.key, ctx.plan, ctx.fmt, ctx.device
        shape, dtype = key[0], key[2]
        if fmt is None:
            if x.shape != shape or x.dtype is not dtype or x.device != device:
                _native._not_as_saved(x, shape, dtype, device)
            x = _channels_last(x)
        else:
            x = _as_saved(x, plan.q8_bytes, torch.uint8, device)
        stats = _as_saved(stats, plan.kept, torch.float32, device)
        w, b, pdtype = _params(weight, bias)
        if w is not None and (w.shape != (shape[1],) or w.device != device):
            _native._not_as_saved(w, (shape[1],), pdtype, device)
        if b is not None and (b.shape != (shape[1],) or b.device != device):
            _native._not_as_saved(b, (shape[1],), pdtype, device)
        if pdtype is not key[3]:
            plan = _native.gn_plan(*key[:3], pdtype, *key[4:])
        if gy.dtype is not dtype:
            gy = gy.to(dtype)
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dx, dw, db = _native.gn_backward(_channels_last(gy), plan, x, fmt, stats, w, b, need_x, need_w or need_b)
        if not need_w:
            dw = None
        elif weight.dtype is not torch.float32:
            dw = dw.to(weight.dtype)
        if not need_b:
            db = None
        elif bias.dtype is not torch.float32:
            db = db.to(bias.dtype)
        return dx, dw, db, None


def _check(x, num_groups, weight, bias, eps, activation, negative_slope, checkpoint) -> None:
    shape = x.shape
    if len(shape) < 2:
        raise ValueError(f"x must be (N, C, ...), got shape {tuple(shape)}")
    c = shape[1]
    if num_groups < 1 or c < 1 or c % num_groups:
        raise ValueError(f"{c} channels do not part into {num_groups} equal groups")
    if x.dtype not in _FLOATS and (x.is_cuda or checkpoint is not None or not x.is_floating_point()):
        raise TypeError(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != (c,):
            raise ValueError(f"{name} must have shape ({c},), got {tuple(t.shape)}")
        if not t.is_floating_point():
            raise TypeError(f"{name} must be a floating type, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"eps must be finite and at least 0, got {eps}")
    if activation not in _native.ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(map(repr, ACTIVATIONS))}, got {activation!r}")
    if not math.isfinite(negative_slope):
        raise ValueError(f"negative_slope must be finite, got {negative_slope}")
    if checkpoint is not None:
        check_format(checkpoint, "checkpoint")


def group_norm_act(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5, *, activation: str = "none",
                   negative_slope: float = 0.01, checkpoint: Optional[str] = None) -> torch.Tensor:
    """act(group_norm(x) * weight + bias), channels last, in x's type.

    x: (N, C, ...). Channels-last activations are read as they lie, others are copied to channels last first; the
        result is channels last either way.
    weight, bias: (C,) or None, of any floating type; their gradients are summed in fp32 or wider.
    activation: 'none', 'relu', 'leaky_relu' (``negative_slope``), 'silu' or 'gelu' (with the normal distribution
        function). relu and leaky_relu take the negative side's slope at 0.
    checkpoint: None, 'int8' or 'e4m3': how x is kept for the backward pass (see ``checkpoint8.pack8``).

    A group that holds a NaN or an infinity is NaN throughout, its gradient too; other groups are not touched. On a
    CUDA device gradients are reverse mode, once; on the CPU as torch has them (with a checkpoint: once). The type
    does not follow autocast: the arithmetic is fp32 whatever x is.
    """
    _check(x, num_groups, weight, bias, eps, activation, negative_slope, checkpoint)
    if not x.is_cuda:
        return _group_norm_torch(x, num_groups, weight, bias, eps, activation, negative_slope, checkpoint)
    for t in (x, weight, bias):
        if t is not None:
            refuse_blind(t)
    code = _native.ACTIVATIONS[activation]
    eps, negative_slope = float(eps), float(negative_slope)      # (plans are kept by them)
    x = _channels_last(x)
    needs = x.requires_grad or weight is not None and weight.requires_grad or bias is not None and bias.requires_grad
    if torch.is_grad_enabled() and needs or torch._C._is_tracing():
        fmt = None if checkpoint is None else _native.Q8_FORMATS[checkpoint]
        return GroupNormActFn.apply(x, weight, bias, (num_groups, eps, code, negative_slope, fmt))
    w, b, pdtype = _params(weight, bias)
    return _native.gn_forward(x, _native.gn_plan(x.shape, num_groups, x.dtype, pdtype, eps, code, negative_slope), w, b,
                              None)[0]


def _act_torch(z, activation, slope):
    if activation == "relu":
        return torch.where(z <= 0, 0.0, z)
    if activation == "leaky_relu":
        return torch.where(z <= 0, z * slope, z)
    if activation == "silu":
        return torch.nn.functional.silu(z)
    if activation == "gelu":
        return torch.nn.functional.gelu(z)
    return z


def _normalised(x, groups, mean, rstd):
    """(x - mean) * rstd per sample and group; x (N, C, ...), mean and rstd (N, groups, 1)."""
    n = x.shape[0]
    return ((x.reshape(n, groups, -1) - mean) * rstd).reshape(x.shape)


def _centred(xg):
    """(x - mean, mean) over the last dimension; the mean of what is left makes up for the first mean's rounding, which
    is not small against a spread far below |mean|."""
    mean = xg.mean(-1, keepdim=True)
    d = xg - mean
    rest = d.mean(-1, keepdim=True)
    return d - rest, mean + rest


def _group_norm_torch(x, groups, weight, bias, eps, activation, slope, checkpoint):
    """The same in torch operations, at least in fp32."""
    if x.numel() == 0:
        y, each = x.clone(), (1, -1) + (1,) * (x.dim() - 2)
        for t in (weight, bias):                         # (they get gradients of 0)
            if t is not None:
                y = y + t.reshape(each).to(x.dtype)
        return y
    if checkpoint is not None and torch.is_grad_enabled():
        return _KeptTorchFn.apply(x, weight, bias, groups, eps, activation, slope, checkpoint)
    acc = torch.promote_types(x.dtype, torch.float32)
    n, c = x.shape[:2]
    d, _ = _centred(x.to(acc).reshape(n, groups, -1))
    z = (d * ((d ** 2).mean(-1, keepdim=True) + eps) ** -0.5).reshape(x.shape)
    each = (1, c) + (1,) * (x.dim() - 2)
    if weight is not None:
        z = z * weight.to(acc).reshape(each)
    if bias is not None:
        z = z + bias.to(acc).reshape(each)
    y = _act_torch(z, activation, slope).to(x.dtype)
    return y.movedim(1, -1).contiguous().movedim(-1, 1)


class _KeptTorchFn(torch.autograd.Function):
    """_group_norm_torch with x kept in 8 bits."""

    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, activation, slope, checkpoint):
        n = x.shape[0]
        d, mean = _centred(x.float().reshape(n, groups, -1))
        rstd = ((d ** 2).mean(-1, keepdim=True) + eps) ** -0.5
        codes, exps = _pack_torch(x.movedim(1, -1).contiguous(), checkpoint)
        ctx.save_for_backward(codes, exps, mean, rstd, weight, bias)
        ctx.args = x.shape, x.dtype, groups, activation, slope, checkpoint
        y = _group_norm_torch(x, groups, weight, bias, eps, activation, slope, None)
        # (a tensor of its own: a view from in here could not be changed in place)
        return torch.empty_strided(y.shape, y.stride(), dtype=y.dtype, device=y.device).copy_(y)

    @staticmethod
    def backward(ctx, gy):
        refuse_twice()
        codes, exps, mean, rstd, weight, bias = ctx.saved_tensors
        shape, dtype, groups, activation, slope, checkpoint = ctx.args
        x = torch.empty((shape[0], *shape[2:], shape[1]), dtype=dtype, device=codes.device)
        x = _unpack_torch(codes, exps, checkpoint, x).movedim(-1, 1).float()
        xh = _normalised(x, groups, mean, rstd)
        each = (1, shape[1]) + (1,) * (len(shape) - 2)
        w = 1.0 if weight is None else weight.float().reshape(each)
        with torch.enable_grad():
            z = (xh * w + (0.0 if bias is None else bias.float().reshape(each))).requires_grad_(True)
            dz, = torch.autograd.grad(_act_torch(z, activation, slope), z, gy.float())
        g = dz * w
        n = shape[0]
        mean_g = g.reshape(n, groups, -1).mean(-1, keepdim=True)
        mean_gx = (g * xh).reshape(n, groups, -1).mean(-1, keepdim=True)
        dx = ((g.reshape(n, groups, -1) - mean_g - xh.reshape(n, groups, -1) * mean_gx) * rstd).reshape(shape)
        dims = (0, *range(2, len(shape)))
        dw = (dz * xh).sum(dims).to(weight.dtype) if ctx.needs_input_grad[1] else None
        db = dz.sum(dims).to(bias.dtype) if ctx.needs_input_grad[2] else None
        return dx.to(dtype), dw, db, None, None, None, None, None


class GroupNormAct3d(nn.GroupNorm):
    """GroupNorm followed by an activation (``activation='none'``: GroupNorm alone), channels last.

    ``checkpoint``: how the input is kept for the backward pass (None, 'int8' or 'e4m3'). With the backend set to
    stock PyTorch it runs the formulas in torch operations.
    """

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation="none", negative_slope=0.01,
                 checkpoint=None, device=None, dtype=None):
        super().__init__(num_groups, num_channels, eps, affine, device=device, dtype=dtype)
        if activation not in _native.ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(map(repr, ACTIVATIONS))}, got {activation!r}")
        if checkpoint is not None:
            check_format(checkpoint, "checkpoint")
        self.activation, self.negative_slope, self.checkpoint = activation, negative_slope, checkpoint

    def forward(self, x):
        from .conv3d_wmma import _wmma_hw
        args = (x, self.num_groups, self.weight, self.bias, self.eps)
        if x.is_cuda and not _wmma_hw():
            _check(*args, self.activation, self.negative_slope, self.checkpoint)
            return _group_norm_torch(*args, self.activation, self.negative_slope, self.checkpoint)
        return group_norm_act(*args, activation=self.activation, negative_slope=self.negative_slope,
                              checkpoint=self.checkpoint)

    def extra_repr(self):
        more = "" if self.checkpoint is None else f", checkpoint={self.checkpoint!r}"
        return f"{super().extra_repr()}, activation={self.activation!r}{more}"


def _activation_of(m: nn.Module):
    """(name, slope) of an activation module that the kernels have, else None (a subclass may have its own forward)."""
    if type(m) is nn.ReLU:
        return "relu", 0.0
    if type(m) is nn.LeakyReLU:
        return "leaky_relu", m.negative_slope
    if type(m) is nn.SiLU:
        return "silu", 0.0
    if type(m) is nn.GELU and m.approximate == "none":
        return "gelu", 0.0
    return None


def fuse_group_norm(model: nn.Module) -> int:
    """Replace each (GroupNorm, ReLU / LeakyReLU / SiLU / GELU) pair inside an
    nn.Sequential with (GroupNormAct3d, Identity). The parameters are the
    GroupNorm's own, not copies. Pairs with hooks on either module stay as they
    are (what the hooks see would be gone). Returns the number of pairs fused."""
    count = 0
    for child in model.children():
        count += fuse_group_norm(child)
    if isinstance(model, nn.Sequential):
        names = list(model._modules.keys())
        for a, b in zip(names, names[1:]):
            norm, act = model._modules[a], _activation_of(model._modules[b])
            if type(norm) is nn.GroupNorm and act is not None and not (has_hooks(norm) or has_hooks(model._modules[b])):
                new = GroupNormAct3d(norm.num_groups, norm.num_channels, norm.eps, norm.affine, act[0], act[1],
                                     device="meta")
                new.weight, new.bias = norm.weight, norm.bias
                model._modules[a] = new.train(norm.training)
                model._modules[b] = nn.Identity()
                count += 1
    return count
