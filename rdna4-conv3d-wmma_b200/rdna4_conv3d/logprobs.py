"""Log-probabilities of given labels, with entropy and the most probable classes.

``log_probs(logits, target)`` reads (N, C, ...) logits -- the per-voxel maps
of the UNet, or (R, C) rows of tokens -- once and answers, for every voxel or
row, how likely the given label is, how unsure the prediction is (entropy),
the log-sum-exp, and with ``top_k`` the most probable classes with their
log-probabilities: a confidence map, a scoring pass, or the export of a
teacher for ``losses.distill_topk``. On a CUDA device it runs on the native
kernels (r4c_logp_*), forward and backward, for bf16, fp16 and fp32 logits;
CPU tensors take the same formulas in torch operations (any float type, so
gradients can be checked in 64 bits). No reference counterpart: the
reference's models end at their logits (benches/unet_e2e.py:35-38).
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _native

_FLOATS = frozenset((torch.bfloat16, torch.float16, torch.float32))
_PROXY = torch._C._TorchDispatchModeKey.PROXY


class LogProbs(NamedTuple):
    """Per voxel or row, all fp32 (indices int32); shape (N, ...), top_* (N, ..., top_k)."""
    logp: Optional[torch.Tensor]        # log-probability of the target, 0 where ignored; None without a target
    entropy: torch.Tensor               # -sum p ln p
    lse: torch.Tensor                   # ln sum exp(logits / temperature)
    top_logp: Optional[torch.Tensor]    # largest first; None with top_k = 0
    top_index: Optional[torch.Tensor]   # their classes, equal logits by lowest class


def check_logits(logits: torch.Tensor, temperature: float) -> None:
    shape = logits.shape
    if len(shape) < 2:
        raise ValueError(f"logits must be (N, C, ...), got shape {tuple(shape)}")
    if shape[1] == 0:
        raise ValueError("logits have no classes")
    if logits.dtype not in _FLOATS and (logits.is_cuda or not logits.is_floating_point()):
        raise TypeError(f"logits must be bf16, fp16 or fp32, got {logits.dtype}")
    if not (math.isfinite(temperature) and temperature > 0):
        raise ValueError(f"temperature must be finite and positive, got {temperature}")


def refuse_twice() -> None:
    """In a backward: the native gradients have no graph of their own."""
    if torch.is_grad_enabled():
        raise RuntimeError("the native gradient of this operator cannot be differentiated again (create_graph)")


def refuse_blind(logits: torch.Tensor) -> None:
    """Before a launch: what would go by it in silence. The kernels drop a forward-mode tangent, and make_fx keeps
    the outputs of this call as constants of its graph."""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(logits).tangent is not None:
        raise RuntimeError("this operator has no forward-mode derivative on a CUDA device")
    if torch._C._len_torch_dispatch_stack() and torch._C._get_dispatch_mode(_PROXY) is not None:
        raise RuntimeError("this operator cannot be traced into a graph of proxies (make_fx) on a CUDA device")


class LogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, top_k, temperature, ignore_index):
        rows = _native.Rows(logits, temperature)
        logp, entropy, lse, top_logp, top_index, stats = _native.logp_forward(rows, target, ignore_index, top_k, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(rows.z, target, entropy, stats)
        ctx.rows, ctx.row_shape, ctx.ignore_index = _native.SavedRows(rows), rows.shape, ignore_index
        if stats is not None:
            ctx.stats_bytes = stats.numel()
        if top_k:
            ctx.mark_non_differentiable(top_logp, top_index)
        return logp, entropy, lse, top_logp, top_index

    @staticmethod
    def backward(ctx, g_logp, g_entropy, g_lse, _top_logp, _top_index):
        refuse_twice()
        z, target, entropy, stats = ctx.saved_tensors
        rows = ctx.rows
        z, desc = rows.logits(z)
        if target is not None:
            target = rows.dense(target, ctx.row_shape, torch.int64)
        entropy = rows.dense(entropy, ctx.row_shape, torch.float32)
        if stats is not None:
            stats = rows.buffer(stats, ctx.stats_bytes)
        dz = _native.logp_backward(z, desc, target, ctx.ignore_index, entropy, stats, g_logp, g_entropy, g_lse)
        return dz, None, None, None, None


def log_probs(logits: torch.Tensor, target: Optional[torch.Tensor] = None, *, top_k: int = 0,
              temperature: float = 1.0, ignore_index: int = -100) -> LogProbs:
    """Log-probabilities under softmax(logits / temperature) over dim 1.

    logits: (N, C, ...); any strides (channels-last is read as it lies).
    target: integer classes (N, ...), or None. ``ignore_index`` gives
        log-probability 0 and no gradient; any other class outside [0, C) is
        an error (on a CUDA device it counts as ignored and sets code 6 in
        ``_native.device_error()``).
    top_k: how many of the most probable classes to return, at most 128.

    ``logp``, ``entropy`` and ``lse`` carry gradients to the logits (reverse
    mode, once; on the CPU as torch has them); ``top_logp`` does not. A row
    without a finite logit has lse, logp and top_logp -inf, entropy 0 and no
    gradient; one that holds a NaN or +inf has no distribution: its values are
    NaN (logp 0 where ignored), its top_index -1, and its gradient NaN, or 0
    where it has no upstream gradient other than 0.
    """
    check_logits(logits, temperature)
    zs = logits.shape
    if not 0 <= top_k <= _native.TOPK_MAX or top_k > zs[1]:
        raise ValueError(f"top_k must be in [0, min({_native.TOPK_MAX}, C = {zs[1]})], got {top_k}")
    if target is not None:
        ts = target.shape
        if len(ts) != len(zs) - 1 or ts[0] != zs[0] or ts[1:] != zs[2:]:
            raise ValueError(f"target must have shape {tuple(zs[:1] + zs[2:])}, got {tuple(target.shape)}")
        if target.dtype != torch.int64 and target.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):
            raise TypeError(f"target must hold integers, got {target.dtype}")
        if target.device != logits.device:
            raise ValueError(f"target is on {target.device}, logits on {logits.device}")
    if not logits.is_cuda:
        return _log_probs_torch(logits, target, top_k, temperature, ignore_index)
    refuse_blind(logits)
    if target is not None:
        if target.dtype != torch.int64:
            target = target.to(torch.int64)
        target = target.contiguous()
    # (torch.jit.trace records a Function, but of bare launches only the empty tensors that they fill)
    if torch.is_grad_enabled() and logits.requires_grad or torch._C._is_tracing():
        return LogProbs(*LogProbsFn.apply(logits, target, top_k, temperature, ignore_index))
    return LogProbs(*_native.logp_forward(_native.Rows(logits, temperature), target, ignore_index, top_k, False)[:5])


class _BadRowsFn(torch.autograd.Function):
    """Values of rows that may be bad (a NaN or +inf logit), as they are; a bad row's logits get a gradient of NaN
    where any of its values has one that is not 0."""
    generate_vmap_rule = True

    @staticmethod
    def forward(z, bad, *values):
        return tuple(v.clone() for v in values)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.save_for_backward(inputs[0], inputs[1])
        ctx.save_for_forward(inputs[1])
        ctx.set_materialize_grads(False)

    @staticmethod
    def backward(ctx, *grads):
        z, bad = ctx.saved_tensors
        hit = torch.zeros_like(bad)
        for g in grads:
            if g is not None:
                hit = hit | (g != 0).unsqueeze(-1)
        return torch.where(hit & bad, float("nan"), torch.zeros_like(z)), None, *grads

    @staticmethod
    def jvp(ctx, _z, _bad, *tangents):
        return tangents


def _log_probs_torch(logits, target, top_k, temperature, ignore_index) -> LogProbs:
    """The same values in torch operations, at least in fp32."""
    acc = torch.promote_types(logits.dtype, torch.float32)
    out = torch.float32 if acc == torch.float32 else acc
    z = logits.movedim(1, -1).to(acc)
    c = z.shape[-1]
    s = z / temperature
    inf = float("inf")
    empty = (z == -inf).all(-1, keepdim=True)
    bad = (z.isnan() | (z == inf)).any(-1, keepdim=True)
    m = s.detach().amax(-1, keepdim=True)
    m = torch.where(empty | bad, torch.zeros_like(m), m)
    d = s - m
    # masked classes leave the sums: their share of the gradient is 0, not 0 * inf
    dead = (d == -inf) | bad
    e = torch.where(dead, torch.zeros_like(d), torch.exp(torch.where(dead, torch.zeros_like(d), d)))
    total = e.sum(-1, keepdim=True)
    ln_s = torch.log(torch.where(empty | bad, torch.ones_like(total), total))
    ln_p = torch.where(empty, torch.full_like(d, -inf), d - ln_s)
    p = e / torch.where(empty | bad, torch.ones_like(total), total)
    entropy = -(p * torch.where(dead, torch.zeros_like(d), ln_p)).sum(-1)
    lse = (m + ln_s).squeeze(-1)
    lse = torch.where(empty.squeeze(-1), torch.full_like(lse, -inf), lse)
    nan = torch.full_like(lse, float("nan"))
    b = bad.squeeze(-1)
    entropy, lse = torch.where(b, nan, entropy), torch.where(b, nan, lse)
    logp = None
    if target is None:
        entropy, lse = _BadRowsFn.apply(z, bad, entropy, lse)
    else:
        t = target.to(torch.int64)
        counted = t != ignore_index
        if bool((((t < 0) | (t >= c)) & counted).any()):
            raise IndexError(f"target out of range [0, {c})")
        at = torch.where(counted, t, torch.zeros_like(t)).unsqueeze(-1)
        logp = torch.where(b, nan, ln_p.gather(-1, at).squeeze(-1))
        logp, entropy, lse = _BadRowsFn.apply(z, bad, logp, entropy, lse)
        logp = torch.where(counted, logp, torch.zeros_like(logp)).to(out)
    top_logp = top_index = None
    if top_k:
        # a stable descending sort keeps equal logits in class order
        order = torch.sort(z.detach(), dim=-1, descending=True, stable=True).indices[..., :top_k]
        top_logp = torch.where(bad, nan.unsqueeze(-1), ln_p.detach().gather(-1, order)).to(out)
        top_index = torch.where(bad, torch.full_like(order, -1), order).to(torch.int32)
    return LogProbs(logp, entropy.to(out), lse.to(out), top_logp, top_index)
