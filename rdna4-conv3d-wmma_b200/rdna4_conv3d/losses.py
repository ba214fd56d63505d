"""Losses over logits on the native kernels: cross-entropy (r4c_ce_*) and
distillation from a teacher's top classes (r4c_distill_*).

``cross_entropy(logits, target)`` is ``F.cross_entropy(logits, target)``
(reduction 'mean', no class weights, ``ignore_index``) for channels_last_3d
bf16/fp16 logits on a CUDA device: one kernel pass forward (per-voxel
log-sum-exp in fp32, deterministic mean) and one backward, with no fp32
copy of the logits and no layout change. Other inputs take F.cross_entropy.

``distill_topk(logits, teacher_logp, teacher_index)`` trains a student on
what ``logprobs.log_probs(teacher_logits, top_k=k)`` gave for a teacher: its
k most probable classes per voxel or token, as they are stored.

No reference counterparts: the reference's training step computes its loss
with stock PyTorch (benches/unet_e2e.py:41-52).
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from . import _native
from .conv3d_wmma import _as_ndhwc
from .logprobs import check_logits, refuse_blind, refuse_twice


class CrossEntropyNDHWCFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, ignore_index):
        loss_count = _native.ce_forward(logits, target, ignore_index)
        ctx.save_for_backward(logits, target, loss_count)
        ctx.ignore_index = ignore_index
        return loss_count[0].clone()

    @staticmethod
    def backward(ctx, grad):
        logits, target, loss_count = ctx.saved_tensors
        dz = None
        if ctx.needs_input_grad[0]:
            # (hooks on saved tensors may give them back in other strides)
            logits, target, loss_count = _as_ndhwc(logits), target.contiguous(), loss_count.contiguous()
            dz = _native.ce_backward(logits, target, ctx.ignore_index, loss_count, grad)
        return dz, None, None


def _native_ok(logits: torch.Tensor, target: torch.Tensor) -> bool:
    return (logits.is_cuda and logits.dim() == 5 and logits.dtype in (torch.bfloat16, torch.float16)
            and logits.is_contiguous(memory_format=torch.channels_last_3d)
            and target.dtype == torch.int64 and target.is_contiguous() and target.device == logits.device
            and tuple(target.shape) == (logits.shape[0],) + tuple(logits.shape[2:]))


def cross_entropy(logits: torch.Tensor, target: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """Mean cross-entropy of (N, C, D, H, W) logits against (N, D, H, W) labels."""
    if _native_ok(logits, target):
        return CrossEntropyNDHWCFn.apply(logits, target, int(ignore_index))
    return F.cross_entropy(logits, target, ignore_index=ignore_index)


class DistillTopKFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_logp, teacher_index, temperature, rest, weight, mean):
        rows = _native.Rows(logits, temperature)
        loss, state = _native.distill_forward(rows, teacher_logp, teacher_index, rest, weight, mean)
        ctx.save_for_backward(rows.z, teacher_logp, teacher_index, weight, state)
        ctx.rows, ctx.rest, ctx.mean = _native.SavedRows(rows), rest, mean
        ctx.teacher = teacher_logp.shape, teacher_logp.dtype, teacher_index.dtype, state.numel()
        return loss

    @staticmethod
    def backward(ctx, grad):
        refuse_twice()
        z, teacher_logp, teacher_index, weight, state = ctx.saved_tensors
        rows, (shape, logp_dtype, index_dtype, nbytes) = ctx.rows, ctx.teacher
        z, desc = rows.logits(z)
        teacher_logp = rows.dense(teacher_logp, shape, logp_dtype)
        teacher_index = rows.dense(teacher_index, shape, index_dtype)
        if weight is not None:
            weight = rows.dense(weight, shape[:-1], torch.float32)
        state = rows.buffer(state, nbytes)
        dz = _native.distill_backward(z, desc, teacher_logp, teacher_index, ctx.rest, weight, ctx.mean, state, grad)
        return dz, None, None, None, None, None, None


def distill_topk(logits: torch.Tensor, teacher_logp: torch.Tensor, teacher_index: torch.Tensor, *,
                 temperature: float = 1.0, rest: bool = False, weight: Optional[torch.Tensor] = None,
                 reduction: str = "mean") -> torch.Tensor:
    """T^2 KL(teacher || student) where the teacher is given by its top classes.

    logits: (N, C, ...) of the student, p = softmax(logits / temperature) over dim 1; any strides.
    teacher_logp, teacher_index: (N, ..., k), the teacher's k log-probabilities
        (at the same temperature) and their classes, k at most 128. A negative
        index or a log-probability of -inf marks an unused place. A class that
        is listed twice counts with both its probabilities.
    rest: False -- the k probabilities are renormalised (so the teacher's
        logits / temperature serve as well); True -- they are taken as they
        are, and what is missing to 1 stands for all other classes together
        (less than 1e-6 is rounding and counts as nothing; so does, where the
        student has no other class, what rounding to bf16 or fp16 explains).
        On a CUDA device it takes four million classes at most.
    weight: (N, ...), >= 0: the weight of each voxel or token (0: masked).
    reduction: 'mean' -- sum(w L) / sum(w), NaN when no row takes part; 'none' -- w L, (N, ...).

    Rows whose places are all unused, whose weight is 0 or whose logits are
    all -inf take no part: loss 0, no share of the mean, no gradient. The
    gradient reaches the logits only (reverse mode, once; on the CPU as torch
    has it). An index beyond the classes is an error (on a CUDA device it is
    unused and sets code 6 in ``_native.device_error()``).
    """
    check_logits(logits, temperature)
    mean = reduction == "mean"
    if not mean and reduction != "none":
        raise ValueError(f"reduction must be 'mean' or 'none', got {reduction!r}")
    zs, ts, dev = logits.shape, teacher_logp.shape, logits.device
    if teacher_index.shape != ts or len(ts) != len(zs) or ts[0] != zs[0] or ts[1:-1] != zs[2:]:
        raise ValueError(f"teacher_logp and teacher_index must have shape {tuple(zs[:1] + zs[2:])} + (k,), got "
                         f"{tuple(ts)} and {tuple(teacher_index.shape)}")
    if not 1 <= ts[-1] <= _native.TOPK_MAX:
        raise ValueError(f"the teacher's classes per row must be in [1, {_native.TOPK_MAX}], got {ts[-1]}")
    if not teacher_logp.is_floating_point():
        raise TypeError(f"teacher_logp must be a floating type, got {teacher_logp.dtype}")
    if teacher_index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"teacher_index must be int32 or int64, got {teacher_index.dtype}")
    if teacher_logp.device != dev or teacher_index.device != dev:
        raise ValueError(f"the teacher is on {teacher_logp.device} and {teacher_index.device}, logits on {dev}")
    if weight is not None:
        if weight.shape != zs[:1] + zs[2:]:
            raise ValueError(f"weight must have shape {tuple(zs[:1] + zs[2:])}, got {tuple(weight.shape)}")
        if weight.device != dev:
            raise ValueError(f"weight is on {weight.device}, logits on {dev}")
    if not logits.is_cuda:
        return _distill_torch(logits, teacher_logp, teacher_index, temperature, rest, weight, reduction)
    refuse_blind(logits)
    if teacher_logp.requires_grad:
        teacher_logp = teacher_logp.detach()
    if teacher_logp.dtype == torch.float64:
        teacher_logp = teacher_logp.float()
    if weight is not None:
        weight = weight.detach().to(torch.float32).contiguous()
    teacher_logp, teacher_index, rest = teacher_logp.contiguous(), teacher_index.contiguous(), bool(rest)
    if torch.is_grad_enabled() and logits.requires_grad or torch._C._is_tracing():
        return DistillTopKFn.apply(logits, teacher_logp, teacher_index, temperature, rest, weight, mean)
    rows = _native.Rows(logits, temperature)
    return _native.distill_forward(rows, teacher_logp, teacher_index, rest, weight, mean)[0]


def _distill_torch(logits, teacher_logp, teacher_index, temperature, rest, weight, reduction):
    """The same loss in torch operations, in 64 bits: the gradient is a difference of probabilities, and torch's
    own roundings of each would be what is left of it where the student agrees with the teacher."""
    acc = torch.float64
    inf = float("inf")
    z = logits.movedim(1, -1).to(acc)
    v, i = teacher_logp.detach().to(acc), teacher_index.to(torch.int64)
    c = z.shape[-1]
    valid = (i >= 0) & (v != -inf)
    if bool((valid & (i >= c)).any()):
        raise IndexError(f"teacher_index out of range [0, {c})")
    zero = torch.zeros((), dtype=acc, device=z.device)
    i = torch.where(valid, i, torch.zeros_like(i))
    w = torch.ones(z.shape[:-1], dtype=acc, device=z.device) if weight is None else weight.detach().to(acc)
    part = valid.any(-1) & ~(z == -inf).all(-1) & (w != 0)
    w = torch.where(part, w, zero)
    z = torch.where(part.unsqueeze(-1), z, zero)
    # differences from a maximum, taken before they are scaled: far from zero, lse would swallow ln S
    m = z.detach().amax(-1, keepdim=True)
    s = (z - m) / temperature
    lse = torch.logsumexp(s, -1, keepdim=True)
    v = torch.where(valid, v, zero - inf)
    if not rest:
        v = v - torch.where(part.unsqueeze(-1), torch.logsumexp(v, -1, keepdim=True), zero)
    q = torch.where(valid, torch.exp(v), zero)
    ln_p = s.gather(-1, i) - lse
    some = valid & ~(q == 0)
    row = torch.where(some, q * (torch.where(some, v, zero) - torch.where(some, ln_p, zero)), zero).sum(-1)
    if rest:
        qr = 1.0 - q.sum(-1)
        seen = torch.zeros(z.shape, dtype=torch.int64, device=z.device).scatter_add(-1, i, valid.long()) > 0
        alive = ~seen & (z != -inf)
        any_alive = alive.any(-1)
        # what the sum's rounding explains is no rest, nor is what that of 16-bit pairs explains against no class
        noise = torch.zeros_like(qr)
        if teacher_logp.dtype in (torch.bfloat16, torch.float16):
            x = (torch.where(q > 0, v, zero) * (0.5 * torch.finfo(teacher_logp.dtype).eps)).abs()
            noise = torch.where(any_alive, noise, (q * (x + x * x)).sum(-1))
        qr = torch.where(qr >= 1e-6 + noise, qr, zero)
        # the unlisted classes from a maximum of their own, which may lie far below the row's
        mr = torch.where(alive, z.detach(), zero - inf).amax(-1, keepdim=True)
        mr = torch.where(any_alive.unsqueeze(-1), mr, m)
        sr = torch.where(alive, (z - mr) / temperature, zero - inf)
        ln_r = torch.logsumexp(torch.where(any_alive.unsqueeze(-1), sr, zero), -1) + ((mr - m) / temperature).squeeze(-1)
        ln_r = torch.where(any_alive, ln_r, zero - inf)
        rest_term = qr * (torch.log(torch.where(qr > 0, qr, zero + 1.0)) - ln_r + lse.squeeze(-1))
        row = row + torch.where(qr > 0, rest_term, zero)
    out = torch.promote_types(logits.dtype, torch.float32)
    row = torch.where(part, temperature * temperature * w * row, zero)
    if reduction == "none":
        return row.to(out)
    return (row.sum() / w.sum()).to(out)
