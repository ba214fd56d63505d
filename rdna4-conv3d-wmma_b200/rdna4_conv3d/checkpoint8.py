"""Activations in 8 bits, kept from the forward to the backward pass.

A training step on volumes is bound by what it keeps: a layer's input stays
until its weight gradient has read it. ``pack8`` writes an activation as one
byte an element and one exponent for every 32 (in memory order), ``unpack8``
reads it back; on a CUDA device both are native kernels (r4c_pack8,
r4c_unpack8), on the CPU the same arithmetic in torch operations with the
same codes. Used by ``Conv3dWmma`` (weight gradients from the kept input) and
``group_norm.GroupNormAct3d`` (whose backward kernels read the 8 bits as they
are) where their ``checkpoint`` is set; ``checkpoint_activations(model)`` sets
it on all of a model's. Forward results do not change; gradients are those at
the values that the 8 bits hold. No reference counterpart (its autograd
keeps activations whole, src/rdna4_conv3d/conv3d_wmma.py:1262-1270).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
import torch.nn as nn

from . import _native
from .logprobs import refuse_blind

_FLOATS = frozenset((torch.bfloat16, torch.float16, torch.float32))
FORMATS = tuple(_native.Q8_FORMATS)


class Packed8(NamedTuple):
    """A dense tensor in 8 bits."""
    codes: torch.Tensor                 # uint8, one an element in memory order
    exponents: torch.Tensor             # uint8, e + 127 for every 32 elements
    shape: torch.Size
    stride: Tuple[int, ...]
    dtype: torch.dtype
    format: str                         # 'int8' or 'e4m3'


def check_format(fmt: str, name: str = "format") -> str:
    if fmt not in _native.Q8_FORMATS:
        raise ValueError(f"{name} must be one of {', '.join(map(repr, FORMATS))}, got {fmt!r}")
    return fmt


def _is_dense(x: torch.Tensor) -> bool:
    """Whether x's elements fill its memory without gaps or overlaps."""
    if x.is_contiguous() or x.dim() == 5 and x.is_contiguous(memory_format=torch.channels_last_3d):
        return True
    if x.numel() == 0:
        return True
    expect = 1
    for stride, size in sorted((st, sz) for sz, st in zip(x.shape, x.stride()) if sz > 1):
        if stride != expect:
            return False
        expect *= size
    return True


def pack8(x: torch.Tensor, format: str = "int8") -> Packed8:
    """x (bf16, fp16 or fp32) in 8 bits.

    Every 32 elements in memory order share the power of two 2^e with the
    smallest e >= -127 that brings their largest finite magnitude to at most
    127 ('int8': whole numbers, an error of at most 2^e / 2) or 448 ('e4m3':
    8-bit floating point, an error of at most 2^-4 of a value, and of 2^e /
    1024 below 2^(e-6)). x / 2^e is rounded to the nearest, ties to even. NaN
    and infinities come back as NaN. A tensor with gaps or overlaps is copied
    first; autograd does not see this call.
    """
    dtype = x.dtype
    code = _native.Q8_FORMATS.get(format)
    if code is None:
        check_format(format)
    if dtype not in _FLOATS:
        raise TypeError(f"pack8 takes bf16, fp16 or fp32, got {dtype}")
    refuse_blind(x)
    _refuse_trace(x)
    return _pack8(x, format, code)


def _pack8(x: torch.Tensor, format: str, code: int) -> Packed8:
    dtype = x.dtype
    if not _is_dense(x):
        x = x.detach().contiguous()
    if not x.is_cuda:
        codes, exps = _pack_torch(x.detach(), format)
    else:
        codes, exps = _native.pack8(x, code)
    return Packed8(codes, exps, x.shape, x.stride(), dtype, format)


def _refuse_trace(t: torch.Tensor) -> None:
    """torch.jit.trace would record the empty tensors that bare launches fill."""
    if t.is_cuda and torch._C._is_tracing():
        raise RuntimeError("pack8 and unpack8 cannot be traced by torch.jit.trace on a CUDA device")


def unpack8(packed: Packed8) -> torch.Tensor:
    """The values that the 8 bits hold, in the packed tensor's type, shape and strides: code * 2^e, at most the
    type's largest finite number."""
    codes, exps, shape, stride, dtype, fmt = packed
    code = _native.Q8_FORMATS.get(fmt)
    if code is None:
        check_format(fmt)
    _refuse_trace(codes)
    count = shape.numel()
    if codes.numel() != count or exps.numel() != (count + 31) // _native.Q8_BLOCK:
        raise ValueError(f"{count} elements need as many codes and {-(-count // _native.Q8_BLOCK)} exponents, got "
                         f"{codes.numel()} and {exps.numel()}")
    if codes.dtype != torch.uint8 or exps.dtype != torch.uint8 or codes.device != exps.device:
        raise ValueError("codes and exponents must be uint8 on one device")
    if dtype not in _FLOATS:
        raise TypeError(f"unpack8 gives bf16, fp16 or fp32, got {dtype}")
    out = torch.empty_strided(shape, stride, dtype=dtype, device=codes.device)
    if not _is_dense(out):
        raise ValueError(f"strides {tuple(stride)} of shape {tuple(shape)} leave gaps or overlap")
    if codes.data_ptr() & 15 or not codes.is_contiguous():
        codes = codes.clone(memory_format=torch.contiguous_format)
    if not exps.is_contiguous():
        exps = exps.contiguous()
    if not codes.is_cuda:
        return _unpack_torch(codes, exps, fmt, out)
    return _native.unpack8(codes, exps, code, out)


def _memory_order(x: torch.Tensor) -> torch.Tensor:
    """A dense tensor's elements as they lie in memory (a view)."""
    return x.as_strided((x.numel(),), (1,))


def _power(byte: torch.Tensor) -> torch.Tensor:
    """2^(byte - 127) in fp32, exactly."""
    byte = byte.to(torch.int32)
    return torch.where(byte == 0, 1 << 22, byte << 23).to(torch.int32).view(torch.float32)


def _pack_torch(x: torch.Tensor, fmt: str):
    flat = _memory_order(x).float()
    count = flat.numel()
    b = torch.nn.functional.pad(flat, (0, -count % _native.Q8_BLOCK)).reshape(-1, _native.Q8_BLOCK)
    finite = b.abs() < float("inf")
    bits = torch.where(finite, b.abs(), 0.0).amax(1, keepdim=True).view(torch.int32)
    if fmt == "int8":
        byte = (bits >> 23) - 6 + ((bits & 0x7fffff) > 0x7e0000)
    else:
        byte = (bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000)
    byte = byte.clamp(min=0)
    q = torch.where(finite, b, 0.0) * _power(254 - byte)
    if fmt == "int8":
        code = torch.where(finite, torch.round(q), -128.0).to(torch.int8).view(torch.uint8)
    else:
        code = torch.where(finite, q.to(torch.float8_e4m3fn).view(torch.uint8), 0x7f)
    return code.reshape(-1)[:count].contiguous(), byte.to(torch.uint8).reshape(-1)


def _unpack_torch(codes: torch.Tensor, exps: torch.Tensor, fmt: str, out: torch.Tensor) -> torch.Tensor:
    count = codes.numel()
    if fmt == "int8":
        q = codes.view(torch.int8).float()
        q = torch.where(q == -128.0, float("nan"), q)
    else:
        q = codes.view(torch.float8_e4m3fn).float()
    scale = _power(exps).repeat_interleave(_native.Q8_BLOCK)[:count]
    limit = torch.finfo(out.dtype).max
    _memory_order(out).copy_((q * scale).clamp(-limit, limit))
    return out


def checkpoint_activations(model: nn.Module, format: Optional[str] = "int8") -> int:
    """Sets ``checkpoint`` on every Conv3dWmma and GroupNormAct3d of a model
    (None: keep activations whole again). Returns how many modules that were."""
    from .conv3d_wmma import Conv3dWmma
    from .group_norm import GroupNormAct3d
    if format is not None:
        check_format(format)
    count = 0
    for m in model.modules():
        if isinstance(m, (Conv3dWmma, GroupNormAct3d)):
            m.checkpoint = format
            count += 1
    return count
