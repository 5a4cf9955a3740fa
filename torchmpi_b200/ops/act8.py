"""Activations kept for the backward pass in 8 bits (csrc/kernels/act8.cu, grouped.cu; autograd in csrc/bindings/experts.cpp).

A checkpoint ``Act8(q, scale)`` holds a tensor ``[..., C]`` as e4m3 numbers ``q`` with one power of two for 32 consecutive
elements of a row, a byte of ``scale [..., ceil(C / 32)]`` that stands for ``2 ** (byte - 127)``: the smallest one, from
``2 ** -126``, under which the block's largest finite element is at most 448.  Every element is rounded once, by at most
half an e4m3 step (a sixteenth of it).  Infinities and NaN are kept as NaN.

``quantize`` / ``dequantize`` make one and read it; ``gelu_gradient(dy, checkpoint of z)`` is the backward pass of a GELU that
kept its input so; ``mlp(x, w1, b1, w2, b2)`` is a whole MLP that keeps its input and its pre-activation so (1.03 bytes an
element instead of 2, and no second copy of the hidden layer): about a quarter of what the two linear layers keep.  Its
gradients are those of the formulas with the checkpoints' values in place of the activations.  What the kernels do not
take (CPU, other dtypes; ``mlp``: other than bf16, widths that are not multiples of 8) runs on PyTorch operations with the same results.
The reference keeps no activations of its own (its models are Torch7's).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
import torch.nn.functional as F

from .. import _native
from .._lib import DTYPES

BLOCK = 32          # elements that share a scale


class Act8(NamedTuple):
    """``q [..., C]`` (``torch.float8_e4m3fn``) and ``scale [..., ceil(C / 32)]`` (``torch.uint8``)."""
    q: torch.Tensor
    scale: torch.Tensor


def __getattr__(name: str):
    if name == "launch_count":               # kernels launched by this module
        return _native.launches(_native.ACT8)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def same_device(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Raises unless all tensors are on one device, and that, if it is a GPU, is the current one (there is one process per GPU)."""
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        raise ValueError(f"{what}: tensors on different devices: {sorted(map(str, devices))}")
    d = devices.pop()
    if d.type == "cuda" and d.index != torch.cuda.current_device():
        raise ValueError(f"{what}: tensors on {d}, but the current device is cuda:{torch.cuda.current_device()}")


def _wide(t: torch.Tensor) -> torch.Tensor:
    """32 bits, or 64 where the tensor has them."""
    return t.to(torch.promote_types(t.dtype, torch.float32))


def _two_to(e: torch.Tensor) -> torch.Tensor:
    return ((e.int() + 127) << 23).view(torch.float32)            # exact, unlike a power function


def _blocks(x: torch.Tensor) -> torch.Tensor:
    return F.pad(x, (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))


def _quantize(x: torch.Tensor) -> Act8:
    b = _blocks(x.float())
    finite = torch.isfinite(b)
    a = torch.where(finite, b.abs(), 0).amax(-1, keepdim=True)
    m, e = torch.frexp(a)                                          # a = m 2^e, 1/2 <= m < 1
    e = torch.where(a > 0, torch.where(m > 0.875, e - 8, e - 9), -126).clamp_min(-126)
    half = torch.div(-e, 2, rounding_mode="floor")                 # 2^126 * 2^-e in two exact steps
    q = torch.where(finite, b * _two_to(half) * _two_to(-e - half), float("nan")).to(torch.float8_e4m3fn)
    return Act8(q.flatten(-2)[..., : x.shape[-1]].contiguous(), (e + 127).to(torch.uint8).squeeze(-1))


def _dequantize(a: Act8, dtype: torch.dtype) -> torch.Tensor:
    scale = (a.scale.int() << 23).view(torch.float32).unsqueeze(-1)
    return (_blocks(a.q.float()) * scale).flatten(-2)[..., : a.q.shape[-1]].to(dtype)


def _checked(what: str, a: Act8) -> None:
    q, scale = a
    if q.dtype != torch.float8_e4m3fn or scale.dtype != torch.uint8:
        raise ValueError(f"{what}: a checkpoint is float8_e4m3fn with uint8 scales, not {q.dtype} and {scale.dtype}")
    if q.dim() < 1 or scale.shape != q.shape[:-1] + ((q.shape[-1] + BLOCK - 1) // BLOCK,):
        raise ValueError(f"{what}: scales {tuple(scale.shape)} do not belong to a checkpoint of {tuple(q.shape)}")


def quantize(x: torch.Tensor) -> Act8:
    """The checkpoint of ``x [..., C]`` (of 64 bits: of their values in 32); not differentiable."""
    if x.is_cuda:
        kept = _native.ext().act8_quantize(x)          # None: nothing for the kernel
        if kept is not None:
            return Act8(*kept)
    if x.dim() < 1 or not x.dtype.is_floating_point:
        raise ValueError(f"quantize expects a floating tensor with at least one dimension, got {x.dtype} {tuple(x.shape)}")
    same_device("quantize", x)
    return _quantize(x.detach())


def dequantize(a: Act8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """What the checkpoint stands for, rounded to ``dtype`` (exact in bf16 and fp32 within their range)."""
    if a[0].is_cuda:
        x = _native.ext().act8_restore(a[0], a[1], DTYPES.get(dtype, -1))
        if x is not None:
            return x
    _checked("dequantize", a)
    same_device("dequantize", *a)
    if not dtype.is_floating_point:
        raise ValueError(f"dequantize: {dtype} is not a floating type")
    return _dequantize(a, dtype)


def _gelu_parts(z: torch.Tensor):
    cdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * 0.3989422804014327


def gelu_gradient(dy: torch.Tensor, a: Act8) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(dy * gelu'(z), gelu(z))`` (erf form) for the values ``z`` of the checkpoint ``a``, both of ``dy``'s dtype; the first is differentiable in ``dy``."""
    if dy.is_cuda:
        both = _native.ext().act8_gelu_gradient(dy, a[0], a[1])
        if both is not None:
            return both
    _checked("gelu_gradient", a)
    if dy.shape != a.q.shape or not dy.dtype.is_floating_point:
        raise ValueError(f"gelu_gradient: a gradient of {dy.dtype} {tuple(dy.shape)} for a checkpoint of {tuple(a.q.shape)}")
    same_device("gelu_gradient", dy, *a)
    g = _wide(dy)
    h, slope = _gelu_parts(_dequantize(a, g.dtype))
    return (g * slope).to(dy.dtype), h.to(dy.dtype)


def refuse_graph() -> None:
    """Called by backward functions whose gradients are constants to autograd: one asked for with a graph would lose its part of what it enters in silence."""
    if torch.is_grad_enabled():
        raise RuntimeError("layers of experts and 8-bit checkpoints can be differentiated once (no create_graph)")


class _Mlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2):
        z = F.linear(_wide(x), _wide(w1), None if b1 is None else _wide(b1))
        ctx.save_for_backward(*_quantize(x), *_quantize(z), w1, b1, w2, b2)
        return F.linear(_gelu_parts(z)[0], _wide(w2), None if b2 is None else _wide(b2)).to(x.dtype)

    @staticmethod
    def backward(ctx, dy):
        refuse_graph()
        xq, xs, zq, zs, w1, b1, w2, b2 = ctx.saved_tensors
        dy = _wide(dy)
        x, z = _dequantize(Act8(xq, xs), dy.dtype), _dequantize(Act8(zq, zs), dy.dtype)
        h, slope = _gelu_parts(z)
        dz = dy @ _wide(w2) * slope
        grads = (dz @ _wide(w1), dz.t() @ x, None if b1 is None else dz.sum(0), dy.t() @ h, None if b2 is None else dy.sum(0))
        return tuple(g if g is None else g.to(t.dtype) for g, t in zip(grads, (w1, w1, b1, w2, b2)))


def mlp(x: torch.Tensor, w1: torch.Tensor, b1: Optional[torch.Tensor], w2: torch.Tensor, b2: Optional[torch.Tensor]) -> torch.Tensor:
    """``gelu(x @ w1.T + b1) @ w2.T + b2`` for ``x [..., C]``, ``w1 [H, C]``, ``w2 [D, H]``; where gradients are wanted, ``x`` and the
    pre-activation are kept in 8 bits.  The checkpoint is that of the fp32 sums, and the GELU is formed from them too."""
    if x.is_cuda:
        y = _native.ext().act8_mlp(x, w1, b1, w2, b2)
        if y is not None:
            return y
    if not (w1.dim() == 2 and w2.dim() == 2 and x.dim() >= 1 and x.shape[-1] == w1.shape[1] and w2.shape[1] == w1.shape[0]
            and (b1 is None or b1.shape == w1.shape[:1]) and (b2 is None or b2.shape == w2.shape[:1])):
        raise ValueError("mlp expects x [..., C], w1 [H, C], b1 [H], w2 [D, H] and b2 [D]")
    tensors = [t for t in (x, w1, b1, w2, b2) if t is not None]
    same_device("mlp", *tensors)
    if len({t.dtype for t in tensors}) > 1 or not x.dtype.is_floating_point:
        raise ValueError(f"mlp: tensors of one floating dtype are expected, got {sorted({str(t.dtype) for t in tensors})}")
    y = _Mlp.apply(x.reshape(-1, x.shape[-1]), w1, b1, w2, b2)
    return y.view(x.shape[:-1] + w2.shape[:1])
