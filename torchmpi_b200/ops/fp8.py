"""Products in 8-bit floating point with a scale for each block of 128 (csrc/kernels/fp8.cu, gemm_fp8.cu; autograd in csrc/bindings/fp8.cpp).

``quantize(x)`` keeps a matrix ``[..., C]`` as e4m3 numbers with one power of two for 128 consecutive elements of a row: the smallest one, from
``2 ** -126``, under which the block's largest finite element is at most 448.  Every element is rounded once, by at most half an e4m3 step (a
sixteenth of it); infinities and NaN become NaN.  ``quantize_columns(x)`` is ``quantize(x.T)``, ``quantize_both(x)`` both from one pass.
``matmul(a, b)`` is ``a @ b.T`` of two such matrices: the tensor cores multiply the numbers and the powers of two, sums are in fp32.

``linear(x, w, bias, gelu)`` is a linear layer whose three products are formed so.  Forward: ``z = Q(x) Q(w).T + bias``, and with ``gelu`` the GELU
(erf form) of the rounded ``z``.  Backward, with ``dz = dy`` or, rounded to the tensors' type, ``dy * gelu'(z)``: ``dx = Q(dz) Q(w.T).T``, ``dw = Q(dz.T)
Q(x.T).T``, ``db`` the sums of ``dz``.  ``Q`` takes its blocks along the dimension that a product sums over.  For backward ``x`` is kept in 8 bits (a byte
an element), ``w`` too, and ``z`` as it is.  With a ``Block8`` in the place of ``w`` (weights kept in 8 bits by a generating program) there is no
backward pass; a few tokens (up to 32) then take one launch that is bound by reading the weights.

Every result is bit-reproducible (the bytes of ``scale`` behind a matrix' last row and block mean nothing and are not); tokens are independent of each other.  How many they are decides about the
kernel and how it cuts K: the order of the sums, and in bf16 the form of the GELU's Phi (absolute error 1.5e-7 up to 32 tokens and where K is cut, else 1.4e-6; of the slope backward 1.4e-6), so that a token
may round otherwise among others.  ``Phi(-inf) * -inf`` is NaN.  What the kernels do not take (CPU, 64 bits, tensors of several
types, nothing to multiply) runs on PyTorch operations.  The reference has no such products (its models are Torch7's).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch
import torch.autograd.forward_ad as fwd
import torch.nn.functional as F

from .. import _native
from .._lib import DTYPES, lib, TorchMPIError
from .act8 import _gelu_parts, _two_to, _wide, same_device

BLOCK = 128         # elements that share a scale


class Block8(NamedTuple):
    """A matrix ``[rows, cols]`` in 8 bits: ``q [rows, cols rounded up to 128]`` (``torch.float8_e4m3fn``, zeros behind the last column) and ``scale`` (``torch.uint8``, one
    dimension), a byte for ``2 ** (byte - 127)``.  Those lie in tiles of 512 bytes for 128 rows and 4 blocks, as the tensor cores read them (``scales`` gives
    them as a matrix)."""
    q: torch.Tensor
    scale: torch.Tensor
    cols: int


def __getattr__(name: str):
    if name == "launch_count":               # kernels launched by this module
        return _native.launches(_native.FP8)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def check_status() -> None:
    """Raises if a CTA of a product gave up on one of its bounded waits since the last call."""
    st = lib.tmpi_gemm_status()
    if st:
        raise TorchMPIError(3, f"products in 8 bits: a bounded wait ran out (code {st})")


# ---------------------------------------------------------------- PyTorch forms
def _extents(rows: int, cols: int) -> Tuple[int, int, int]:
    blocks = -(-cols // BLOCK)
    return -(-rows // 128), blocks, -(-blocks // 4)


def _tiled(bytes_: torch.Tensor) -> torch.Tensor:
    """``[rows, blocks]`` -> the scales of a ``Block8``."""
    rows, blocks = bytes_.shape
    tiles, _, groups = _extents(rows, blocks * BLOCK)
    full = F.pad(bytes_, (0, groups * 4 - blocks, 0, tiles * 128 - rows), value=1)
    return full.view(tiles, 4, 32, groups, 4).permute(0, 3, 2, 1, 4).reshape(-1)          # row = 32 i + j: j, i, block


def scales(a: Block8) -> torch.Tensor:
    """The bytes of a matrix' scales as ``[rows, blocks]``."""
    _checked("scales", a)
    tiles, blocks, groups = _extents(a.q.shape[0], a.cols)
    return a.scale.view(tiles, groups, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles * 128, groups * 4)[: a.q.shape[0], :blocks].contiguous()


def _quantize(x: torch.Tensor) -> Block8:
    rows, cols = x.shape
    b = F.pad(x.float(), (0, -cols % BLOCK)).view(rows, -(-cols // BLOCK), BLOCK)
    finite = torch.isfinite(b)
    a = torch.where(finite, b.abs(), 0).amax(-1, keepdim=True)
    m, e = torch.frexp(a)                                          # a = m 2^e, 1/2 <= m < 1
    e = torch.where(a > 0, torch.where(m > 0.875, e - 8, e - 9), -126).clamp_min(-126)
    half = torch.div(-e, 2, rounding_mode="floor")                 # 2^126 * 2^-e in two exact steps
    q = torch.where(finite, b * _two_to(half) * _two_to(-e - half), float("nan")).to(torch.float8_e4m3fn)
    return Block8(q.view(rows, b.shape[1] * BLOCK), _tiled((e + 127).to(torch.uint8).view(rows, b.shape[1])), cols)


def _dequantize(a: Block8, dtype: torch.dtype) -> torch.Tensor:
    two = (scales(a).int() << 23).view(torch.float32).unsqueeze(-1)
    return (a.q.float().unflatten(-1, (-1, BLOCK)) * two).flatten(-2)[:, : a.cols].to(dtype)


def _checked(what: str, *matrices: Block8) -> None:
    for a in matrices:
        q, scale, cols = a
        if q.dtype != torch.float8_e4m3fn or scale.dtype != torch.uint8 or q.dim() != 2 or scale.dim() != 1:
            raise ValueError(f"{what}: a matrix in 8 bits is float8_e4m3fn [rows, pitch] with uint8 scales in one dimension, not {q.dtype} {tuple(q.shape)} and {scale.dtype} {tuple(scale.shape)}")
        tiles, blocks, groups = _extents(q.shape[0], cols)
        if cols < 1 or q.shape[1] != blocks * BLOCK or scale.shape[0] != tiles * groups * 512:
            raise ValueError(f"{what}: {tuple(q.shape)} numbers and {scale.shape[0]} bytes of scales are no matrix of {cols} columns")


def _matrix(what: str, x: torch.Tensor) -> torch.Tensor:
    if x.dim() < 1 or not x.dtype.is_floating_point or x.shape[-1] < 1:
        raise ValueError(f"{what} expects a floating tensor [..., C], got {x.dtype} {tuple(x.shape)}")
    return x.detach() if x.dim() == 2 else x.detach().reshape(-1, x.shape[-1])


# ---------------------------------------------------------------- entry points
def quantize(x: torch.Tensor) -> Block8:
    """The rows of ``x [..., C]`` in 8 bits (of 64 bits: of their values in 32); not differentiable."""
    if x.is_cuda:
        kept = _native.ext().fp8_quantize(x, True, False)          # None: nothing for the kernel
        if kept is not None:
            return Block8(*kept, x.shape[-1])
    x2 = _matrix("quantize", x)
    same_device("quantize", x2)
    return _quantize(x2)


def quantize_columns(x: torch.Tensor) -> Block8:
    """The columns of ``x [..., C]``: ``quantize(x.reshape(-1, C).T)``."""
    if x.is_cuda:
        kept = _native.ext().fp8_quantize(x, False, True)
        if kept is not None:
            return Block8(*kept, x.numel() // x.shape[-1])
    x2 = _matrix("quantize_columns", x)
    if not x2.shape[0]:
        raise ValueError("quantize_columns: there are no rows")
    same_device("quantize_columns", x2)
    return _quantize(x2.t())


def quantize_both(x: torch.Tensor) -> Tuple[Block8, Block8]:
    """``(quantize(x), quantize_columns(x))``, reading ``x`` once."""
    if x.is_cuda:
        kept = _native.ext().fp8_quantize(x, True, True)
        if kept is not None:
            return Block8(kept[0], kept[1], x.shape[-1]), Block8(kept[2], kept[3], x.numel() // x.shape[-1])
    x2 = _matrix("quantize_both", x)
    if not x2.shape[0]:
        raise ValueError("quantize_both: there are no rows")
    same_device("quantize_both", x2)
    return _quantize(x2), _quantize(x2.t())


def dequantize(a: Block8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """What the matrix stands for, ``[rows, cols]``, rounded to ``dtype`` (exact in bf16 and fp32 within their range)."""
    if a.q.is_cuda:
        x = _native.ext().fp8_restore(a.q, a.scale, a.cols, DTYPES.get(dtype, -1))
        if x is not None:
            return x
    _checked("dequantize", a)
    same_device("dequantize", a.q, a.scale)
    if not dtype.is_floating_point:
        raise ValueError(f"dequantize: {dtype} is not a floating type")
    return _dequantize(a, dtype)


def matmul(a: Block8, b: Block8, bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ b.T (+ bias)`` for ``a [M, K]`` and ``b [N, K]`` in 8 bits, summed in fp32 and rounded once to ``dtype``, which the bias has too; not differentiable."""
    if a.q.is_cuda and a.cols == b.cols:
        c = _native.ext().fp8_matmul(a.q, a.scale, b.q, b.scale, a.cols, bias, DTYPES.get(dtype, -1))
        if c is not None:
            return c
    _checked("matmul", a, b)
    if a.cols != b.cols or not dtype.is_floating_point or (bias is not None and (bias.shape != b.q.shape[:1] or bias.dtype != dtype)):
        raise ValueError(f"matmul expects a [M, K], b [N, K] and a bias [N] of the result's floating type, got {a.cols} and {b.cols} columns, {dtype}")
    same_device("matmul", a.q, a.scale, b.q, b.scale, bias)
    wide = torch.promote_types(dtype, torch.float32)
    return F.linear(_dequantize(a, wide), _dequantize(b, wide), None if bias is None else bias.detach().to(wide)).to(dtype)


class _Linear(torch.autograd.Function):
    """The layer on PyTorch operations."""

    @staticmethod
    def forward(ctx, x, w, bias, gelu):
        wide = torch.promote_types(x.dtype, torch.float32)
        q = lambda t: _dequantize(_quantize(t), wide)      # noqa: E731
        z = F.linear(q(x), q(w), None if bias is None else bias.to(wide)).to(x.dtype)
        ctx.save_for_backward(x, w, z if gelu else None)
        ctx.bias = bias is not None
        return _gelu_parts(z.to(wide))[0].to(x.dtype) if gelu else z

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("products in 8 bits can be differentiated once (no create_graph)")
        x, w, z = ctx.saved_tensors
        wide = torch.promote_types(x.dtype, torch.float32)
        q = lambda t: _dequantize(_quantize(t), wide) if t.numel() else t.to(wide)      # noqa: E731
        dz = dy if z is None else (dy.to(wide) * _gelu_parts(z.to(wide))[1]).to(dy.dtype)
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = (q(dz) @ q(w.t()).t()).to(x.dtype)
        if ctx.needs_input_grad[1]:
            dw = (q(dz.t()) @ q(x.t()).t()).to(w.dtype)
        if ctx.bias and ctx.needs_input_grad[2]:
            db = dz.to(wide).sum(0).to(dy.dtype)
        return dx, dw, db, None


def linear(x: torch.Tensor, w: Union[torch.Tensor, Block8], bias: Optional[torch.Tensor] = None, gelu: bool = False) -> torch.Tensor:
    """``x @ w.T (+ bias)``, with ``gelu`` the GELU of it, for ``x [..., K]``, ``w [N, K]``, ``bias [N]`` of one floating type, through products in 8 bits (see
    the module).  ``w`` may be a ``Block8``: then nothing may ask for a gradient."""
    if isinstance(w, Block8):
        if x.is_cuda and x.dim() >= 1:
            y = _native.ext().fp8_linear_kept(x, w.q, w.scale, w.cols, bias, gelu)
            if y is not None:
                return y
        _checked("linear", w)
        if x.dim() < 1 or x.shape[-1] != w.cols or not x.dtype.is_floating_point or (bias is not None and (bias.shape != w.q.shape[:1] or bias.dtype != x.dtype)):
            raise ValueError(f"linear expects x [..., {w.cols}] and a bias [{w.q.shape[0]}] of its type, got {x.dtype} {tuple(x.shape)}")
        if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
            raise ValueError("linear: weights kept in 8 bits have no backward pass (use the tensor, or torch.no_grad())")
        if any(t is not None and fwd.unpack_dual(t).tangent is not None for t in (x, bias)):
            raise ValueError("linear: the derivative of products in 8 bits is formed backward, not forward")
        same_device("linear", x, w.q, w.scale, bias)
        wide = torch.promote_types(x.dtype, torch.float32)
        z = F.linear(_dequantize(_quantize(x.reshape(-1, w.cols)), wide), _dequantize(w, wide), None if bias is None else bias.to(wide)).to(x.dtype)
        z = _gelu_parts(_wide(z))[0].to(x.dtype) if gelu else z
        return z.view(x.shape[:-1] + z.shape[1:])
    if x.is_cuda and x.dim() >= 1:
        y = _native.ext().fp8_linear(x, w, bias, gelu)
        if y is not None:
            return y
    if not (x.dim() >= 1 and w.dim() == 2 and w.shape[1] >= 1 and x.shape[-1] == w.shape[1] and (bias is None or bias.shape == w.shape[:1])):
        raise ValueError("linear expects x [..., K], w [N, K] and bias [N]")
    tensors = [t for t in (x, w, bias) if t is not None]
    if len({t.dtype for t in tensors}) > 1 or not x.dtype.is_floating_point:
        raise ValueError(f"linear: tensors of one floating dtype are expected, got {sorted({str(t.dtype) for t in tensors})}")
    same_device("linear", *tensors)
    y = _Linear.apply(x.reshape(-1, x.shape[-1]), w, bias, gelu)
    return y.view(x.shape[:-1] + w.shape[:1])
