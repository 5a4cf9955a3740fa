"""Layers of experts (csrc/kernels/route.cu, experts.cu, grouped.cu; autograd in csrc/bindings/experts.cpp).

``route(logits, k)`` chooses ``k`` experts for each token and puts all choices in the order of the experts; ``mlp(x, routing,
w1, b1, w2, b2)`` sends the tokens through the chosen experts' MLPs and adds what comes back; ``Experts`` is the module, gate
included.  The parts can be had one by one: ``dispatch`` (rows to their experts' places), ``grouped_linear`` (a linear
layer with a weight for each group of rows) and ``combine`` (the weighted sum of a token's rows).  All are differentiable.

The sizes of the groups stay on the device: no call waits for the GPU, so a step can be captured into a graph and replayed with other
logits.  Every result is bit-reproducible (nothing is summed by atomics).  What the kernels do not take (CPU, products in
other dtypes than bf16 or with widths that are not multiples of 8, more than 256 experts or 32 for a token) runs on
PyTorch operations, some of which wait for the sizes.  The reference has no such layer (its models are MNIST networks).
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import _native
from .._lib import lib, TorchMPIError
from . import act8 as _act8
from .act8 import _wide, same_device


class Routing(NamedTuple):
    """``weights [T, k]`` (fp32, differentiable), ``chosen [T, k]`` (experts, -1: none), ``order [T * k]`` (the entry ``t * k + j`` at each
    place, -1 behind the last), ``place [T, k]`` (the place of each entry, -1: none), ``offsets [E + 1]`` (expert ``e`` has the
    places from ``offsets[e]`` to ``offsets[e + 1]``); the last four int32."""
    weights: torch.Tensor
    chosen: torch.Tensor
    order: torch.Tensor
    place: torch.Tensor
    offsets: torch.Tensor


def __getattr__(name: str):
    if name == "launch_count":               # kernels launched by this module
        return _native.launches(_native.EXPERTS)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def check_status() -> None:
    """Raises if a CTA of a grouped product gave up on one of its bounded waits since the last call."""
    st = lib.tmpi_gemm_status()
    if st:
        raise TorchMPIError(3, f"grouped products: a bounded wait ran out (code {st})")


# ---------------------------------------------------------------- PyTorch forms
def _route(logits: torch.Tensor, k: int, renormalize: bool) -> Routing:
    l = _wide(logits)
    T, E = l.shape
    nan = torch.isnan(l)
    bad = nan.any(1, keepdim=True)
    usable = torch.where(nan, -math.inf, l)
    key, index = torch.sort(usable, dim=1, descending=True, stable=True)
    key, index = key[:, :k], index[:, :k]
    used = key > -math.inf
    top = torch.where(used[:, :1], key[:, :1], 0).detach()
    scores = torch.where(used, torch.exp(torch.gather(usable, 1, index) - top), 0)
    total = scores.sum(1, keepdim=True) if renormalize else torch.exp(usable - top).sum(1, keepdim=True)
    weights = torch.where(used, scores / torch.where(used[:, :1], total, 1), 0)
    # a token with a NaN: its weights are NaN, and so are the gradients of the logits that enter them, the chosen ones or all
    one, zero = torch.ones_like(l[:, :1]), torch.zeros_like(l[:, :1])
    poison = torch.where(bad, math.nan, one) if renormalize else torch.where(bad, (l * torch.where(bad, math.nan, zero)).sum(1, keepdim=True), one)
    weights = (weights * poison).float()
    expert, order = torch.sort(torch.where(used, index, E).reshape(-1), stable=True)
    slot = torch.arange(T * k, device=l.device)
    place = torch.empty_like(slot)
    place[order] = torch.where(expert < E, slot, -1)
    offsets = torch.searchsorted(expert, torch.arange(E + 1, device=l.device))
    return Routing(weights, torch.where(used, index, -1).int(), torch.where(expert < E, order, -1).int(), place.view(T, k).int(), offsets.int())


def _combine(rows, weights, place):
    at = place.long()
    picked = torch.where((at >= 0).unsqueeze(2), _wide(rows)[at.clamp_min(0)], 0)
    return (picked * weights.unsqueeze(2)).sum(1).to(rows.dtype)


def _dispatch(x, order, k):
    token = torch.div(order.long(), k, rounding_mode="floor")
    wide = _wide(x)          # so that the gradients of a token's rows are added in fp32
    return torch.where((token >= 0).unsqueeze(1), wide[token.clamp_min(0)], 0).to(x.dtype)


def _groups(offsets, rows):
    ends = offsets.tolist()
    if ends != sorted(ends) or ends[0] != 0 or ends[-1] > rows:
        raise ValueError(f"offsets of groups ascend from 0 to at most the number of rows, {rows}")
    return [(e, a, b) for e, (a, b) in enumerate(zip(ends[:-1], ends[1:])) if b > a]


def _grouped(x, w, bias, offsets, gelu):
    parts, at = [F.linear(x[:0], w[0], None if bias is None else bias[0])], 0      # no row, but gradients where there are no groups
    for e, a, b in _groups(offsets, x.shape[0]):
        y = F.linear(_wide(x[a:b]), _wide(w[e]), None if bias is None else _wide(bias[e]))
        parts.append((F.gelu(y) if gelu else y).to(x.dtype))
        at = b
    if at < x.shape[0]:
        parts.append(x.new_zeros(x.shape[0] - at, w.shape[1]))
    return torch.cat(parts)


class _Mlp8(torch.autograd.Function):
    """The experts' MLPs with 8-bit checkpoints, on PyTorch operations."""

    @staticmethod
    def forward(ctx, x, weights, w1, b1, w2, b2, order, place, offsets):
        k, xs = place.shape[1], _dispatch(_wide(x), order, place.shape[1])
        z, ys = xs.new_zeros(xs.shape[0], w1.shape[1]), torch.zeros_like(xs)
        for e, a, b in _groups(offsets, xs.shape[0]):
            z[a:b] = F.linear(xs[a:b], _wide(w1[e]), None if b1 is None else _wide(b1[e]))
            ys[a:b] = F.linear(_act8._gelu_parts(z[a:b])[0], _wide(w2[e]), None if b2 is None else _wide(b2[e]))
        ctx.save_for_backward(*_act8._quantize(x), *_act8._quantize(z), weights, w1, b1, w2, b2, order, place, offsets)
        return _combine(ys, weights, place).to(x.dtype)

    @staticmethod
    def backward(ctx, dy):
        _act8.refuse_graph()
        xq, xs, zq, zs, weights, w1, b1, w2, b2, order, place, offsets = ctx.saved_tensors
        k, n = place.shape[1], order.shape[0]
        g = _dispatch(_wide(dy), order, k)
        x, z = _act8._dequantize(_act8.Act8(xq, xs), g.dtype), _act8._dequantize(_act8.Act8(zq, zs), g.dtype)
        x = _dispatch(x, order, k)
        wt = weights.reshape(-1)[order.long().clamp_min(0)].unsqueeze(1)
        h, slope = _act8._gelu_parts(z)
        dxs, dwe = torch.zeros_like(g), g.new_zeros(n)
        dw1, db1, dw2, db2 = (None if t is None else torch.zeros_like(t, dtype=g.dtype) for t in (w1, b1, w2, b2))
        for e, a, b in _groups(offsets, n):
            dh = g[a:b] @ _wide(w2[e])
            dwe[a:b] = (dh * h[a:b]).sum(1)
            dz, gw = wt[a:b] * dh * slope[a:b], wt[a:b] * g[a:b]
            dw2[e], dw1[e], dxs[a:b] = gw.t() @ h[a:b], dz.t() @ x[a:b], dz @ _wide(w1[e])
            if b2 is not None:
                dwe[a:b] += (g[a:b] * _wide(b2[e])).sum(1)
                db2[e] = gw.sum(0)
            if b1 is not None:
                db1[e] = dz.sum(0)
        dweights = torch.where(place >= 0, dwe[place.long().clamp_min(0)], 0)
        dx = _combine(dxs, torch.ones_like(weights), place)
        grads = [t if t is None else t.to(w1.dtype) for t in (dw1, db1, dw2, db2)]
        return (dx.to(dy.dtype), dweights, *grads, None, None, None)


# ---------------------------------------------------------------- entry points
def route(logits: torch.Tensor, k: int, renormalize: bool = True) -> Routing:
    """The ``k`` largest of each token's ``logits [T, E]``, largest first, of equal ones that with the lowest index.  The weights are the softmax over
    the chosen logits, or (``renormalize=False``) over all of the token's.  An expert whose logit is -inf is never used, so a
    token may get fewer than ``k``, and one without any gets none (a padded position).  NaN is not chosen either, and makes the token's weights NaN,
    and in backward the gradients of the logits that the weights are formed from."""
    if logits.is_cuda:
        r = _native.ext().expert_route(logits, k, renormalize)          # None: nothing for the kernel
        if r is not None:
            return Routing(*r)
    if logits.dim() != 2 or not logits.dtype.is_floating_point or not 1 <= k <= logits.shape[1]:
        raise ValueError(f"route expects floating logits [T, E] and 1 <= k <= E, got {logits.dtype} {tuple(logits.shape)} and k = {k}")
    same_device("route", logits)
    return _route(logits, k, renormalize)


def _check_routing(what: str, r: Routing, tokens: Optional[int] = None) -> None:
    T, k = r.place.shape
    if any(t.dtype != torch.int32 for t in r[1:]) or r.weights.dtype != torch.float32 or r.weights.shape != (T, k) or r.chosen.shape != (T, k) \
            or r.order.shape != (T * k,) or r.offsets.dim() != 1 or r.offsets.shape[0] < 2:
        raise ValueError(f"{what}: not a routing as route() returns it")
    if tokens is not None and tokens != T:
        raise ValueError(f"{what}: {tokens} rows for a routing of {T} tokens")


def dispatch(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """``x [T, C]`` -> ``[T * k, C]``: the token's row at each place, zeros behind the last."""
    if x.is_cuda:
        rows = _native.ext().expert_dispatch(x, routing.place, routing.offsets)
        if rows is not None:
            return rows
    if x.dim() != 2 or not x.dtype.is_floating_point:
        raise ValueError(f"dispatch expects floating rows [T, C], got {x.dtype} {tuple(x.shape)}")
    _check_routing("dispatch", routing, x.shape[0])
    same_device("dispatch", x, routing.order, routing.place, routing.offsets)
    return _dispatch(x, routing.order, routing.place.shape[1])


def combine(rows: torch.Tensor, routing: Routing) -> torch.Tensor:
    """``rows [T * k, C]`` -> ``[T, C]``: each token's rows times their weights, added in fp32 (of 64 bits: in those) and rounded once."""
    if rows.is_cuda:
        y = _native.ext().expert_combine(rows, routing.weights, routing.place, routing.offsets)
        if y is not None:
            return y
    if rows.dim() != 2 or not rows.dtype.is_floating_point or rows.shape[0] != routing.order.shape[0]:
        raise ValueError(f"combine expects floating rows [T * k, C], got {rows.dtype} {tuple(rows.shape)}")
    _check_routing("combine", routing)
    same_device("combine", rows, *routing)
    return _combine(rows, routing.weights, routing.place)


def grouped_linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], offsets: torch.Tensor, gelu: bool = False) -> torch.Tensor:
    """``y[r] = gelu?(x[r] @ w[e].T + bias[e])`` for ``offsets[e] <= r < offsets[e + 1]``: ``x [R, K]``, ``w [E, N, K]``, ``bias [E, N]`` or None,
    ``offsets [E + 1]`` int32, ascending, with 0 first.  Groups may be empty; rows of ``x`` behind the last group give zeros and get no gradient.
    The kernel cannot refuse offsets that do not ascend (that would wait for the GPU): it stays inside the tensors, and its results mean nothing."""
    if x.is_cuda:
        y = _native.ext().grouped_linear(x, w, bias, offsets, gelu)
        if y is not None:
            return y
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[2] or (bias is not None and bias.shape != w.shape[:2]) \
            or offsets.shape != (w.shape[0] + 1,) or offsets.dtype != torch.int32 or w.shape[0] < 1:
        raise ValueError("grouped_linear expects x [R, K], w [E, N, K], bias [E, N] and int32 offsets [E + 1]")
    if not x.dtype.is_floating_point or w.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise ValueError(f"grouped_linear: tensors of one floating dtype are expected, got {x.dtype}, {w.dtype}")
    same_device("grouped_linear", x, w, bias, offsets)
    return _grouped(x, w, bias, offsets, gelu)


def mlp(x: torch.Tensor, routing: Routing, w1: torch.Tensor, b1: Optional[torch.Tensor], w2: torch.Tensor, b2: Optional[torch.Tensor],
        act8: bool = False) -> torch.Tensor:
    """The weighted sum over a token's experts of ``gelu(x @ w1[e].T + b1[e]) @ w2[e].T + b2[e]``: ``x [..., C]`` with the routing of its ``T`` rows,
    ``w1 [E, H, C]``, ``b1 [E, H]``, ``w2 [E, C, H]``, ``b2 [E, C]``.  Kept for backward are ``x`` and the pre-activations, with ``act8`` in 8 bits
    (``ops.act8``), and no dispatched rows; the backward pass forms everything else from those."""
    if x.is_cuda:
        y = _native.ext().expert_mlp(x, *routing, w1, b1, w2, b2, act8)
        if y is not None:
            return y
    if not (w1.dim() == 3 and w2.dim() == 3 and x.dim() >= 1 and x.shape[-1] == w1.shape[2] and w2.shape == (w1.shape[0], w1.shape[2], w1.shape[1])
            and (b1 is None or b1.shape == w1.shape[:2]) and (b2 is None or b2.shape == w2.shape[:2])):
        raise ValueError("mlp expects x [..., C], w1 [E, H, C], b1 [E, H], w2 [E, C, H] and b2 [E, C]")
    tensors = [t for t in (x, w1, b1, w2, b2) if t is not None]
    if len({t.dtype for t in tensors}) > 1 or not x.dtype.is_floating_point:
        raise ValueError(f"mlp: tensors of one floating dtype are expected, got {sorted({str(t.dtype) for t in tensors})}")
    x2 = x.reshape(-1, x.shape[-1])
    _check_routing("mlp", routing, x2.shape[0])
    if routing.offsets.shape[0] != w1.shape[0] + 1:
        raise ValueError(f"mlp: weights of {w1.shape[0]} experts for a routing to {routing.offsets.shape[0] - 1}")
    same_device("mlp", *tensors, *routing)
    if act8:
        y = _Mlp8.apply(x2, routing.weights, w1, b1, w2, b2, *routing[2:])
    else:
        h = grouped_linear(dispatch(x2, routing), w1, b1, routing.offsets, gelu=True)
        y = combine(grouped_linear(h, w2, b2, routing.offsets), routing)
    return y.view(x.shape)


class Experts(nn.Module):
    """A layer of ``experts`` MLPs ``width -> hidden -> width`` of which a gate chooses ``k`` for each token: the place of an MLP in a transformer
    block.  ``act8``: activations are kept in 8 bits.  ``last_offsets`` holds the last call's group bounds (for load statistics)."""

    def __init__(self, width: int, hidden: int, experts: int, k: int = 2, act8: bool = False, renormalize: bool = True):
        super().__init__()
        if not 1 <= k <= experts:
            raise ValueError(f"Experts: k = {k} of {experts}")
        self.k, self.act8, self.renormalize = k, act8, renormalize
        self.gate = nn.Linear(width, experts, bias=False)
        self.w1 = nn.Parameter(torch.empty(experts, hidden, width))
        self.b1 = nn.Parameter(torch.zeros(experts, hidden))
        self.w2 = nn.Parameter(torch.empty(experts, width, hidden))
        self.b2 = nn.Parameter(torch.zeros(experts, width))
        nn.init.normal_(self.w1, std=0.02)
        nn.init.normal_(self.w2, std=0.02)
        self.last_offsets: Optional[torch.Tensor] = None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        from . import gemm
        logits = gemm.linear(x.reshape(-1, x.shape[-1]), self.gate.weight)
        r = route(logits, self.k, self.renormalize)
        self.last_offsets = r.offsets
        return mlp(x, r, self.w1, self.b1, self.w2, self.b2, self.act8)
