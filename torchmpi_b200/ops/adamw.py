"""AdamW over many tensors at once, with states in 32 or 8 bits, and the norm of many gradients (csrc/kernels/adamw.cu, csrc/bindings/adamw.cpp).

``AdamW(params, lr, ...).step()`` updates all parameters that have a gradient, in one launch for up to 980 tensors of a type:

    g = gradient * grad_scale * min(1, max_norm / (norm + 1e-6));   m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
    w = (1 - lr * weight_decay) w - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

in fp32 (an element that never had a gradient stays, also with ``eps = 0``; with 8 bits ``eps`` counts as 1e-18 at least).  Parameters of 16 bits have fp32 masters (``master_weights=True``) that the step goes by and whose rounding the parameter becomes; without, the
parameter itself is updated and rounded.  A gradient of another type than its parameter's (``grad_dtype``) counts as it is, at the price of a copy.  ``bits=8`` keeps ``m`` and the root of ``v`` as a byte an element with an fp32 scale for 128 (2.06 bytes an element
in the place of the 8 of 32 bits, to read and to write): ``m = sign(c) c^2 top / 127^2``, ``sqrt(v) = c^2 top / 255^2``, where ``top`` is the block's
largest magnitude; a root that is not zero never becomes zero.  An average that changes by less than half a code in a step, its block's largest
standing still, keeps its code.  A block with an element that is not finite becomes NaN.

Step counts and the clipping coefficient lie on the device and nothing waits for it, so that a step can be captured into a graph; a
replay takes the learning rates of the capture, unless they are fp32 tensors on the device.  Elements are independent and the norm is summed in a fixed order:
results are bit-reproducible.  Parameters on the CPU take the same arithmetic in PyTorch.  The reference has SGD alone.
"""
from __future__ import annotations

import math
from typing import Dict, Iterable, List, Optional, Sequence, Tuple, Union

import torch
import torch.nn.functional as F

from .. import _native
from .._lib import DTYPES

BLOCK = 128         # elements of 8-bit states that share a scale
_LEAST = 2.0 ** -100
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def __getattr__(name: str):
    if name == "launch_count":               # kernels launched by this module
        return _native.launches(_native.ADAMW)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


# ---------------------------------------------------------------- 8-bit states on PyTorch operations
def _keep_m(m: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    top = m.abs().amax(1)
    top = torch.where(torch.isfinite(top), top, math.nan)
    code = 127 * torch.sqrt(m.abs() / top.clamp_min(_LEAST).unsqueeze(1))
    return torch.copysign(torch.round(code), m).nan_to_num(0).to(torch.int8), top


def _value_m(code: torch.Tensor, top: torch.Tensor) -> torch.Tensor:
    c = code.float()
    return c * c.abs() * (top * (1 / 16129)).unsqueeze(1)


def _keep_v(v: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    r = torch.sqrt(v)
    top = r.amax(1)
    top = torch.where(torch.isfinite(top), top, math.nan)
    code = torch.round(255 * torch.sqrt(r / top.clamp_min(_LEAST).unsqueeze(1)))
    return torch.where(r > 0, code.clamp_min(1), 0).nan_to_num(0).to(torch.uint8), top


def _value_v(code: torch.Tensor, top: torch.Tensor) -> torch.Tensor:
    c = code.float()
    return (c * c * (top * (1 / 65025)).unsqueeze(1)).square()


def grad_norm(tensors: Iterable[torch.Tensor]) -> torch.Tensor:
    """The 2-norm of all tensors together, a 0-dimensional fp32 tensor on their device (of 64 bits: fp64); nothing waits for it.  On the GPU squares are formed in fp32: elements
    beyond 1e19 make the norm infinite (a clipped step then takes its gradients for zero), and those below 1e-23 count as zero in it."""
    tensors = [t.detach() for t in tensors]
    if not tensors:
        return torch.zeros(())
    if any(not t.dtype.is_floating_point for t in tensors) or len({t.device for t in tensors}) > 1:
        raise ValueError("grad_norm expects floating tensors on one device")
    if tensors[0].is_cuda:
        n = _native.ext().grad_norm(tensors)          # None: nothing for the kernel
        if n is not None:
            return n
    total = sum(t.double().square().sum() for t in tensors)
    return total.sqrt().to(torch.promote_types(torch.float32, max((t.dtype for t in tensors), key=lambda d: d.itemsize)))


def _is_dense(p: torch.Tensor) -> bool:
    """Whether the elements fill their storage without gaps, in whatever order."""
    expected = 1
    for size, stride in sorted(((s, t) for s, t in zip(p.shape, p.stride()) if s != 1), key=lambda x: (x[1], x[0])):
        if stride != expected:
            return False
        expected *= size
    return True


class AdamW:
    """``params``: tensors, or groups of them (``{"params": ..., "lr": ..., "betas": ..., "eps": ..., "weight_decay": ...}``, up to 8) as ``param_groups`` holds
    them then; their options may be changed between steps, ``lr`` may be a 0-dimensional fp32 tensor on the device.  ``max_norm``: gradients are scaled down to
    that norm of all of them together, which ``grad_norm`` holds after a step (times ``grad_scale``).  ``state[p]`` holds views of a parameter's states: ``step`` (int32), ``master``
    (where it has one), and ``exp_avg`` and ``exp_avg_sq``, of the parameter's shape in 32 bits; in 8 the codes ``[blocks, 128]`` (int8, and uint8 of
    the second moment's root), with ``exp_avg_scale`` and ``exp_avg_sq_scale``."""

    def __init__(self, params: Union[Iterable[torch.Tensor], Iterable[dict]], lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, bits: int = 32, master_weights: bool = True, max_norm: Optional[float] = None, grad_scale: float = 1.0):
        if bits not in (8, 32):
            raise ValueError(f"AdamW: states have 8 or 32 bits, not {bits}")
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"AdamW: max_norm = {max_norm}")
        self.bits, self.max_norm, self.grad_scale = bits, max_norm, grad_scale
        groups = list(params)
        if not groups:
            raise ValueError("AdamW: no parameters")
        if not isinstance(groups[0], dict):
            groups = [{"params": groups}]
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        self.param_groups: List[dict] = []
        for g in groups:
            extra = set(g) - {"params", *defaults}
            if extra:
                raise ValueError(f"AdamW: unknown options {sorted(extra)}")
            ps = g["params"]
            self.param_groups.append({**defaults, **g, "params": [ps] if isinstance(ps, torch.Tensor) else list(ps)})
        if len(self.param_groups) > 8:
            raise ValueError(f"AdamW: {len(self.param_groups)} groups of parameters, up to 8 are taken")
        self._options()
        self._params: List[torch.Tensor] = [p for g in self.param_groups for p in g["params"]]
        self._made = [(p.dtype, p.shape, self._order(p)) for p in self._params]          # the states' order
        group = [i for i, g in enumerate(self.param_groups) for _ in g["params"]]
        if not self._params or len({id(p) for p in self._params}) < len(self._params):
            raise ValueError("AdamW: no parameters, or one of them twice")
        device = self._params[0].device
        for p in self._params:
            if p.dtype not in _TYPES or p.device != device or not p.is_leaf:
                raise ValueError(f"AdamW: parameters are leaves of bf16, fp16 or fp32 on one device, got {p.dtype} on {p.device}")
            if not _is_dense(p):
                raise ValueError(f"AdamW: a parameter {tuple(p.shape)} with strides {p.stride()} does not fill its storage")
        if device.type == "cuda" and device.index != torch.cuda.current_device():
            raise ValueError(f"AdamW: parameters on {device}, but the current device is cuda:{torch.cuda.current_device()}")
        self._places = [0]
        for p in self._params:
            self._places.append(self._places[-1] + -(-p.numel() // BLOCK) * BLOCK)
        total, count = self._places[-1], len(self._params)
        zeros = lambda n, dtype: torch.zeros(n, dtype=dtype, device=device)      # noqa: E731
        self._m = zeros(total, torch.float32) if bits == 32 else zeros(total, torch.int8)
        self._v = zeros(total, torch.float32) if bits == 32 else zeros(total, torch.uint8)
        self._m_top, self._v_top = (None, None) if bits == 32 else (zeros(total // BLOCK, torch.float32), zeros(total // BLOCK, torch.float32))
        self._master = zeros(total, torch.float32) if master_weights and any(p.dtype != torch.float32 for p in self._params) else None
        self._steps, self._counter, self._norm = zeros(count, torch.int32), zeros(1, torch.int32), zeros((), torch.float32)
        self.state: Dict[torch.Tensor, Dict[str, torch.Tensor]] = {}
        for i, p in enumerate(self._params):
            a, b = self._places[i], self._places[i + 1]
            like = lambda flat: flat[a: a + p.numel()].as_strided(p.shape, p.stride())      # noqa: B023, E731
            st = {"step": self._steps[i]}
            if bits == 32:
                st["exp_avg"], st["exp_avg_sq"] = like(self._m), like(self._v)
            else:
                blocks = slice(a // BLOCK, b // BLOCK)
                st["exp_avg"], st["exp_avg_scale"] = self._m[a:b].view(-1, BLOCK), self._m_top[blocks]
                st["exp_avg_sq"], st["exp_avg_sq_scale"] = self._v[a:b].view(-1, BLOCK), self._v_top[blocks]
            if self._has_master(p):
                st["master"] = like(self._master)
            self.state[p] = st
        self.refresh_master()
        self._native = None
        if device.type == "cuda":
            self._native = _native.ext().AdamW(self._params, self._places[:-1], group, self._m, self._v, self._m_top, self._v_top, self._master, self._steps, self._counter, self._norm, bits)

    @staticmethod
    def _order(p: torch.Tensor) -> List[int]:
        return [t for s, t in zip(p.shape, p.stride()) if s != 1]

    def _has_master(self, p: torch.Tensor) -> bool:
        return self._master is not None and p.dtype != torch.float32

    def _options(self, groups: Optional[Sequence[dict]] = None):
        options, rates = [], []
        for g in self.param_groups if groups is None else groups:
            lr, (b1, b2), eps, decay = g["lr"], g["betas"], g["eps"], g["weight_decay"]
            on_device = isinstance(lr, torch.Tensor)
            if not (0 <= b1 < 1 and 0 <= b2 < 1 and eps >= 0 and decay >= 0 and (on_device or lr >= 0)):
                raise ValueError(f"AdamW: lr = {lr}, betas = {(b1, b2)}, eps = {eps}, weight_decay = {decay}")
            options.append((0.0 if on_device else lr, b1, b2, eps, decay))
            rates.append(lr if on_device else None)
        return options, rates

    def refresh_master(self) -> None:
        """Copies the parameters into their fp32 masters (after they were loaded or broadcast)."""
        with torch.no_grad():
            for p in self._params:
                if self._has_master(p):
                    self.state[p]["master"].copy_(p)

    def synchronize(self, root: int = 0) -> None:
        """Collective: makes every rank hold rank ``root``'s averages, step counts and masters, as the replicas of a model hold its parameters."""
        from ..collectives import broadcast_tensor
        for flat in (self._m, self._v, self._m_top, self._v_top, self._master, self._steps):
            if flat is not None and flat.numel():
                broadcast_tensor(root, flat)

    # ---- one step
    def step(self, lr: Optional[Union[float, torch.Tensor]] = None) -> None:
        """``lr``: the learning rate of all groups from now on, in the place of rates of their own and of tensors on the device."""
        options, rates = self._options(None if lr is None else [{**g, "lr": lr} for g in self.param_groups])
        if self._native is not None:
            self._native.step(options, rates, self.max_norm, self.grad_scale)
        else:
            self._step(options, rates)
        if lr is not None:                       # not by a step that was refused
            for g in self.param_groups:
                g["lr"] = lr

    @torch.no_grad()
    def _step(self, options, rates) -> None:
        for p, made in zip(self._params, self._made):          # all of them before anything changes
            if p.grad is None:
                continue
            if (p.dtype, p.shape, self._order(p)) != made:
                raise ValueError(f"AdamW: a parameter has changed: {p.dtype} {tuple(p.shape)} with strides {p.stride()}")
            if p.grad.is_sparse or p.grad.shape != p.shape:
                raise ValueError(f"AdamW: a gradient that is not its parameter's: {tuple(p.grad.shape)}")
        scale = self.grad_scale
        if self.max_norm is not None:
            grads = [p.grad for p in self._params if p.grad is not None]
            self._norm.copy_(abs(scale) * grad_norm(grads) if grads else torch.zeros(()))
            scale = scale * torch.clamp_max(self.max_norm / (self._norm + 1e-6), 1)
        which = [i for i, g in enumerate(self.param_groups) for _ in g["params"]]
        for p, i in zip(self._params, which):
            if p.grad is None or not p.numel():
                continue
            st, (rate, b1, b2, eps, decay) = self.state[p], options[i]
            rate = float(rate if rates[i] is None else rates[i])
            st["step"] += 1
            t = int(st["step"])
            w = st["master"] if "master" in st else p.float()
            m, v = self.moments(p)
            g = p.grad.float() * scale
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
            w = (1 - rate * decay) * w - rate / (1 - b1 ** t) * m / (torch.sqrt(v) / math.sqrt(1 - b2 ** t) + max(eps, 1e-37 if self.bits == 32 else 1e-18))
            if "master" in st:
                st["master"].copy_(w)
            p.copy_(w)
            if self.bits == 32:
                st["exp_avg"].copy_(m)
                st["exp_avg_sq"].copy_(v)
            else:
                for name, x, keep in (("exp_avg", m, _keep_m), ("exp_avg_sq", v, _keep_v)):
                    flat = torch.empty_strided(p.shape, p.stride()).copy_(x).as_strided((p.numel(),), (1,))
                    code, top = keep(F.pad(flat, (0, -p.numel() % BLOCK)).view(-1, BLOCK))
                    st[name].copy_(code)
                    st[name + "_scale"].copy_(top)

    def zero_grad(self, set_to_none: bool = True) -> None:
        for p in self._params:
            if p.grad is not None:
                if set_to_none:
                    p.grad = None
                else:
                    p.grad.detach_().zero_()

    @property
    def grad_norm(self) -> torch.Tensor:
        """The norm of the last step's gradients (0-dimensional, on the device; of ``max_norm`` alone)."""
        return self._norm

    # ---- what the states stand for
    def moments(self, p: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """The averages of the gradient and of its square: those of parameter ``p`` in fp32 and its shape, or without one all of them, each parameter's from the next multiple of
        128 on, in the order of the groups.  Of 8-bit states copies (all of them: in ``dtype``, bf16 if not given)."""
        if p is None:
            if self.bits == 32:
                return (self._m, self._v) if dtype is None else (self._m.to(dtype), self._v.to(dtype))
            dtype = torch.bfloat16 if dtype is None else dtype
            if self._native is not None and dtype in _TYPES:
                return _native.ext().adamw_values(self._m, self._m_top, self._v, self._v_top, DTYPES[dtype])
            return (_value_m(self._m.view(-1, BLOCK), self._m_top).view(-1).to(dtype), _value_v(self._v.view(-1, BLOCK), self._v_top).view(-1).to(dtype))
        st = self.state[p]
        if self.bits == 32:
            return st["exp_avg"], st["exp_avg_sq"]
        like = lambda flat: flat.view(-1)[: p.numel()].as_strided(p.shape, p.stride())      # noqa: E731
        return like(_value_m(st["exp_avg"], st["exp_avg_scale"])), like(_value_v(st["exp_avg_sq"], st["exp_avg_sq_scale"]))

    def masters(self) -> Optional[torch.Tensor]:
        """All fp32 masters, laid out as ``moments()``; None where there are none."""
        return self._master

    # ---- checkpointing
    def state_dict(self) -> dict:
        """Options of the groups, and for each parameter its states and, as ``layout``, its shape and order (the strides of its dimensions), in the order of the groups (copies)."""
        options = [{k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in g.items() if k != "params"} for g in self.param_groups]
        layout = [[list(shape), order] for _, shape, order in self._made]
        return {"bits": self.bits, "param_groups": options, "layout": layout, "state": [{k: v.clone() for k, v in self.state[p].items()} for p in self._params]}

    def load_state_dict(self, state: dict) -> None:
        """Loads a ``state_dict`` of an optimizer of the same parameters, number of bits and masters; anything else raises, and nothing has changed then.  Codes of 8 bits are
        those of parameters of the same order, too.  A learning rate that is a tensor here stays that tensor and takes the saved value."""
        saved: Sequence[dict] = state["state"]
        if state["bits"] != self.bits or len(saved) != len(self._params) or len(state["param_groups"]) != len(self.param_groups):
            raise ValueError(f"AdamW: states of {state['bits']} bits for {len(saved)} parameters, not {self.bits} bits for {len(self._params)}")
        for p, st in zip(self._params, saved):
            mine = self.state[p]
            if set(st) != set(mine) or any(st[k].shape != mine[k].shape or st[k].dtype != mine[k].dtype for k in mine):
                raise ValueError("AdamW: a parameter's states are not those of this optimizer's")
        if self.bits == 8 and "layout" in state:
            for (_, shape, order), (saved_shape, saved_order) in zip(self._made, state["layout"]):
                if list(shape) != list(saved_shape) or order != list(saved_order):
                    raise ValueError(f"AdamW: 8-bit states of a parameter {list(saved_shape)} in the order of strides {list(saved_order)}, not {list(shape)} and {order}")
        for g, options in zip(self.param_groups, state["param_groups"]):
            own = {k: options.get(k, g[k]) for k in ("lr", "betas", "eps", "weight_decay")}          # others are the program's
            if any(isinstance(v, torch.Tensor) and (k != "lr" or v.numel() != 1) for k, v in own.items()) or not isinstance(own["betas"], (tuple, list)):
                raise ValueError(f"AdamW: a group's options are none: {own}")
            self._options([own])
        with torch.no_grad():
            for g, options in zip(self.param_groups, state["param_groups"]):
                for k, v in options.items():
                    if k == "lr" and isinstance(g[k], torch.Tensor):
                        g[k].copy_(torch.as_tensor(v).reshape(g[k].shape))                # where a captured step reads it
                    elif k == "lr" and isinstance(v, torch.Tensor):
                        g[k] = v.to(self._steps.device, torch.float32, copy=True)
                    elif k != "params":
                        g[k] = v.clone() if isinstance(v, torch.Tensor) else v
            for p, st in zip(self._params, saved):
                for k, v in self.state[p].items():
                    v.copy_(st[k])
