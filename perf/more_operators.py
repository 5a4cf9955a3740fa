"""Products in 8-bit floating point with a scale for each block of 128, and AdamW over many tensors, as measurable cases.

Each case is one pass through an operator of ``torchmpi_b200.ops.fp8`` or ``torchmpi_b200.ops.adamw``: what a training or
generating program calls.  ``listed()`` gives the named cases, ``draw(rng)`` more of the same ranges, ``prepare`` the inputs,
weights and optimizer states that a program holds before the call, ``run`` the pass (with ``own`` through the package, else in
elementary operations in 32 bits), ``exact`` the same results in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 128         # elements that share a scale
LR, BETAS, EPS, DECAY, MAX_NORM, STEPS = 3e-4, (0.9, 0.99), 1e-8, 0.1, 1.0, 200
LEAST = 2.0 ** -100  # of the scales of 8-bit optimizer states


def listed():
    return [
        # the layer-norm output of a few tokens in 8 bits (latency counts); rows that end inside a block
        {"name": "quantize_few", "kind": "quantize", "rows": 48, "cols": 1000, "dtype": "fp32", "both": False},
        # the gradient of GPT-2 medium's hidden layer, 8 x 1024 tokens, as the operand of both products of a backward pass
        {"name": "quantize_gradient", "kind": "quantize", "rows": 8192, "cols": 4096, "dtype": "bf16", "both": True},
        # the up-projection of GPT-2 medium for one generated token, weights kept in 8 bits: bound by them and by latency
        {"name": "linear_token", "kind": "linear", "tokens": 1, "inp": 1024, "out": 4096, "gelu": True, "bias": True, "dtype": "bf16", "train": False},
        # the down-projection for a generating batch of 13
        {"name": "linear_batch", "kind": "linear", "tokens": 13, "inp": 4096, "out": 1024, "gelu": False, "bias": True, "dtype": "bf16", "train": False},
        # the up-projection of a prompt, an odd number of tokens
        {"name": "linear_prompt", "kind": "linear", "tokens": 4099, "inp": 1024, "out": 4096, "gelu": True, "bias": True, "dtype": "bf16", "train": False},
        # one training step of a projection of odd widths for a ragged batch
        {"name": "linear_ragged", "kind": "linear", "tokens": 1237, "inp": 1000, "out": 523, "gelu": False, "bias": True, "dtype": "bf16", "train": True},
        # one training step of the up-projection of GPT-2 medium's MLP with its GELU, 8 x 1024 tokens
        {"name": "linear_up", "kind": "linear", "tokens": 8192, "inp": 1024, "out": 4096, "gelu": True, "bias": True, "dtype": "bf16", "train": True},
        # one training step of its attention's output projection
        {"name": "linear_proj", "kind": "linear", "tokens": 8192, "inp": 1024, "out": 1024, "gelu": False, "bias": True, "dtype": "bf16", "train": True},
        # the optimizer step of a very small transformer in fp32 (latency counts)
        {"name": "adamw_tiny", "kind": "adamw", "bits": 32, "layers": 2, "width": 128, "vocab": 512, "dtype": "fp32", "master": False, "clip": False},
        # the optimizer step of a transformer of GPT-2 medium's size: bf16 weights with fp32 masters, gradients clipped by their norm
        {"name": "adamw_medium", "kind": "adamw", "bits": 32, "layers": 24, "width": 1024, "vocab": 50257, "dtype": "bf16", "master": True, "clip": True},
        # a small transformer of odd widths with states in 8 bits
        {"name": "adamw8_small", "kind": "adamw", "bits": 8, "layers": 4, "width": 333, "vocab": 5003, "dtype": "fp32", "master": False, "clip": True},
        # the large one with states in 8 bits
        {"name": "adamw8_medium", "kind": "adamw", "bits": 8, "layers": 24, "width": 1024, "vocab": 50257, "dtype": "bf16", "master": True, "clip": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Any width, a multiple of 64 three times in four."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.25 else max(64, n // 64 * 64)


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "linear", "adamw", "adamw"])
    if kind == "quantize":
        return {"kind": kind, "rows": _log(rng, 1, 8192), "cols": _width(rng, 16, 4096), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "both": rng.random() < 0.5}
    if kind == "linear":
        train = rng.random() < 0.5
        return {"kind": kind, "tokens": _log(rng, 32, 8192) if train else _log(rng, 1, 8192), "inp": _width(rng, 64, 4096), "out": _width(rng, 64, 2048 if train else 4096),
                "gelu": rng.random() < 0.4, "bias": rng.random() < 0.7, "dtype": rng.choice(["bf16", "bf16", "bf16", "fp16"]), "train": train}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    return {"kind": kind, "bits": rng.choice([8, 32]), "layers": _log(rng, 1, 24), "width": _width(rng, 16, 1024), "vocab": _log(rng, 64, 50257),
            "dtype": dtype, "master": dtype != "fp32" and rng.random() < 0.8, "clip": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs
def _randn(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _activations(g, rows, cols, dtype):
    """Rows of different sizes, some elements far out, a few columns of zeros."""
    x = torch.randn(rows, cols, generator=g, device=DEV) * torch.exp(0.7 * torch.randn(rows, 1, generator=g, device=DEV))
    x = torch.where(torch.rand(rows, cols, generator=g, device=DEV) < 0.002, 8 * x, x)
    x[:, : min(cols, 3)] = 0
    return x.to(dtype)


def _shapes(case):
    """The tensors of a transformer: those that weight decay applies to, and the biases and norms."""
    C, V, L = case["width"], case["vocab"], case["layers"]
    return [(V, C)] + [(C, C)] * (4 * L) + [(4 * C, C), (C, 4 * C)] * L, [(C,)] * (9 * L + 2) + [(4 * C,)] * L


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, s, dt = case["kind"], {"case": case}, DTYPES[case["dtype"]]
    if kind == "quantize":
        s["x"] = _activations(g, case["rows"], case["cols"], dt)
    elif kind == "linear":
        T, K, N = case["tokens"], case["inp"], case["out"]
        s.update(x=_activations(g, T, K, dt), w=_randn(g, (N, K), dt, K ** -0.5), b=_randn(g, (N,), dt, 0.1) if case["bias"] else None, dy=_randn(g, (T, N), dt))
        if own and not case["train"]:
            from torchmpi_b200.ops import fp8
            s["w8"] = fp8.quantize(s["w"])                # a generating program keeps its weights so
        elif not case["train"]:
            s["w8"] = _quantize(s["w"].float())
        elif own:
            for n in ("x", "w", "b"):
                if s[n] is not None:
                    s[n].requires_grad_(True)
    else:
        decayed, others = _shapes(case)
        shapes = decayed + others
        sizes = [math.prod(x) for x in shapes]
        starts = [0]
        for n in sizes:                                   # weights and gradients lie in flat buckets, as data-parallel training has them
            starts.append(starts[-1] + _padded(n))
        total, real = starts[-1], torch.zeros(starts[-1], dtype=torch.bool, device=DEV)
        for a, n in zip(starts, sizes):
            real[a: a + n] = True
        # gradients of different sizes from place to place; the averages are those of gradients like them
        size = torch.exp(torch.randn(total // BLOCK, 1, generator=g, device=DEV)).expand(-1, BLOCK).reshape(-1).mul_(1e-3).mul_(real)
        one = lambda: torch.randn(total, generator=g, device=DEV).mul_(size)      # noqa: E731
        grad, m, v = one(), one().mul_(0.2), one().square_().mul_(0.7).add_(size.square().mul_(0.3))
        weight = torch.randn(total, generator=g, device=DEV).mul_(0.02).mul_(real)
        s.update(weights=weight.to(dt, copy=True), grads=grad.to(dt), master=weight if case["master"] else None, decayed=starts[len(decayed)], step=STEPS)
        s["m"], s["v"] = (m, v) if case["bits"] == 32 else (_keep_m(m), _keep_v(v))
        if own:
            from torchmpi_b200.ops import adamw
            view = lambda flat, i: flat[starts[i]: starts[i] + sizes[i]].view(shapes[i])      # noqa: E731
            params, k = [torch.nn.Parameter(view(s["weights"], i)) for i in range(len(shapes))], len(decayed)
            opt = adamw.AdamW([{"params": params[:k], "weight_decay": DECAY}, {"params": params[k:], "weight_decay": 0.0}], lr=LR, betas=BETAS, eps=EPS,
                              bits=case["bits"], master_weights=case["master"], max_norm=MAX_NORM if case["clip"] else None)
            for i, p in enumerate(params):
                p.grad, st = view(s["grads"], i), opt.state[p]
                st["step"].fill_(STEPS)
                if case["master"]:
                    st["master"].copy_(view(weight, i))
                if case["bits"] == 32:
                    st["exp_avg"].copy_(view(m, i))
                    st["exp_avg_sq"].copy_(view(v, i))
                else:
                    blocks = slice(starts[i] // BLOCK, starts[i + 1] // BLOCK)
                    for name, kept in (("exp_avg", s["m"]), ("exp_avg_sq", s["v"])):
                        st[name].copy_(kept[0][blocks])
                        st[name + "_scale"].copy_(kept[1][blocks].view(-1))
            s = {"case": case, "weights": s["weights"], "params": params, "opt": opt}
    return s


# ---------------------------------------------------------------- plain forms, 32 bits
def _blocks(x):
    rows, cols = x.shape
    return torch.nn.functional.pad(x, (0, -cols % BLOCK)).view(rows, -1, BLOCK)


def _two_to(e):
    """2^e in fp32 for -126 <= e <= 127, exactly."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantize(x):
    """e4m3 numbers of the rows of x (fp32) and the exponent of the power of two that 128 of them share."""
    b = _blocks(x)
    a = torch.where(torch.isfinite(b), b.abs(), 0).amax(2, keepdim=True)
    m, e = torch.frexp(a)                                                 # a = m 2^e, 1/2 <= m < 1
    e = torch.where(m > 0.875, e - 8, e - 9).clamp_min(-126)              # a <= 448 * 2^e
    e = torch.where(a == 0, -126, e)
    q = torch.where(torch.isfinite(b), b * _two_to(-e // 2) * _two_to(-e - -e // 2), math.nan).to(torch.float8_e4m3fn)
    return q, e, x.shape[1]


def _restore(kept):
    q, e, cols = kept
    return (q.float() * _two_to(e)).flatten(1)[:, :cols]


def _rounded8(x):
    return _restore(_quantize(x))


def _gelu(z):
    return z * (0.5 * (1 + torch.erf(z * 0.5 ** 0.5)))


def _gelu_slope(z):
    return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5


# 8-bit optimizer states: a block's largest magnitude, and for each element the nearest multiple of 1/127 (of 1/255) to the root of its share of that.
# Of the second moment it is the root that is kept so, and none that is not zero becomes zero.
def _keep_m(m):
    b = m.view(-1, BLOCK)
    top = b.abs().amax(1, keepdim=True)
    code = torch.floor(127 * torch.sqrt(b.abs() / top.clamp_min(LEAST)) + 0.5)
    return (code * torch.sign(b)).to(torch.int8), top


def _value_m(kept):
    c = kept[0].float()
    return (c * c.abs() * (kept[1] / 16129)).view(-1)


def _keep_v(v):
    r = torch.sqrt(v).view(-1, BLOCK)
    top = r.amax(1, keepdim=True)
    code = torch.floor(255 * torch.sqrt(r / top.clamp_min(LEAST)) + 0.5)
    return torch.where(r > 0, code.clamp_min(1), 0).to(torch.uint8), top


def _value_v(kept):
    c = kept[0].float()
    return (c * c * (kept[1] / 65025)).square().view(-1)


def _plain_adamw(s):
    case, (b1, b2) = s["case"], BETAS
    s["step"] += 1
    g, w, out = s["grads"].float(), s["weights"].float() if s["master"] is None else s["master"], {}
    if case["clip"]:
        out["norm"] = torch.sqrt(torch.sum(g * g, dtype=torch.float64)).float()
        g = g * torch.clamp_max(MAX_NORM / (out["norm"] + 1e-6), 1)
    m, v = (s["m"], s["v"]) if case["bits"] == 32 else (_value_m(s["m"]), _value_v(s["v"]))
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    w[: s["decayed"]] *= 1 - LR * DECAY
    w -= LR / (1 - b1 ** s["step"]) * m / (torch.sqrt(v) / math.sqrt(1 - b2 ** s["step"]) + EPS)
    out["weights"] = s["weights"].copy_(w)
    if case["master"]:
        out["master"] = w
    if case["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        out["m"], out["v"] = s["m"], s["v"]
    else:
        s["m"], s["v"] = _keep_m(m), _keep_v(v)
        out["m"], out["v"] = _value_m(s["m"]).bfloat16(), _value_v(s["v"]).bfloat16()
    return out


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "adamw":
        return _plain_adamw(s)
    x, dt = s["x"].float(), s["x"].dtype
    if kind == "quantize":
        out = {"rows": _rounded8(x).to(dt)}
        if case["both"]:
            out["columns"] = _rounded8(x.t()).to(dt)
        return out
    if not case["train"]:
        y = _rounded8(x) @ _restore(s["w8"]).t()
        y = y if s["b"] is None else y + s["b"].float()
        return {"y": (_gelu(y.to(dt).float()) if case["gelu"] else y).to(dt)}
    w, dz = s["w"].float(), s["dy"].float()
    z = _rounded8(x) @ _rounded8(w).t()
    z = (z if s["b"] is None else z + s["b"].float()).to(dt)
    out = {"y": _gelu(z.float()).to(dt) if case["gelu"] else z}
    if case["gelu"]:
        dz = (dz * _gelu_slope(z.float())).to(dt).float()          # of what is kept of z, its rounded values; rounded as the gradient of a layer apart
    out["dx"] = (_rounded8(dz) @ _rounded8(w.t()).t()).to(dt)
    out["dw"] = (_rounded8(dz.t()) @ _rounded8(x.t()).t()).to(dt)
    if s["b"] is not None:
        out["db"] = dz.sum(0).to(dt)
    return out


# ---------------------------------------------------------------- through the package
def _package(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "adamw":
        opt = s["opt"]
        opt.step()
        out = {"norm": opt.grad_norm} if case["clip"] else {}
        out["weights"] = s["weights"]
        if case["master"]:
            out["master"] = opt.masters()
        out["m"], out["v"] = opt.moments()
        return out
    from torchmpi_b200.ops import fp8
    if kind == "quantize":
        if not case["both"]:
            return {"rows": fp8.dequantize(fp8.quantize(s["x"]), s["x"].dtype)}
        a, b = fp8.quantize_both(s["x"])
        return {"rows": fp8.dequantize(a, s["x"].dtype), "columns": fp8.dequantize(b, s["x"].dtype)}
    if not case["train"]:
        return {"y": fp8.linear(s["x"], s["w8"], s["b"], gelu=case["gelu"])}
    y = fp8.linear(s["x"], s["w"], s["b"], gelu=case["gelu"])
    wanted = [n for n in ("x", "w", "b") if s[n] is not None]
    return {"y": y.detach(), **dict(zip(["d" + n for n in wanted], torch.autograd.grad(y, [s[n] for n in wanted], s["dy"])))}


def run(state):
    return _package(state) if own else _plain(state)


def work(case):
    kind, b = case["kind"], SIZE[case["dtype"]]
    if kind == "quantize":
        # read, kept in each direction (a byte and a scale for 128), and those values given out again
        n, d = case["rows"] * case["cols"], 2 if case["both"] else 1
        return {"bytes": int(n * (b + d * (b + 2 * (1 + 1 / BLOCK)))), "flops": 4 * n * d}
    if kind == "linear":
        T, K, N = case["tokens"], case["inp"], case["out"]
        if case["train"]:
            return {"bytes": 2 * b * (T * K + T * N + K * N + (N if case["bias"] else 0)), "flops": 6 * T * K * N}
        return {"bytes": b * (T * K + T * N + (N if case["bias"] else 0)) + N * K + N * K // BLOCK, "flops": 2 * T * K * N}
    decayed, others = _shapes(case)
    n = sum(math.prod(x) for x in decayed + others)
    weights = b + 8 if case["master"] else 2 * b
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 4            # in 8 bits: read, written, and given out as values
    return {"bytes": int(n * (b + weights + states)), "flops": 20 * n}


# ---------------------------------------------------------------- the definitions in 64 bits
def _power(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _kept(x):
    """What the rows of x are in 8 bits: the nearest multiple of the e4m3 step at each value, half to even."""
    x = x.double()
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], BLOCK):
        b = x[:, c: c + BLOCK]
        top = b.abs().nan_to_num(0, 0, 0).amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.clamp_min(top, 2.0 ** -140) / 448))
        e = torch.where(top > 448 * _power(e), e + 1, torch.where(top <= 448 * _power(e - 1), e - 1, e)).clamp_min(-126)
        v = b / _power(e)
        step = _power(torch.frexp(v.abs().nan_to_num(1, 1, 1).clamp_min(2.0 ** -6))[1] - 4)
        out[:, c: c + BLOCK] = torch.where(torch.isfinite(b), torch.round(v / step) * step * _power(e), math.nan)
    return out


def _phi(z):
    return torch.special.ndtr(z)


def _companded(x, codes):
    """The values that `codes` levels of the root stand for, nearest to the roots of x over the block's largest; x >= 0, [blocks, 128]."""
    top = x.amax(1, keepdim=True)
    edges = ((torch.arange(codes, dtype=torch.float64, device=DEV) + 0.5) / codes).square()
    code = torch.bucketize(x / top.clamp_min(LEAST), edges, right=True).double()
    return code, top / codes ** 2


def _exact_adamw(case, seed):
    """From the inputs that the plain form takes."""
    s = _prepare_plain(case, seed)
    (b1, b2), t = BETAS, STEPS + 1
    grad, out = s["grads"].double(), {}
    weight = s["weights"].double() if s["master"] is None else s["master"].double()
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(grad)
        grad *= min(1.0, MAX_NORM / (float(out["norm"]) + 1e-6))
    if case["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        (mc, ms), (vc, vs) = s["m"], s["v"]
        m = (torch.sign(mc.double()) * (mc.double() / 127) ** 2 * ms.double()).view(-1)
        v = ((vc.double() / 255) ** 4 * vs.double() ** 2).view(-1)
    del s["m"], s["v"]
    m = torch.lerp(grad, m, b1)
    v = torch.lerp(grad.square_(), v, b2)
    weight[: s["decayed"]] -= LR * DECAY * weight[: s["decayed"]]
    weight -= LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt_() + EPS)
    out["weights"] = weight
    if case["master"]:
        out["master"] = weight
    if case["bits"] == 8:
        code, unit = _companded(m.abs().view(-1, BLOCK), 127)
        m = (torch.sign(m).view(-1, BLOCK) * code.square() * unit).view(-1)
        root = v.sqrt_().view(-1, BLOCK)
        code, unit = _companded(root, 255)
        v = (torch.where(root > 0, code.clamp_min(1), 0).square_() * unit).square_().view(-1)
    out["m"], out["v"] = m, v
    return out


def _prepare_plain(case, seed):
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def exact(case, seed):
    kind = case["kind"]
    if kind == "adamw":
        return _exact_adamw(case, seed)
    s = _prepare_plain(case, seed)
    x = s["x"].double()
    if kind == "quantize":
        return {"rows": _kept(x), "columns": _kept(x.t())} if case["both"] else {"rows": _kept(x)}
    w, dz = s["w"].double(), s["dy"].double()
    z = _kept(x).matmul(_kept(w).t())
    if s["b"] is not None:
        z = z + s["b"].double()
    if case["gelu"]:
        z = z.to(s["x"].dtype).double()
    y = z * _phi(z) if case["gelu"] else z
    if not case["train"]:
        return {"y": y}
    if case["gelu"]:
        dz = (dz * (_phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))).to(s["x"].dtype).double()
    out = {"y": y, "dx": _kept(dz).matmul(_kept(w.t()).t()), "dw": _kept(dz.t()).matmul(_kept(x.t()).t())}
    if s["b"] is not None:
        out["db"] = dz.sum(0)
    return out
