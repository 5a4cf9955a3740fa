"""Layers of experts and 8-bit activation checkpoints, as measurable cases.

Each case is one pass through an operator of ``torchmpi_b200.ops.act8`` or ``torchmpi_b200.ops.experts``: what a training
or generating program calls.  ``listed()`` gives the named cases, ``draw(rng)`` more of the same ranges, ``prepare`` the
inputs and weights a program holds before the call, ``run`` the pass (with ``own`` through the package, else in elementary
operations in 32 bits), ``exact`` the same results in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 32          # elements of a checkpoint that share a scale


def listed():
    return [
        # the activations of a few tokens kept in 8 bits and read back (latency counts); rows that end inside a block
        {"name": "store_few", "kind": "store", "rows": 48, "cols": 1000, "dtype": "fp32"},
        # the attention outputs or layer-norm outputs of several micro-batches of GPT-2 medium
        {"name": "store_activations", "kind": "store", "rows": 32768, "cols": 1024, "dtype": "bf16"},
        # the GELU of GPT-2 medium's MLP in backward, 8 x 1024 tokens, from an 8-bit checkpoint
        {"name": "gelu_backward", "kind": "gelu", "rows": 8192, "cols": 4096, "dtype": "bf16"},
        # one training step of a small MLP with 8-bit checkpoints: an odd number of tokens
        {"name": "mlp8_small", "kind": "mlp8", "rows": 251, "width": 512, "hidden": 2048},
        # one training step of the MLP of a GPT-2 medium block, 8 x 1024 tokens, with 8-bit checkpoints
        {"name": "mlp8_gpt2", "kind": "mlp8", "rows": 8192, "width": 1024, "hidden": 4096},
        # routing of a batch of single tokens while text is generated
        {"name": "route_tokens", "kind": "route", "tokens": 16, "experts": 8, "k": 2, "dtype": "bf16", "renormalize": True, "masked": 0.0, "train": False},
        # routing of a long batch over many experts, forward and backward, a part of it padding
        {"name": "route_batch", "kind": "route", "tokens": 65536, "experts": 64, "k": 8, "dtype": "fp32", "renormalize": False, "masked": 0.1, "train": True},
        # the experts' up-projection for the tokens of a generating batch: bound by the weights
        {"name": "grouped_tokens", "kind": "grouped", "rows": 16, "experts": 8, "inp": 1024, "out": 4096, "gelu": True, "train": False, "behind": 0},
        # the same of a training batch: 8 x 1024 tokens, two experts each
        {"name": "grouped_up", "kind": "grouped", "rows": 16384, "experts": 8, "inp": 1024, "out": 4096, "gelu": True, "train": False, "behind": 0},
        # many small experts, forward and backward: ragged, odd sizes, padding rows behind the last expert's
        {"name": "grouped_ragged", "kind": "grouped", "rows": 5003, "experts": 64, "inp": 520, "out": 1000, "gelu": False, "train": True, "behind": 37},
        # a layer of experts for a few generated tokens
        {"name": "experts_tokens", "kind": "experts", "tokens": 4, "experts": 8, "k": 2, "width": 1024, "hidden": 4096, "train": False, "act8": False, "masked": 0.0},
        # one training step of a layer of experts in place of GPT-2 medium's MLP, 8 x 1024 tokens, with 8-bit checkpoints
        {"name": "experts_train", "kind": "experts", "tokens": 8192, "experts": 8, "k": 2, "width": 1024, "hidden": 4096, "train": True, "act8": True, "masked": 0.02},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "gelu", "mlp8", "mlp8", "route", "grouped", "grouped", "grouped", "experts", "experts"])
    if kind in ("store", "gelu"):
        # any width: a multiple of the block three times in four
        cols = _log(rng, 16, 4096)
        cols = cols if rng.random() < 0.25 else max(32, cols // 32 * 32)
        return {"kind": kind, "rows": _log(rng, 1, 8192), "cols": cols, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    width, hidden = rng.choice([128, 256, 520, 768, 1024]), rng.choice([256, 512, 1000, 2048, 4096])
    if kind == "mlp8":
        return {"kind": kind, "rows": _log(rng, 8, 8191), "width": width, "hidden": hidden}
    if kind == "route":
        experts = _log(rng, 2, 256)
        return {"kind": kind, "tokens": _log(rng, 1, 32768), "experts": experts, "k": rng.randint(1, min(8, experts)),
                "dtype": rng.choice(["fp32", "bf16"]), "renormalize": rng.random() < 0.5, "masked": rng.choice([0.0, 0.2]),
                "train": rng.random() < 0.5}
    if kind == "grouped":
        return {"kind": kind, "rows": _log(rng, 2, 12288), "experts": _log(rng, 1, 64), "inp": width, "out": hidden,
                "gelu": rng.random() < 0.5, "train": rng.random() < 0.6, "behind": rng.choice([0, 0, 13])}
    experts = _log(rng, 2, 64)
    return {"kind": kind, "tokens": _log(rng, 1, 4096), "experts": experts, "k": rng.randint(1, min(4, experts)), "width": width,
            "hidden": hidden, "train": rng.random() < 0.6, "act8": rng.random() < 0.6, "masked": rng.choice([0.0, 0.1])}


# ---------------------------------------------------------------- inputs
def _randn(g, shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _pre_activation(g, rows, cols, dtype):
    """Rows of different sizes, some elements far out, a few blocks of zeros: what reaches a GELU in training."""
    x = torch.randn(rows, cols, generator=g, device=DEV) * torch.exp(0.7 * torch.randn(rows, 1, generator=g, device=DEV))
    x = torch.where(torch.rand(rows, cols, generator=g, device=DEV) < 0.002, 8 * x, x)
    x[:, : min(cols, 3)] = 0
    return x.to(dtype)


def _logits(g, tokens, experts, dtype, masked):
    """A gate's outputs: some experts are preferred; padding tokens have no expert at all, and some experts are closed."""
    l = torch.randn(tokens, experts, generator=g, device=DEV) + 0.5 * torch.randn(experts, generator=g, device=DEV)
    if masked:
        l = torch.where(torch.rand(tokens, experts, generator=g, device=DEV) < masked, -math.inf, l)
        l = torch.where(torch.rand(tokens, 1, generator=g, device=DEV) < masked, -math.inf, l)
    return l.to(dtype)


def _sizes(g, rows, experts):
    """Ragged shares of `rows`, one expert in eight without a row."""
    share = torch.rand(experts, generator=g, device=DEV) ** 2 * (torch.rand(experts, generator=g, device=DEV) > 0.125)
    share[0] += 1e-3
    ends = torch.round(torch.cumsum(share, 0) / share.sum() * rows).to(torch.int32)
    return torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), ends])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, s = case["kind"], {"case": case}
    if kind == "store":
        s["x"] = _pre_activation(g, case["rows"], case["cols"], DTYPES[case["dtype"]])
    elif kind == "gelu":
        dt = DTYPES[case["dtype"]]
        s["dy"] = _randn(g, (case["rows"], case["cols"]), dt)
        s["q"], s["scale"] = _quantize(_pre_activation(g, case["rows"], case["cols"], dt).float())
    elif kind == "mlp8":
        T, C, H = case["rows"], case["width"], case["hidden"]
        s.update(x=_randn(g, (T, C)), w1=_randn(g, (H, C), scale=C ** -0.5), b1=_randn(g, (H,), scale=0.1), w2=_randn(g, (C, H), scale=H ** -0.5),
                 b2=_randn(g, (C,), scale=0.1), dy=_randn(g, (T, C)))
    elif kind == "route":
        s["logits"] = _logits(g, case["tokens"], case["experts"], DTYPES[case["dtype"]], case["masked"])
        s["dweights"] = torch.randn(case["tokens"], case["k"], generator=g, device=DEV)
    elif kind == "grouped":
        R, E, K, N = case["rows"], case["experts"], case["inp"], case["out"]
        s.update(x=_randn(g, (R + case["behind"], K)), w=_randn(g, (E, N, K), scale=K ** -0.5), b=_randn(g, (E, N), scale=0.1),
                 dy=_randn(g, (R + case["behind"], N)), offsets=_sizes(g, R, E))
        s["ends"] = s["offsets"].tolist()
    else:
        T, E, C, H = case["tokens"], case["experts"], case["width"], case["hidden"]
        s.update(x=_randn(g, (T, C)), logits=_logits(g, T, E, torch.bfloat16, case["masked"]), w1=_randn(g, (E, H, C), scale=C ** -0.5),
                 b1=_randn(g, (E, H), scale=0.1), w2=_randn(g, (E, C, H), scale=H ** -0.5), b2=_randn(g, (E, C), scale=0.1), dy=_randn(g, (T, C)))
    if own:
        for n in ("x", "w1", "b1", "w2", "b2", "w", "b", "logits"):
            if n in s and case.get("train", kind == "mlp8"):
                s[n].requires_grad_(True)
    return s


# ---------------------------------------------------------------- plain forms, 32 bits
def _blocks(x):
    rows, cols = x.shape
    return torch.nn.functional.pad(x, (0, -cols % BLOCK)).view(rows, -1, BLOCK)


def _two_to(e):
    """2^e in fp32 for -126 <= e <= 127, exactly."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantize(x):
    """The checkpoint of x (fp32): e4m3 numbers and one power of two for 32 of them."""
    rows, cols = x.shape
    b = _blocks(x)
    a = torch.where(torch.isfinite(b), b.abs(), 0).amax(2, keepdim=True)
    m, e = torch.frexp(a)                                                 # a = m 2^e, 1/2 <= m < 1
    e = torch.where(m > 0.875, e - 8, e - 9).clamp_min(-126)              # a <= 448 * 2^e
    e = torch.where(a == 0, -126, e)
    q = torch.where(torch.isfinite(b), b * _two_to(-e // 2) * _two_to(-e - -e // 2), math.nan).to(torch.float8_e4m3fn)
    return q.view(rows, -1)[:, :cols].contiguous(), (e + 127).to(torch.uint8).view(rows, -1)


def _restore(q, scale):
    rows, cols = q.shape
    e = scale.int().unsqueeze(2) - 127
    return (_blocks(q.float()) * _two_to(e)).view(rows, -1)[:, :cols]


def _rounded8(x):
    return _restore(*_quantize(x))


def _gelu(z):
    return z * (0.5 * (1 + torch.erf(z * 0.5 ** 0.5)))


def _gelu_slope(z):
    return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5


def _route(logits, k, renormalize):
    """weights, chosen, order, place, offsets, all probabilities"""
    l = logits.float()
    T, E = l.shape
    key, index = torch.sort(torch.where(torch.isnan(l), -math.inf, l), dim=1, descending=True, stable=True)
    key, index = key[:, :k], index[:, :k]
    used = key > -math.inf
    top = torch.where(used[:, :1], key[:, :1], 0)
    p = torch.exp(l - top)
    p = p / torch.where(used[:, :1], p.sum(1, keepdim=True), 1)
    if renormalize:
        w = torch.exp(key - top)
        w = w / torch.where(used[:, :1], w.sum(1, keepdim=True), 1)
    else:
        w = torch.gather(p, 1, index)
    w = torch.where(torch.isnan(l).any(1, keepdim=True), math.nan, torch.where(used, w, 0))
    expert = torch.where(used, index, E).reshape(-1)
    expert, order = torch.sort(expert, stable=True)
    slot = torch.arange(T * k, device=l.device)
    place = torch.empty_like(slot)
    place[order] = torch.where(expert < E, slot, -1)
    offsets = torch.searchsorted(expert, torch.arange(E + 1, device=l.device))
    return (w, torch.where(used, index, -1).int(), torch.where(expert < E, order, -1).int(), place.view(T, k).int(), offsets.int(), p)


def _route_gradient(w, chosen, p, dw, renormalize):
    inner = (w * dw).sum(1, keepdim=True)
    at = chosen.clamp_min(0).long()
    share = torch.zeros_like(p).scatter_add_(1, at, torch.where(chosen >= 0, w * dw, 0))
    base = torch.zeros_like(p).scatter_add_(1, at, torch.where(chosen >= 0, w, 0)) if renormalize else p
    return share - base * inner


def _groups(ends):
    return [(e, a, b) for e, (a, b) in enumerate(zip(ends[:-1], ends[1:])) if b > a]


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "store":
        return {"restored": _rounded8(s["x"].float()).to(s["x"].dtype)}
    if kind == "gelu":
        z, dt = _restore(s["q"], s["scale"]), s["dy"].dtype
        return {"dz": (s["dy"].float() * _gelu_slope(z)).to(dt), "h": _gelu(z).to(dt)}
    if kind == "mlp8":
        x, w1, b1, w2, b2, dy = (s[n].float() for n in ("x", "w1", "b1", "w2", "b2", "dy"))
        z = x @ w1.t() + b1
        y = _gelu(z) @ w2.t() + b2
        x, z = _rounded8(x), _rounded8(z)
        dz = (dy @ w2) * _gelu_slope(z)
        out = {"y": y, "dx": dz @ w1, "dw1": dz.t() @ x, "db1": dz.sum(0), "dw2": dy.t() @ _gelu(z), "db2": dy.sum(0)}
        return {n: t.to(s["x"].dtype) for n, t in out.items()}
    if kind == "route":
        w, chosen, order, place, offsets, p = _route(s["logits"], case["k"], case["renormalize"])
        out = {"weights": w, "chosen": chosen, "order": order, "place": place, "offsets": offsets}
        if case["train"]:
            out["dlogits"] = _route_gradient(w, chosen, p, s["dweights"], case["renormalize"]).to(s["logits"].dtype)
        return out
    if kind == "grouped":
        x, w, b, dy = (s[n].float() for n in ("x", "w", "b", "dy"))
        z, groups, out = torch.zeros_like(dy), _groups(s["ends"]), {}
        for e, r0, r1 in groups:
            z[r0:r1] = x[r0:r1] @ w[e].t() + b[e]
        out["y"] = _gelu(z) if case["gelu"] else z
        if case["train"]:
            out.update(dx=torch.zeros_like(x), dw=torch.zeros_like(w), db=torch.zeros_like(b))
            dz = dy * _gelu_slope(z) if case["gelu"] else dy
            for e, r0, r1 in groups:
                out["dx"][r0:r1] = dz[r0:r1] @ w[e]
                out["dw"][e] = dz[r0:r1].t() @ x[r0:r1]
                out["db"][e] = dz[r0:r1].sum(0)
        return {n: t.to(s["x"].dtype) for n, t in out.items()}
    T, k = case["tokens"], case["k"]
    weights, chosen, order, place, offsets, p = _route(s["logits"], k, True)
    x, w1, b1, w2, b2, dy = (s[n].float() for n in ("x", "w1", "b1", "w2", "b2", "dy"))
    ends = offsets.tolist()
    n, groups = ends[-1], _groups(ends)
    entry = order[:n].long()
    token, wt = entry // k, weights.reshape(-1)[entry].unsqueeze(1)
    xs, z, ys = x[token], x.new_empty(n, case["hidden"]), x.new_empty(n, case["width"])
    for e, r0, r1 in groups:
        z[r0:r1] = xs[r0:r1] @ w1[e].t() + b1[e]
        ys[r0:r1] = _gelu(z[r0:r1]) @ w2[e].t() + b2[e]
    out = {"y": torch.zeros_like(x).index_add_(0, token, wt * ys)}
    if case["train"]:
        if case["act8"]:
            xs, z = _rounded8(x)[token], _rounded8(z)
        g, h, dxs, dwt = dy[token], _gelu(z), torch.empty_like(xs), torch.zeros(T * k, device=DEV)
        dw1, db1, dw2, db2 = (torch.zeros_like(t) for t in (w1, b1, w2, b2))
        dwe = x.new_empty(n)
        for e, r0, r1 in groups:
            dh = g[r0:r1] @ w2[e]
            dwe[r0:r1] = (dh * h[r0:r1]).sum(1) + (g[r0:r1] * b2[e]).sum(1)
            dz = wt[r0:r1] * dh * _gelu_slope(z[r0:r1])
            dw2[e], db2[e] = (wt[r0:r1] * g[r0:r1]).t() @ h[r0:r1], (wt[r0:r1] * g[r0:r1]).sum(0)
            dw1[e], db1[e] = dz.t() @ xs[r0:r1], dz.sum(0)
            dxs[r0:r1] = dz @ w1[e]
        dwt[entry] = dwe
        out.update(dx=torch.zeros_like(x).index_add_(0, token, dxs), dlogits=_route_gradient(weights, chosen, p, dwt.view(T, k), True),
                   dw1=dw1, db1=db1, dw2=dw2, db2=db2)
    return {n: t.to(s["x"].dtype) for n, t in out.items()}


# ---------------------------------------------------------------- through the package
def _package(s):
    from torchmpi_b200.ops import act8, experts
    case, kind = s["case"], s["case"]["kind"]
    if kind == "store":
        return {"restored": act8.dequantize(act8.quantize(s["x"]), s["x"].dtype)}
    if kind == "gelu":
        dz, h = act8.gelu_gradient(s["dy"], act8.Act8(s["q"], s["scale"]))
        return {"dz": dz, "h": h}
    if kind == "mlp8":
        wanted = ("x", "w1", "b1", "w2", "b2")
        y = act8.mlp(*(s[n] for n in wanted))
        return {"y": y.detach(), **dict(zip(("d" + n for n in wanted), torch.autograd.grad(y, [s[n] for n in wanted], s["dy"])))}
    if kind == "route":
        r = experts.route(s["logits"], case["k"], renormalize=case["renormalize"])
        out = {"weights": r.weights.detach(), "chosen": r.chosen, "order": r.order, "place": r.place, "offsets": r.offsets}
        if case["train"]:
            out["dlogits"], = torch.autograd.grad(r.weights, s["logits"], s["dweights"])
        return out
    if kind == "grouped":
        y = experts.grouped_linear(s["x"], s["w"], s["b"], s["offsets"], gelu=case["gelu"])
        out = {"y": y.detach()}
        if case["train"]:
            out["dx"], out["dw"], out["db"] = torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["dy"])
        return out
    wanted = ("x", "logits", "w1", "b1", "w2", "b2")
    routing = experts.route(s["logits"], case["k"])
    y = experts.mlp(s["x"], routing, s["w1"], s["b1"], s["w2"], s["b2"], act8=case["act8"])
    out = {"y": y.detach()}
    if case["train"]:
        out.update(zip(("d" + n for n in wanted), torch.autograd.grad(y, [s[n] for n in wanted], s["dy"])))
    return out


def run(state):
    return _package(state) if own else _plain(state)


def work(case):
    kind = case["kind"]
    if kind == "store":
        n, b = case["rows"] * case["cols"], SIZE[case["dtype"]]
        return {"bytes": n * (2 * b + 2) + 2 * case["rows"] * -(-case["cols"] // BLOCK), "flops": 4 * n}
    if kind == "gelu":
        n, b = case["rows"] * case["cols"], SIZE[case["dtype"]]
        return {"bytes": n * (3 * b + 1) + case["rows"] * -(-case["cols"] // BLOCK), "flops": 30 * n}
    if kind == "mlp8":
        T, C, H = case["rows"], case["width"], case["hidden"]
        return {"bytes": 2 * (4 * T * C + 4 * C * H + 2 * (C + H)), "flops": 12 * T * C * H}
    if kind == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        b = SIZE[case["dtype"]]
        return {"bytes": T * E * b * (2 if case["train"] else 1) + T * k * (20 if case["train"] else 16) + 4 * (E + 1), "flops": T * E * (k + 4)}
    if kind == "grouped":
        R, E, K, N = case["rows"] + case["behind"], case["experts"], case["inp"], case["out"]
        used = min(E, case["rows"])
        rows, weights = 2 * R * (K + N), 2 * used * N * (K + 1)
        if case["train"]:
            return {"bytes": 2 * rows + weights + 2 * E * N * (K + 1), "flops": 6 * case["rows"] * K * N}
        return {"bytes": rows + weights, "flops": 2 * case["rows"] * K * N}
    T, E, C, H, k = case["tokens"], case["experts"], case["width"], case["hidden"], case["k"]
    weights = 2 * (2 * C * H + C + H)
    if case["train"]:
        return {"bytes": 2 * (4 * T * C + 2 * T * E) + weights * (min(E, T * k) + E), "flops": 12 * T * k * C * H}
    return {"bytes": 2 * (2 * T * C + T * E) + weights * min(E, T * k), "flops": 4 * T * k * C * H}


# ---------------------------------------------------------------- the definitions in 64 bits
def _power(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _kept(x):
    """What a checkpoint of x stands for: the nearest multiple of the e4m3 step at each value, half to even."""
    x = x.double()
    rows, cols = x.shape
    out = torch.empty_like(x)
    for c in range(0, cols, BLOCK):
        b = x[:, c:c + BLOCK]
        top = b.abs().nan_to_num(0, 0, 0).amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.clamp_min(top, 2.0 ** -140) / 448))
        e = torch.where(top > 448 * _power(e), e + 1, torch.where(top <= 448 * _power(e - 1), e - 1, e)).clamp_min(-126)
        v = b / _power(e)
        step = _power(torch.frexp(v.abs().nan_to_num(1, 1, 1).clamp_min(2.0 ** -6))[1] - 4)
        out[:, c:c + BLOCK] = torch.where(torch.isfinite(b), torch.round(v / step) * step * _power(e), math.nan)
    return out


def _phi(z):
    return torch.special.ndtr(z)


def _density(z):
    return torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def _choices(logits, k, renormalize):
    l = logits.double()
    T, E = l.shape
    left, chosen, w = torch.where(torch.isnan(l), -math.inf, l), [], []
    index = torch.arange(E, device=DEV).expand(T, E)
    for _ in range(k):
        best = left.amax(1, keepdim=True)
        at = torch.where(left == best, index, E).amin(1, keepdim=True)
        chosen.append(torch.where(best > -math.inf, at, -1))
        left = left.scatter(1, at, -math.inf)
    chosen = torch.cat(chosen, 1)
    mask = torch.zeros(T, E + 1, dtype=torch.bool, device=DEV).scatter_(1, torch.where(chosen >= 0, chosen, E), True)[:, :E]
    p = torch.softmax(torch.where(mask, l, -math.inf) if renormalize else l, 1).nan_to_num(0)
    return p, chosen, torch.where(chosen >= 0, p.gather(1, chosen.clamp_min(0)), 0)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    d = {n: t.detach().double() for n, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point() and t.dtype != torch.float8_e4m3fn}
    if kind == "store":
        return {"restored": _kept(d["x"])}
    if kind == "gelu":
        z = s["q"].double() * _power(s["scale"].int() - 127).repeat_interleave(BLOCK, 1)[:, : case["cols"]]
        return {"dz": d["dy"] * (_phi(z) + z * _density(z)), "h": z * _phi(z)}
    if kind == "mlp8":
        z = torch.addmm(d["b1"], d["x"], d["w1"].t())
        y = torch.addmm(d["b2"], z * _phi(z), d["w2"].t())
        x, z = _kept(d["x"]), _kept(z)
        dz = d["dy"].matmul(d["w2"]) * (_phi(z) + z * _density(z))
        return {"y": y, "dx": dz.matmul(d["w1"]), "dw1": dz.t().matmul(x), "db1": dz.sum(0), "dw2": d["dy"].t().matmul(z * _phi(z)), "db2": d["dy"].sum(0)}
    if kind == "grouped":
        with torch.enable_grad():
            x, w, b = (d[n].requires_grad_(True) for n in ("x", "w", "b"))
            parts = []
            for e, (r0, r1) in enumerate(zip(s["ends"][:-1], s["ends"][1:])):
                z = x[r0:r1].matmul(w[e].t()) + b[e]
                parts.append(z * _phi(z) if case["gelu"] else z)
            y = torch.cat(parts + [torch.zeros(case["behind"], case["out"], dtype=torch.float64, device=DEV)])
            out = {"y": y.detach()}
            if case["train"]:
                out.update(zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), d["dy"])))
        return out
    T, E, k = case["tokens"], case["experts"], case["k"]
    renormalize = case.get("renormalize", True)
    p, chosen, weights = _choices(d["logits"], k, renormalize)
    if kind == "route":
        entries = torch.arange(T * k, device=DEV)
        lists = [entries[chosen.reshape(-1) == e] for e in range(E)]
        n = sum(len(x) for x in lists)
        order = torch.full((T * k,), -1, device=DEV)
        order[:n] = torch.cat(lists)
        place = torch.full((T * k,), -1, device=DEV)
        place[order[:n]] = entries[:n]
        offsets = torch.tensor([0] + [len(x) for x in lists], device=DEV).cumsum(0)
        out = {"weights": weights, "chosen": chosen.int(), "order": order.int(), "place": place.view(T, k).int(), "offsets": offsets.int()}
        if case["train"]:
            dp = torch.zeros(T, E + 1, dtype=torch.float64, device=DEV).scatter_(1, torch.where(chosen >= 0, chosen, E), s["dweights"].double())[:, :E]
            out["dlogits"] = p * (dp - (p * dp).sum(1, keepdim=True))
        return out
    y, dx, dp = torch.zeros_like(d["x"]), torch.zeros_like(d["x"]), torch.zeros_like(p)
    grads = {n: torch.zeros_like(d[n]) for n in ("w1", "b1", "w2", "b2")}
    kept = _kept(d["x"]) if case["act8"] else d["x"]
    for e in range(E):
        t = (chosen == e).any(1).nonzero().squeeze(1)
        if not len(t):
            continue
        w1, b1, w2, b2 = (d[n][e] for n in ("w1", "b1", "w2", "b2"))
        a = p[t, e].unsqueeze(1)
        z = d["x"][t].matmul(w1.t()) + b1
        y[t] += a * ((z * _phi(z)).matmul(w2.t()) + b2)
        if case["train"]:
            z = _kept(z) if case["act8"] else z
            h, g = z * _phi(z), d["dy"][t]
            dp[t, e] = (g * (h.matmul(w2.t()) + b2)).sum(1)
            dz = (a * g).matmul(w2) * (_phi(z) + z * _density(z))
            dx[t] += dz.matmul(w1)
            grads["w1"][e], grads["b1"][e] = dz.t().matmul(kept[t]), dz.sum(0)
            grads["w2"][e], grads["b2"][e] = (a * g).t().matmul(h), (a * g).sum(0)
    out = {"y": y}
    if case["train"]:
        out.update(dx=dx, dlogits=p * (dp - (p * dp).sum(1, keepdim=True)), dw1=grads["w1"], db1=grads["b1"], dw2=grads["w2"], db2=grads["b2"])
    return out
