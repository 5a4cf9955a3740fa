"""64-bit forms of 8-bit checkpoints and of layers of experts, with bounds of what the kernels' roundings may add.

A bound is carried beside each value: a rounding to bf16 adds 2^-8 of the value, a product adds the products of
magnitudes with the operands' bounds, and sums in fp32 add n 2^-24 of the sum of magnitudes for n terms (taken twice).  The
GELU's normal distribution is off by at most 1.4e-6 (the forms of csrc/kernels/gelu.cuh), the formulas around it by a few
fp32 roundings: 1.6e-6 + 4e-7 (1 + |z|), where the quicker form's value is off by 1.1e-6 and its slope by 1.4e-6.
"""
import torch

BF16 = 2.0 ** -8          # half a step, relative
BLOCK = 32


class V:
    """A value in 64 bits and how far a kernel may be from it."""

    def __init__(self, v, e=None):
        self.v = v.double()
        self.e = torch.zeros_like(self.v) if e is None else e

    def rounded(self, half=BF16):
        subnormal = 2.0 ** -25 if half == 2.0 ** -11 else 0.0           # half a step below fp16's smallest normal number
        return V(self.v, self.e + half * (self.v.abs() + self.e) + subnormal)

    def __getitem__(self, i):
        return V(self.v[i], self.e[i])

    def t(self):
        return V(self.v.t(), self.e.t())


def matmul(a, b):
    """a b with sums in fp32"""
    mag = a.v.abs() @ b.v.abs()
    err = a.e @ b.v.abs() + a.v.abs() @ b.e + a.e @ b.e
    return V(a.v @ b.v, err + 2 * a.v.shape[1] * 2.0 ** -24 * (mag + err))


def add(a, b):
    return V(a.v + b.v, a.e + b.e + 2.0 ** -23 * (a.v.abs() + b.v.abs()))


def mul(a, b):
    return V(a.v * b.v, a.e * b.v.abs() + a.v.abs() * b.e + a.e * b.e + 2.0 ** -23 * (a.v * b.v).abs())


def total(a, dim):
    n = a.v.shape[dim]
    return V(a.v.sum(dim), a.e.sum(dim) + 2 * n * 2.0 ** -24 * (a.v.abs() + a.e).sum(dim))


def gelu(z):
    """value and slope at z, whose bound has to be 0 (slopes are at most 1.13: a bound of z would pass with that factor)"""
    slack = 1.6e-6 + 4e-7 * (1 + z.v.abs())
    cdf, pdf = torch.special.ndtr(z.v), torch.exp(-z.v * z.v / 2) * 0.3989422804014327
    return V(z.v * cdf, slack + 1.13 * z.e), V(cdf + z.v * pdf, slack + z.e)


def power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def kept(x):
    """What an 8-bit checkpoint of x stands for."""
    x = x.double()
    pad = torch.nn.functional.pad(x, (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    finite = torch.isfinite(pad)
    a = torch.where(finite, pad.abs(), 0).amax(-1, keepdim=True)
    m, e = torch.frexp(a)
    e = torch.where(a > 0, torch.where(m > 0.875, e - 8, e - 9), -126).clamp_min(-126)
    v = torch.where(finite, pad, 0) / power(e)
    step = power(torch.frexp(v.abs().clamp_min(2.0 ** -6))[1] - 4)
    out = torch.where(finite, torch.round(v / step) * step * power(e), float("nan"))
    return out.flatten(-2)[..., : x.shape[-1]]


def close(got, want, what=""):
    """Every element inside its bound (and NaN where the value is)."""
    g = got.detach().double().to(want.v.device)
    assert g.shape == want.v.shape, (what, g.shape, want.v.shape)
    off = (g - want.v).abs()
    ok = (off <= want.e) | (torch.isnan(g) & torch.isnan(want.v))
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} off, the worst {float((off - want.e).nan_to_num(9e9).max()):.3g} beyond its bound"


def grid(g, shape, step, top, device):
    """Multiples of `step` up to `top` in magnitude: products of two such tensors have sums that fp32 holds exactly."""
    n = int(top / step)
    return torch.randint(-n, n + 1, shape, generator=g).mul(step).to(device)


def route(logits, k, renormalize):
    """weights (64 bits), chosen, order, place, offsets by the definition, one token after the other"""
    l = logits.detach().double().cpu()
    T, E = l.shape
    weights, chosen = torch.zeros(T, k, dtype=torch.float64), torch.full((T, k), -1)
    lists = [[] for _ in range(E)]
    for t in range(T):
        nan = bool(torch.isnan(l[t]).any())
        row = [(float("-inf") if v != v else v) for v in l[t].tolist()]
        best = [e for e in sorted(range(E), key=lambda e: (-row[e], e)) if row[e] > float("-inf")][:k]
        over = torch.tensor([row[e] for e in best] if renormalize else row, dtype=torch.float64)
        p = torch.softmax(over, 0)
        for j, e in enumerate(best):
            chosen[t, j] = e
            weights[t, j] = p[j if renormalize else e]
            lists[e].append(t * k + j)
        if nan:
            weights[t] = float("nan")
    order, place, offsets = torch.full((T * k,), -1), torch.full((T * k,), -1), [0]
    for entries in lists:
        for i, entry in enumerate(entries):
            order[offsets[-1] + i], place[entry] = entry, offsets[-1] + i
        offsets.append(offsets[-1] + len(entries))
    return weights, chosen, order, place.view(T, k), torch.tensor(offsets)


def mlp8(x, w1, b1, w2, b2, dy):
    """(y, dx, dw1, db1, dw2, db2) of act8.mlp in bf16, where x w1^T + b1 is exact in fp32 (see grid)."""
    z = V(x.double() @ w1.double().t() + b1.double())
    y = add(matmul(gelu(z)[0].rounded(), V(w2).t()), V(b2)).rounded()
    zk, xk = V(kept(z.v)), V(kept(x))
    h, slope = gelu(zk)
    dz = mul(matmul(V(dy), V(w2)).rounded(), slope).rounded()
    return (y, matmul(dz, V(w1)).rounded(), matmul(dz.t(), xk.rounded()).rounded(), total(dz, 0).rounded(),
            matmul(V(dy).t(), h.rounded()).rounded(), total(V(dy), 0).rounded())


def experts(x, weights, chosen, w1, b1, w2, b2, dy, act8, parts=False, exact_z=True):
    """(y, dx, dweights, dw1, db1, dw2, db2) of experts.mlp in bf16, where x w1^T + b1 is exact in fp32 (or, without
    act8, carries its bound: exact_z=False).  parts: of combine, two
    grouped_linear and dispatch one by one, which round the weighted rows of dy, and take the weights' gradient from what the experts returned."""
    T, k = chosen.shape
    E, (H, C) = w1.shape[0], w1.shape[1:]
    z0 = lambda *s: V(torch.zeros(*s, dtype=torch.float64, device=x.device))
    y, dx, dwt = z0(T, C), z0(T, C), z0(T, k)
    dw1, db1, dw2, db2 = z0(E, H, C), z0(E, H), z0(E, C, H), z0(E, C)
    zero_b = lambda b, e, n: V(torch.zeros(n, dtype=torch.float64, device=x.device)) if b is None else V(b[e])

    def into(to, at, what):
        s = add(to[at], what)
        to.v[at], to.e[at] = s.v, s.e

    xk = V(kept(x)).rounded() if act8 else V(x)
    for e in range(E):
        t, j = (chosen == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        wt = V(weights[t, j].double().unsqueeze(1))
        z = V(x[t].double() @ w1[e].double().t() + zero_b(b1, e, H).v) if exact_z else add(matmul(V(x[t]), V(w1[e]).t()), zero_b(b1, e, H))
        ys = add(matmul(gelu(z)[0].rounded(), V(w2[e]).t()), zero_b(b2, e, C)).rounded()
        into(y, t, mul(wt, ys))
        zk = V(kept(z.v)) if act8 else z.rounded()
        g = V(dy[t])
        h, slope = gelu(zk)
        dh = matmul(g, V(w2[e])).rounded()
        dwe = add(total(mul(dh, h), 1), total(mul(g, zero_b(b2, e, C)), 1))
        dz, hw, gw = mul(mul(wt, dh), slope).rounded(), mul(wt, h).rounded(), mul(wt, g)
        grad_w2 = matmul(g.t(), hw)
        if parts:
            gw = gw.rounded()
            dz, dwe, grad_w2 = mul(matmul(gw, V(w2[e])).rounded(), slope).rounded(), total(mul(g, ys), 1), matmul(gw.t(), h.rounded())
        dwt.v[t, j], dwt.e[t, j] = dwe.v, dwe.e
        for to, what in ((dw1, matmul(dz.t(), xk[t])), (db1, total(dz, 0)), (dw2, grad_w2), (db2, total(gw, 0))):
            r = what.rounded()
            to.v[e], to.e[e] = r.v, r.e
        into(dx, t, matmul(dz, V(w1[e])).rounded())
    return y.rounded(), dx.rounded(), dwt, dw1, db1, dw2, db2
