"""Products in 8 bits with a scale for each block of 128, in 64 bits, with bounds of what rounding may change."""
import torch

BLOCK = 128


def kept(x):
    """What the rows of ``x`` stand for in 8 bits: the nearest multiple of the e4m3 step under each block's power of two, half to even."""
    x = x.double()
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], BLOCK):
        b = x[:, c: c + BLOCK]
        fine = torch.isfinite(b)
        top = torch.where(fine, b.abs(), 0).amax(1, keepdim=True)
        e = torch.full_like(top, -126)
        for _ in range(260):                                  # the smallest e from -126 with top <= 448 * 2^e
            e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
        v = torch.where(fine, b, 0) / torch.exp2(e)
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
        out[:, c: c + BLOCK] = torch.where(fine, torch.round(v / step) * step * torch.exp2(e), float("nan"))
    return out


def half_step(t, dtype):
    """How far rounding to ``dtype`` moves a value at most."""
    info = torch.finfo(dtype)
    return t.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def sums_bound(a, b):
    """How far fp32 sums of a row's products may be off: each of K additions by one unit in the last place (2^-23) of at most the sum of the magnitudes."""
    return (a.shape[1] + 2) * 2.0 ** -23 * (a.abs() @ b.abs().t())


def phi(z):
    return torch.special.ndtr(z)


def slope(z):
    return phi(z) + z * torch.exp(-z * z / 2) * 0.3989422804014327


def close(got, want, bound, name=""):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), name
    off = torch.where(nan, 0, (got - want).abs() - bound)
    assert bool((off <= 0).all()), (name, float(off.max()), int((off > 0).sum()))


def product(a, b, bias=None):
    """The exact product of what ``a`` and ``b`` stand for (64-bit matrices), and the bound of its fp32 sums."""
    y = a @ b.t()
    bound = sums_bound(a, b)
    if bias is not None:
        y = y + bias.double()
        bound = bound + y.abs() * 2.0 ** -23
    return y, bound


def grid(g, shape, step, most):
    """Multiples of ``step`` up to ``most``: numbers that 8 bits hold, and whose products' sums fp32 holds."""
    n = int(most / step)
    return torch.randint(-n, n + 1, shape, generator=g).double() * step
