"""What the operators on rows of 8-bit integers compute, in 64 bits on the CPU, and how far fp32 steps may be off it."""
import torch

U = 2.0 ** -24  # half a step of fp32, relative


def rows(y):
    """(whole numbers before they are rounded, scales) of rows: nan scales where a row holds no numbers only."""
    y = y.double().cpu()
    most = y.abs().amax(dim=1)
    t = torch.where(most[:, None] > 0, y * (127 / most[:, None]), torch.zeros_like(y))
    return t, most / 127


def check_rows(q, scale, y, t_roundings, scale_roundings):
    """``q`` and ``scale`` against the rows ``y`` (finite): every scale within so many fp32 roundings; every whole number the
    nearest one, either neighbour where the value lies within so many roundings of the middle between two."""
    t, want = rows(y)
    q, scale = q.cpu().double(), scale.cpu().double()
    # (a scale below fp32's normal numbers is rounded to a multiple of 2^-149)
    assert ((scale - want).abs() <= scale_roundings * U * want + 2.0 ** -150).all()
    assert (q == q.round()).all() and (q.abs() <= 127).all()
    off = (q - t).abs()
    slack = 127 * t_roundings * U
    assert (off <= 0.5 + slack).all(), float(off.max())
    # halves that are exact go to the even neighbour
    half = (t * 2 == (t * 2).round()) & ((t * 2) % 2 != 0) & (t_roundings == 0)
    assert (q[half] % 2 == 0).all()


def norm(x, gain, eps, add=None):
    """(the sum as fp32 holds it, the normed rows in 64 bits)"""
    h = x.float().cpu() if add is None else x.float().cpu() + add.float().cpu()
    d = h.double()
    return h, d / torch.sqrt((d * d).mean(dim=1, keepdim=True) + eps) * gain.double().cpu()


def sums(a, w):
    """sum_k a.q w.q times both scales, in 64 bits (exact up to the scales' two products)"""
    return (a.q.cpu().double() @ w.q.cpu().double().t()) * a.scale.cpu().double()[:, None] * w.scale.cpu().double()[None, :]


def gate(name, z, u, limit=0.0):
    if name == "silu":
        return z * torch.sigmoid(z) * u
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3))) * u
    g = torch.clamp(z, max=limit)
    return g * torch.sigmoid(1.702 * g) * (torch.clamp(u, -limit, limit) + 1)


def product(a, w, bias=None, base=None):
    """(y, how far fp32 steps may be off): three roundings of the product (the sum to fp32, two scales), one of each addition."""
    y = sums(a, w)
    tol = 3 * U * y.abs()
    for t in (bias, base):
        if t is not None:
            y = y + t.double().cpu()
            tol = tol + U * y.abs()
    return y, tol * 1.001 + 2.0 ** -149


def stored(tol, y, dtype):
    """The tolerance with the rounding to the output's type."""
    return tol + y.abs() * 2.0 ** -8 if dtype == torch.bfloat16 else tol
