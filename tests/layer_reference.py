"""The transformer layers' definitions in 64 bits, for their tests.  Everything takes and returns torch tensors on one device; what
is called `bound` is how far a float32 computation of the same may be off, counted in half steps (E = 2^-24) by the operations
behind it; `rounded` adds the rounding to the output's type."""
import math

import numpy as np
import torch

E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(value, bound, dtype):
    """What a result may be off after its rounding to dtype; subnormal numbers are off by half of the smallest."""
    return bound * (1 + half_step(dtype)) + half_step(dtype) * value.abs() + torch.finfo(dtype).smallest_normal * half_step(dtype)


def check(got, want, bound, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert not torch.isnan(off).any(), what
    assert worst <= 0.0, "%s: off by %.3g where %.3g is allowed" % (what, off.flatten()[(off - bound).argmax()],
                                                                   bound.expand_as(off).flatten()[(off - bound).argmax()])


class Grid:
    """The 8-bit grid of a tensor (or of a given range): the float32 operations of fake quantization, by numpy."""

    def __init__(self, pkg, t, minmax=None):
        v = t.detach().float().cpu().numpy()
        lo, hi = minmax if minmax is not None else (v.min(), v.max())
        lo, hi = np.float32(lo), np.float32(hi)
        if lo == hi:   # a range of no width: everything is 0 on it
            low = high = scale = np.float32(0)
            self.zero = 0
            codes = np.zeros(v.shape, np.int64)
        else:
            low, high, scale, self.zero = pkg.fake_quant.nudge(lo, hi)
            snapped = pkg.fake_quant.fake_quant_with_min_max_vars(v, lo, hi)
            codes = np.rint((snapped.astype(np.float64) - np.float64(low)) / np.float64(scale)).astype(np.int64)
        assert codes.size == 0 or (codes.min() >= 0 and codes.max() <= 255)   # they are indexes into the table below
        self.scale = float(scale)
        self.codes = torch.from_numpy(codes).to(t.device)
        self.inside = torch.from_numpy((v >= low) & (v <= high)).to(t.device)
        self.values = (self.codes - self.zero).double() * self.scale


def product(table, x, k):
    """(product, bound) of two grids through the table (uint16[65536])."""
    a, b = x.codes, k.codes
    T = torch.from_numpy(np.ascontiguousarray(table).astype(np.int64)).to(a.device).view(256, 256)
    total = torch.zeros((a.shape[0], b.shape[1]), dtype=torch.int64, device=a.device)
    for i in range(a.shape[1]):
        total += T[:, b[i]][a[:, i]]
    total += a.shape[1] * x.zero * k.zero - k.zero * a.sum(1)[:, None] - x.zero * b.sum(0)
    z = total.double() * (x.scale * k.scale)
    return z, 3.01 * E * z.abs()


ACTIVATIONS = {
    None: lambda z: z,
    "relu": lambda z: torch.where(z > 0, z, torch.zeros_like(z)),
    "gelu": lambda z: z * 0.5 * torch.erfc(-z / math.sqrt(2.0)),
    "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))),
    "silu": lambda z: z * torch.sigmoid(z),
}


def slope(z, activation):
    z = z.double().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(ACTIVATIONS[activation](z).sum(), z)[0]


def dense(table, x, k, bias=None, residual=None, activation=None):
    """(output, pre, bounds of both)"""
    z, off = product(table, x, k)
    if bias is not None:
        z = z + bias.double()
        off = off + 1.01 * E * z.abs()
    y = ACTIVATIONS[activation](z)
    # slopes are below 1.13; an exponential or error function of a float32 argument u is off by a few half steps of its own and
    # by |u| of them for its argument's rounding, which the factor in front, z or smaller, makes z (16 + 4 z^2) exp(-..) at most
    act = off if activation in (None, "relu") else 1.13 * off + 64 * E * (z.abs() + y.abs())
    if residual is not None:
        y = y + residual.double()
        act = act + 1.01 * E * y.abs()
    return y, z, act, off


def dense_gradients(dz, dz_bound, x, k, x_dtype, k_dtype):
    """((gradient, bound) for the input, the kernel, the bias), dz in 64 bits with a bound of its own."""
    # A term of dz below the smallest normal number, 2^-126 in float32 and bfloat16, may count as 0: an exponential's result
    # that small does, and the matrix instructions take such operands for 0.  At most the value and each of its three terms.
    dz_bound = dz_bound + 4 * 2.0 ** -126
    def through(a, b, a_bound, dtype, depth):
        # gradients are rounded to terms of 8 bits: one for bfloat16, two for float16, three for float32
        terms = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -16, torch.float32: 2.0 ** -24}[dtype]
        size = a.abs() @ b.abs()
        return a @ b, a_bound @ b.abs() + (terms + 3 * E * (depth + 300)) * size
    gx, bx = through(dz, k.values.t().contiguous(), dz_bound, x_dtype, dz.shape[1])
    gk, bk = through(dz.t().contiguous(), x.values, dz_bound.t().contiguous(), k_dtype, dz.shape[0])
    gk, bk = gk.t(), bk.t()
    gb = dz.sum(0)
    bb = dz_bound.sum(0) + (dz.shape[0] + 8) * E * dz.abs().sum(0)
    out = ((gx * x.inside, bx * x.inside), (gk * k.inside, bk * k.inside), (gb, bb))
    return tuple((v, rounded(v, b, t)) for (v, b), t in zip(out, (x_dtype, k_dtype, k_dtype)))


def loss(z, z_bound, targets, ignore):
    """(rows' losses, bound, softmax, its bound relative to itself)"""
    counted = targets != ignore
    lse = torch.logsumexp(z, 1)
    at = z.gather(1, targets.clamp(min=0)[:, None])[:, 0]
    rows = torch.where(counted, lse - at, torch.zeros_like(lse))
    most = z_bound.max(1).values
    spread = (z.max(1).values[:, None] - z).clamp(max=100.0).max(1).values   # arguments of exponentials
    off = most + E * (z.shape[1] / 64 + 256 + 4 * spread) + 4 * E * lse.abs()
    bound = (off + z_bound.gather(1, targets.clamp(min=0)[:, None])[:, 0] + 2 * E * at.abs()) * counted
    p = (z - lse[:, None]).exp()
    return rows, bound, p, (off + most)[:, None] + E * (16 + 4 * (z - lse[:, None]).abs())


def normed(v, kind, eps):
    """(norm, reciprocal root, bound of the norm)"""
    mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    d = v - mean
    r = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    # sums of a row: at most 32 values a thread, then 22 more additions; the mean's error is one of every difference
    n = d * r
    mean_off = 64 * E * v.abs().mean(1, keepdim=True) * r * (kind == "layer")
    return n, r, 64 * E * n.abs() + mean_off * (1 + n.abs()) + 2 * E * (v.abs() * r)


def norm_backward(g, g_bound, v, kind, eps):
    """(gradient of v, bound) from that of norm(v)."""
    n, r, n_off = normed(v, kind, eps)
    mg = g.mean(1, keepdim=True) if kind == "layer" else 0.0
    mgn = (g * n).mean(1, keepdim=True)
    dv = (g - n * mgn - mg) * r
    size = g.abs() + n.abs() * (g * n).abs().mean(1, keepdim=True) + g.abs().mean(1, keepdim=True)
    off = g_bound + n_off * mgn.abs() + n.abs() * ((n_off * g.abs()).mean(1, keepdim=True) + (g_bound * n.abs()).mean(1, keepdim=True))
    off = off + g_bound.mean(1, keepdim=True) + 128 * E * size
    return dv, off * r + 64 * E * dv.abs()
