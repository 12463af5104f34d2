"""The attention operators' definitions in 64 bits, and buffers that show writes outside their views."""
import math

import torch


def eps(dtype):
    return torch.finfo(dtype).eps


class Fenced:
    """A tensor of the given shape inside a larger buffer of a known pattern; intact() says whether the rest still has it."""

    def __init__(self, shape, dtype, device="cuda", fill=None, gap=16):
        # every row of the last axis is followed by `gap` elements (16-byte boundaries are kept), and rows by half as many rows
        *lead, dim = shape
        wide = torch.empty([n + 1 for n in lead] + [dim + gap], dtype=dtype, device=device)
        self.raw = wide.view(torch.uint8)
        self.raw.fill_(0x5A)
        self.view = wide[tuple(slice(0, n) for n in lead) + (slice(0, dim),)]
        if fill is not None:
            self.view.copy_(fill)
        self.mask = torch.ones_like(wide, dtype=torch.bool)
        self.mask[tuple(slice(0, n) for n in lead) + (slice(0, dim),)] = False
        self.wide = wide

    def intact(self):
        size = self.wide.element_size()
        outside = self.raw.view(*self.wide.shape[:-1], self.wide.shape[-1], size)[self.mask]
        return bool((outside == 0x5A).all())


def rotate(x, positions, freq, interleaved):
    """x float64 [n][heads][dim]."""
    if freq is None:
        return x
    rot = 2 * len(freq)
    angle = (positions.double()[:, None] * freq)[:, None]
    c, s = angle.cos(), angle.sin()
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y


def attend(q, k, v, seen, scale):
    """float64 q [n][d], k, v [m][d], seen bool [n][m]: out, lse, the weighted sum of |v| (with the plain sum, see tolerance()), and the largest sum of |q||k|."""
    x = (q @ k.T) * scale
    x = torch.where(seen, x, torch.full_like(x, -math.inf))
    v = torch.where(seen.any(0)[:, None], v, torch.zeros_like(v))
    lse = torch.logsumexp(x, -1) if x.shape[1] else torch.full((len(q),), -math.inf, dtype=torch.float64, device=q.device)
    w = torch.where(seen, (x - lse[:, None]).exp(), torch.zeros_like(x)) if x.shape[1] else x
    return w @ v, lse, (w @ v.abs(), seen.double() @ v.abs()), scale * (q.abs() @ k.abs().T).amax(-1) if x.shape[1] else lse * 0


def tolerance(want, sums, product, n, dim, out, weight):
    """How far an output may be off. The result is rounded once (half a step of its type), each weight once (half a step of
    the 16-bit type it is multiplied in, relative to that weight: weight_eps / 2 of sum w |v|). A score is a sum of dim
    products in 32 bits, off by at most (dim + 8) 2^-23 of the sum of |q||k| (the eight: scaling, subtracting the
    reference, and the exponential's argument); the exponential by 2^-21, the sum of n weights by n 2^-23. Each of these moves a
    weight, and the sum that divides it, by that share. Below a type's smallest normal number steps no longer shrink: a
    result is off by half the smallest step there (fp16: 2^-25), and so is each weight, of which the largest is at least 1 and
    their sum therefore too: that step of the plain sum of |v|. out and weight: the types, out None for uint8."""
    weighted, plain = sums
    out_eps, step = (eps(out), torch.finfo(out).smallest_normal * eps(out) / 2) if out is not None else (0, 0)
    weight_eps, weight_step = eps(weight), torch.finfo(weight).smallest_normal * eps(weight) / 2
    share = (dim + 8) * 2.0 ** -23 * product + n * 2.0 ** -23 + 2.0 ** -20
    return out_eps / 2 * want.abs() + (weight_eps / 2 + 2.5 * share[..., None]) * weighted * 1.01 + step + weight_step * plain


def lse_tolerance(lse, product, n, dim):
    return (dim + 8) * 2.0 ** -23 * product + n * 2.0 ** -23 + 2.0 ** -20 + 2.0 ** -21 * lse.abs()
