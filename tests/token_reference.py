"""Plain float64 forms of the token operators (numpy-free torch on the CPU) and the error bounds their tests use.

Bounds count roundings: u = 2^-24 is half a step of float32, relative; half_step(T) that of the output type.  A quantity that the kernel
forms from float32 terms t_i is off by at most (number of roundings on its way) * u * sum |t_i|; the magnitude sums are computed here too."""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def bound(want, magnitude, roundings, dtype):
    """|got - want| <= this: `roundings` float32 roundings of terms whose absolute values sum to `magnitude`, one to the output type (whose
    smallest step, for values that underflow, is the subnormal one)."""
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return magnitude * (roundings * U) * (1 + half_step(dtype)) + want.abs() * half_step(dtype) + tiny


def assert_within(got, want, limit, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, tuple(got.shape), tuple(want.shape))
    bad = ~((got - want).abs() <= limit)
    assert not bad.any(), "%s: %d of %d outside; worst %.3e of its bound, at %s" % (
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / limit).nan_to_num(nan=math.inf).max()), bad.nonzero()[0].tolist())


def pair_index(sections, paired):
    R = sum(sections)
    p = torch.arange(R // 2)
    return (2 * p, 2 * p + 1) if paired == "interleaved" else (p, p + R // 2)


def angles(pos, sections, theta, B, N, frequencies=None):
    """(B, N, R/2) angles in float64"""
    if frequencies is None:
        frequencies = torch.tensor([theta ** (-2.0 * j / s) for s in sections for j in range(s // 2)], dtype=torch.float64)
    axis = torch.tensor([a for a, s in enumerate(sections) for _ in range(s // 2)])
    pos = pos.detach().cpu().double()
    if pos.dim() == 2:
        pos = pos[None].expand(B, -1, -1)
    return (pos[..., axis] * frequencies).expand(B, N, -1)


def rotate(x, phi, sections, paired, inverse=False):
    """(rotated, magnitude |a| + |b| of each channel's pair) of x (B, N, H, D) in float64"""
    ia, ib = pair_index(sections, paired)
    c, s = torch.cos(phi)[:, :, None], torch.sin(phi)[:, :, None]
    if inverse:
        s = -s
    a, b = x[..., ia], x[..., ib]
    out, mag = x.clone(), x.abs()
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = a.abs() + b.abs()
    mag[..., ib] = mag[..., ia]
    return out, mag


# cosine and sine: the remainder in quarter turns rounds once (2^-24 * pi/4 of angle), the sums and their dropped terms stay under 2 u, the
# rotation multiplies and adds: 2 more.  Five, and one to spare for the sign of what is compounded.
ROTATION = 6


def norm_rotary(x, w, phi, sections, paired, eps):
    """(out, magnitude, roundings)"""
    D = x.shape[-1]
    rho = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    y = x * rho * (w if w is not None else 1.0)
    out, mag = rotate(y, phi, sections, paired)
    # the sum of D squares: every square and every addition rounds once, at most D + 1 on a term's way, and half of it reaches rho; mean, eps,
    # root and quotient 4, the two products 2
    return out, mag, ROTATION + (D + 1) / 2 + 6


def norm_rotary_backward(dy, x, w, phi, sections, paired, eps):
    """dx, its magnitude, dw, its magnitude, roundings (of both, without the length of dw's sum)"""
    D = x.shape[-1]
    rho = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    wv = w if w is not None else torch.ones(D, dtype=torch.float64)
    g, gmag = rotate(dy, phi, sections, paired, inverse=True)
    xh = x * rho
    dx = rho * (g * wv - xh * (g * wv * xh).mean(-1, keepdim=True))
    dx_mag = rho * (gmag * wv.abs() + xh.abs() * (gmag * wv.abs() * xh.abs()).mean(-1, keepdim=True))
    # rotation, rho twice more than once (its square in the mean's factor): 3 (D + 1)/2 + 12, the mean's own sum D + 1, products 6
    return dx, dx_mag, (g * xh).sum((0, 1, 2)), (gmag * xh.abs()).sum((0, 1, 2)), ROTATION + 3 * (D + 1) / 2 + 12 + D + 1 + 6
