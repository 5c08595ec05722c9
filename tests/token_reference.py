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


# ---- gated feed-forward block: values with error bounds carried through the block's own roundings ----
class V:
    """A float64 value and a bound on how far the kernel's may be from it."""

    def __init__(self, val, err=None):
        self.val, self.err = val, torch.zeros_like(val) if err is None else err

    def rounded(self, dtype):
        """rounded to the tensors' type: half a step, or half the subnormal one"""
        tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        return V(self.val, self.err + (self.val.abs() + self.err) * half_step(dtype) + tiny)

    def top(self):
        return self.val.abs() + self.err

    def __mul__(self, o):  # one float32 product
        return V(self.val * o.val, self.err * o.top() + self.val.abs() * o.err + self.top() * o.top() * U)

    def t(self):
        return V(self.val.t(), self.err.t())


def product(a, b):
    """a b^T summed in float32 in any order: K products and additions, each term rounded at most K + 1 times, twice that for what the matrix
    core keeps of the smaller addend"""
    K = a.val.shape[1]
    val = a.val @ b.val.t()
    err = a.err @ b.top().t() + a.val.abs() @ b.err.t() + (2 * (K + 1) * U) * (a.top() @ b.top().t())
    return V(val, err)


def plus(a, b):
    return V(a.val + b.val, a.err + b.err + (a.top() + b.top()) * U)


def act(z, kind):
    """(activation, derivative) of V z; |act'| < 1.13, |act''| < 0.81; the float32 evaluation loses a few roundings of z, and of (1 + |z|)^3 in the
    tanh form's polynomial factor"""
    x = z.val
    if kind == "silu":
        s = torch.sigmoid(x)
        a, d = x * s, s * (1 + x * (1 - s))
    elif kind == "gelu":
        c = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
        a, d = x * c, c + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    else:
        k, c = math.sqrt(2 / math.pi), 0.044715
        t = torch.tanh(k * (x + c * x ** 3))
        a, d = 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * k * (1 + 3 * c * x * x)
    return V(a, 1.13 * z.err + 16 * U * x.abs()), V(d, 0.81 * z.err + 16 * U * (1 + x.abs()) ** 3)


def gated_ffn(x, wg, wu, wd, kind, dtype, dy=None):
    """y, or (y, dx, dwg, dwu, dwd), as V of their final rounding; hidden, dgate and dup are rounded to `dtype` where the block rounds them"""
    x, wg, wu, wd = (V(t.double()) for t in (x, wg, wu, wd))
    gate, up = product(x, wg), product(x, wu)
    hidden = (act(gate, kind)[0] * up).rounded(dtype)
    y = product(hidden, wd).rounded(dtype)
    if dy is None:
        return y
    dy = V(dy.double())
    dh = product(dy, wd.t())
    a, d = act(gate, kind)
    dgate, dup = (dh * up * d).rounded(dtype), (dh * a).rounded(dtype)
    dx = plus(product(dgate, wg.t()), product(dup, wu.t())).rounded(dtype)
    return y, dx, product(dgate.t(), x.t()).rounded(dtype), product(dup.t(), x.t()).rounded(dtype), product(dy.t(), hidden.t()).rounded(dtype)
