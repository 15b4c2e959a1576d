"""Plain 64-bit forms of group norm with an activation, rotary positions and 4-bit products, with bounds on what a correct
kernel may be off: the magnitudes that each rounding touches, from the 64-bit form itself.  ``u`` is half a step of the
storage type, ``U32`` that of 32 bits."""
import math

import torch

from decoder_ref import U32, UNIT

SERIAL = 64   # cells that one thread adds up one after the other, at the sizes tested; up to 256 threads follow each other


def tiny(dtype):
    return 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126


def activated(z, kind, slope=0.01):
    """The activation, its derivative, and a bound on that derivative's own."""
    if kind is None:
        return z, torch.ones_like(z), 0.0
    if kind == 'silu':
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p)), 0.5
    if kind == 'gelu':
        p = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 0.8
    low = slope if kind == 'leaky_relu' else 0.0
    d = torch.where(z > 0, 1.0, low)
    return torch.where(z > 0, z, z * low), d, 0.0


def group_norm(x, groups, weight, bias, eps, kind=None, slope=0.01, grad=None):
    """[(y, bound)] or, with `grad`, those of y, dx, dweight, dbias."""
    u, dtype = UNIT[x.dtype], x.dtype
    shape, C = x.shape, x.shape[-1]
    x = x.detach().double().cpu().reshape(shape[0], -1, groups, C // groups)
    uw = u if weight is None else UNIT[weight.dtype]
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight.detach().double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if bias is None else bias.detach().double().cpu()
    w, b = w.view(groups, -1), b.view(groups, -1)
    over = lambda t: t.mean((1, 3), keepdim=True)   # noqa: E731
    d = x - over(x)
    var = over(d * d)
    r = 1 / torch.sqrt(var + eps)
    h = d * r
    z = h * w + b
    # sums of differences from a value among those of the thread: their squares are at most eight times the variance
    e_mean, e_r = U32 * (SERIAL + 8) * (8 * var).sqrt(), 4 * U32 * (SERIAL + 8)
    e_h = h.abs() * (e_r + 4 * U32) + r * (e_mean + U32 * d.abs())
    e_z = w.abs() * e_h + 2 * U32 * ((h * w).abs() + z.abs())
    y, dy, bend = activated(z, kind, slope)
    own = {'silu': 2 * U32 * (z.abs() + 8), 'gelu': 2 * U32 * (z * z + 16)}.get(kind, U32)
    flat = lambda t: t.reshape(shape)   # noqa: E731
    out = [(flat(y), flat(1.13 * e_z + (own + u) * y.abs() + tiny(dtype)))]
    if grad is None:
        return out
    g = grad.detach().double().cpu().reshape(x.shape)
    gz = g * dy
    e_gz = g.abs() * (bend * e_z + own * 2 * (1 + dy.abs())) + U32 * gz.abs()
    if kind in ('relu', 'leaky_relu'):   # on the other side of the border
        e_gz = e_gz + g.abs() * (z.abs() <= e_z)
    chain = U32 * (SERIAL + 256 + 8)
    m1, m2 = over(w * gz), over(w * gz * h)
    e_m1 = over(w.abs() * e_gz) + chain * over((w * gz).abs())
    e_m2 = over(w.abs() * (e_gz * h.abs() + gz.abs() * e_h)) + chain * over((w * gz * h).abs())
    inner = w * gz - m1 - h * m2
    e_in = w.abs() * e_gz + e_m1 + h.abs() * e_m2 + e_h * m2.abs() + 4 * U32 * ((w * gz).abs() + m1.abs() + (h * m2).abs())
    dx = r * inner
    out.append((flat(dx), flat(r * e_in * (1 + e_r) + (e_r + 2 * U32 + u) * dx.abs() + tiny(dtype))))
    for terms, off in ((gz * h, e_gz * h.abs() + gz.abs() * e_h), (gz, e_gz)):
        t = terms.sum((0, 1)).flatten()
        out.append((t, (off + chain * terms.abs()).sum((0, 1)).flatten() + uw * t.abs() + tiny(dtype)))
    return out


def rotary(x, positions, frequencies, neighbours, back=False):
    """(y, bound)."""
    u, dtype = UNIT.get(x.dtype, 0.0), x.dtype
    x, f = x.detach().double().cpu(), frequencies.double().cpu()
    at = positions.cpu().double()
    pairs = f.shape[1]
    angle = (at @ f).unsqueeze(-2)
    e_angle = 2.0 ** -51 * (at.abs() @ f.abs()).unsqueeze(-2) * (f.shape[0] + 2)
    c, s = angle.cos(), angle.sin() * (-1 if back else 1)
    first = torch.arange(pairs) * (2 if neighbours else 1)
    second = first + (1 if neighbours else pairs)
    a, b = x[..., first], x[..., second]
    y, off = x.clone(), torch.zeros_like(x)
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    size = (a.abs() + b.abs()) * (6 * U32 + e_angle)
    off[..., first], off[..., second] = size, size
    off += (u * y.abs() + tiny(dtype)) * (off > 0)
    return y, off


LEVELS = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def to_codes(t):
    """The nearest level, of two the even code, found among all of them."""
    off = (t.double().abs().unsqueeze(-1) - LEVELS).abs()
    near = off == off.amin(-1, keepdim=True)
    even = near & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.int().argmax(-1), near.int().argmax(-1))
    return (code + 8 * (t < 0)).to(torch.uint8)


def quantize_groups(w, group):
    """(codes, scales) as the operator documents them."""
    n, k = w.shape
    t = torch.nn.functional.pad(w.float().cpu(), (0, -k % 128)).view(n, -1, group)
    scales = (t.abs().amax(2) / 6.0).clamp(min=2.0 ** -126)
    codes = to_codes(t * (1.0 / scales)[..., None]).view(n, -1, 16, 8)
    place = torch.tensor([4 * (p % 4) + p // 4 for p in range(16)])   # of piece p
    out = torch.empty_like(codes)
    out[:, :, place] = codes
    return (out[..., 0::2] | out[..., 1::2] << 4).reshape(n, -1), scales


def group_values(codes, scales, inputs):
    """What the codes stand for, in 64 bits."""
    codes, scales = codes.cpu(), scales.cpu().double()
    n = codes.shape[0]
    c = torch.stack((codes & 15, codes >> 4), -1).view(n, -1, 16, 8)
    place = torch.tensor([4 * (p % 4) + p // 4 for p in range(16)])
    c = c[:, :, place].reshape(n, scales.shape[1], -1).long()
    return (LEVELS[c & 7] * (1 - 2 * (c >> 3)) * scales[..., None]).reshape(n, -1)[:, :inputs]


def group_linear(x, codes, scales, bias):
    """(y, bound): sums of up to 128 exact products by the matrix units, those sums one after the other."""
    u, dtype = UNIT[x.dtype], x.dtype
    x = x.double().cpu()
    w = group_values(codes, scales, x.shape[-1])
    y, mass = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y = y + bias.cpu().to(dtype).double()
    return y, u * y.abs() + U32 * (132 + scales.shape[1] + 8) * mass + U32 * y.abs() + tiny(dtype)
