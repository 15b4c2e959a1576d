"""Plain 64-bit forms of the region decoders' operators, with bounds on what a correct kernel may be off.

The bounds follow from the roundings that the operators document: unit roundoff ``u`` of the storage type for each
result and, in attention, for the weights and their gradients before the second product; 2^-24 for each step in 32 bits.
Each is the sum of the magnitudes that a rounding touches, taken from the 64-bit form itself."""
import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -24


def valid_keys(batch, keys, mask, lengths):
    keep = torch.ones(batch, keys, dtype=torch.bool)
    if lengths is not None:
        keep &= torch.arange(keys) < lengths.cpu()[:, None]
    if mask is not None:
        keep &= mask.cpu()
    return keep


def attention(q, k, v, mask=None, lengths=None, scale=None, grad=None):
    """[(output, bound)] or, with `grad`, those of output, dq, dk, dv."""
    u = UNIT[q.dtype]
    tiny = 2.0 ** -24 if q.dtype == torch.float16 else 2.0 ** -126   # results below the normal numbers
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    keep = valid_keys(B, Lk, mask, lengths)
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    go = None if grad is None else grad.detach().double().cpu()
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    tq, tk, tv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        at = keep[b].nonzero()[:, 0]
        if not at.numel():
            continue
        for h in range(H):
            g = h // (H // Hk)
            qq, kk, vv = q[b, :, h], k[b, at, g], v[b, at, g]
            s = scale * qq @ kk.t()
            p = torch.softmax(s, 1)
            o = p @ vv
            # a score is off by its products' and its own roundings; a weight by twice that, the sum's error and its rounding
            e_s = U32 * ((D + 4) * (abs(scale) * qq.abs() @ kk.abs().t()).amax(1, keepdim=True) + 4 * s.abs().amax(1, keepdim=True))
            e_p = 2 * e_s + U32 * (16 + len(at) / 16) + (u if u > U32 else 0)
            t = 2 * e_p * (p @ vv.abs()) + u * o.abs() + tiny
            out[b, :, h], tol[b, :, h] = o, t
            if go is None:
                continue
            dd = go[b, :, h]
            dp = dd @ vv.t()
            ds = p * (dp - (dd * o).sum(1, keepdim=True))
            e_d = U32 * (D + 4) * (dd.abs() @ vv.abs().t()) + (dd.abs() * (t + U32 * (D + 4) * o.abs())).sum(1, keepdim=True)
            e_ds = (2 * e_p + U32 * 8) * ds.abs() + p * e_d
            grow = 1 + U32 * (16 + (Lq * H // Hk + len(at)) / 16)
            dq[b, :, h] = scale * ds @ kk
            tq[b, :, h] = grow * abs(scale) * e_ds @ kk.abs() + U32 * len(at) / 8 * abs(scale) * ds.abs() @ kk.abs()
            dk[b, at, g] += scale * ds.t() @ qq
            tk[b, at, g] += grow * abs(scale) * e_ds.t() @ qq.abs() + U32 * Lq / 8 * abs(scale) * ds.abs().t() @ qq.abs()
            dv[b, at, g] += p.t() @ dd
            tv[b, at, g] += grow * (2 * e_p * p).t() @ dd.abs() + U32 * Lq / 8 * p.t() @ dd.abs()
    if go is None:
        return [(out, tol)]
    return [(out, tol), *((d, t + u * d.abs() + tiny) for d, t in ((dq, tq), (dk, tk), (dv, tv)))]


def add_rms_norm(x, residual, weight, eps, grad=None, grad_sum=None):
    """y, h and, with `grad`, dh and dweight, each with its bound."""
    u, uw = UNIT[x.dtype], UNIT[weight.dtype]
    tiny = 2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126
    kind = x.dtype
    x, w = x.detach().double().cpu(), weight.detach().double().cpu()
    h = x
    if residual is not None:
        h = (x + residual.detach().double().cpu()).to(kind).double()
    C = x.shape[-1]
    few = U32 * (16 + C / 64)   # sums of a row: pairwise over lanes, a few terms per lane
    n = torch.rsqrt((h * h).mean(-1, keepdim=True) + eps)
    y = h * n * w
    got = [(y, (u + few + 4 * U32) * y.abs() + tiny), (h, torch.zeros_like(h))]
    if grad is None:
        return got
    g = grad.detach().double().cpu()
    gw = g * w
    c = (gw * h).mean(-1, keepdim=True)
    back = h * n ** 3 * c
    dh = n * gw - back
    slack = (few + 8 * U32) * ((n * gw).abs() + back.abs() + (h * n ** 3).abs() * (gw * h).abs().mean(-1, keepdim=True))
    if grad_sum is not None:
        dh = dh + grad_sum.detach().double().cpu()
    got.append((dh, slack + (u + U32) * dh.abs() + tiny))
    terms = (g * h * n).reshape(-1, C)
    dw = terms.sum(0)
    got.append((dw, (few + U32 * (16 + len(terms) / 8)) * terms.abs().sum(0) + uw * dw.abs() + tiny))
    return got


def blocks(x, rows):
    """What quantize_blocks gives, in the operator's own steps: scale and its reciprocal in 32 bits."""
    n, k = x.shape
    t = torch.nn.functional.pad(x.float(), (0, -k % 128, 0, -n % rows))
    t = t.reshape(t.shape[0] // rows, rows, t.shape[1] // 128, 128)
    scales = (t.abs().amax((1, 3)) / 448.0).clamp(min=2.0 ** -126)
    q = (t * (1.0 / scales)[:, None, :, None]).reshape(t.shape[0] * rows, -1)[:n]
    return q.to(torch.float8_e4m3fn), scales


def values(q, scales, rows):
    return q.cpu().float().double() * scales.cpu().double().repeat_interleave(rows, 0)[:q.shape[0]].repeat_interleave(128, 1)


def block_linear(q, q_scales, w, w_scales, bias, dtype):
    """(y, bound): within a block the matrix core keeps 16 bits below the largest of the terms that it adds at once."""
    a, b = values(q, q_scales, 1), values(w, w_scales, 128)
    y = a @ b.t()
    mass = a.abs() @ b.abs().t()
    if bias is not None:
        y = y + bias.cpu().to(dtype).double()
    return y, UNIT[dtype] * y.abs() + (2.0 ** -13 + U32 * (a.shape[1] / 128 + 8)) * mass + (2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126)


def check(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    worst = over.argmax()
    assert over.max() <= 0, (f"{what}: {int((over > 0).sum())} of {got.numel()} off, the worst by "
                             f"{(got - want).abs().flatten()[worst]:.3g} (bound {bound.flatten()[worst]:.3g}, value {want.flatten()[worst]:.3g})")


def slope(f, tensors, directions, step=1e-4):
    """Directional derivative of f in 64 bits by central differences."""
    ahead = f(*(t + step * d for t, d in zip(tensors, directions)))
    behind = f(*(t - step * d for t, d in zip(tensors, directions)))
    return (ahead - behind) / (2 * step)


def attention_value(q, k, v, grad, keep, scale):
    """sum(output * grad), for differences."""
    B, Lq, H, D = q.shape
    r = H // k.shape[2]
    s = torch.einsum('bihd,bjhd->bhij', q, k.repeat_interleave(r, 2)) * scale
    p = torch.softmax(s.masked_fill(~keep[:, None, None], -math.inf), -1).nan_to_num(0.0)
    return (torch.einsum('bhij,bjhd->bihd', p, v.repeat_interleave(r, 2)) * grad).sum()
