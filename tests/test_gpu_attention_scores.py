"""Attention whose scores are far from zero: a softmax does not change when all scores of a row do by the same amount."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def run(q, k, v, go, **rest):
    import medvision_amd.ops as ops
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = ops.cross_attention(q, k, v, **rest)
    return (out, *torch.autograd.grad(out, (q, k, v), go))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries,keys,heads,dim", [(32, 96, 1, 96), (200, 120, 2, 120), (3, 64, 4, 64), (70, 31, 1, 31)])
@pytest.mark.parametrize("size", [40.0, 300.0, 5001.0, 60000.0])
def test_one_key_takes_all(dtype, queries, keys, heads, dim, size):
    """Scores of `size` squared for one key of a query and zero for the others: its value, and all of the gradient, to the bit."""
    size = torch.tensor(size).to(dtype).item()
    g = torch.Generator().manual_seed(queries)
    which = torch.randint(0, keys, (queries, heads), generator=g)
    q = torch.zeros(1, queries, heads, dim).scatter_(3, which[None, ..., None], size)
    k = (torch.eye(keys, dim) * size)[None, :, None].expand(1, keys, heads, dim)
    v = torch.randint(-8, 9, (1, keys, heads, dim), generator=g) / 8
    go = torch.randint(-8, 9, (1, queries, heads, dim), generator=g) / 8   # (sums of those, and their products with v, are exact)
    want = torch.stack([v[0, which[:, h], h] for h in range(heads)], 1)[None]
    want_dv = torch.zeros(1, keys, heads, dim)
    for h in range(heads):
        want_dv[0, :, h].index_add_(0, which[:, h], go[0, :, h])
    out, dq, dk, dv = run(*(t.to(dtype).to(DEV) for t in (q, k, v, go)), scale=1.0)
    assert torch.equal(out.float().cpu(), want)
    assert torch.equal(dv.float().cpu(), want_dv.to(dtype).float())
    assert not dq.any() and not dk.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries,keys,heads", [(20, 300, 2), (300, 50, 1), (150, 1500, 1), (3, 9000, 1)])
@pytest.mark.parametrize("offset", [0, 2 ** 9, 3 * 2 ** 12, -3 * 2 ** 12, 5 * 2 ** 18, -7 * 2 ** 18])
def test_scores_with_a_common_part(dtype, queries, keys, heads, offset):
    """Scores that 32 bits hold exactly, up to 2^21 from zero; later keys have larger ones, so that the largest so far grows."""
    D = 32
    g = torch.Generator().manual_seed(keys)
    half = lambda *s: torch.randint(-2, 3, s, generator=g) / 2   # noqa: E731
    q, k = half(1, queries, heads, D), half(1, keys, heads, D)
    power = 2 ** (math.frexp(abs(offset) or 1)[1] // 2)
    q[..., 0], k[..., 0] = power, offset / power
    q[..., 1], k[..., 1] = 1.0, (torch.arange(keys)[None, :, None] * 8 // keys).float()
    v = torch.randn(1, keys, heads, D, generator=g).to(dtype).float()
    go = torch.randn(1, queries, heads, D, generator=g).to(dtype).float()
    got = run(*(t.to(dtype).to(DEV) for t in (q, k, v, go)), scale=1.0)

    u = UNIT[dtype]
    tiny = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126
    # of a weight: the difference of two scores and its factor, exponential and sums in 32 bits, the rounding of 16-bit weights;
    # a common part of up to 2^12 may be taken off by a sum in 32 bits, twice
    e_common = U32 * min(2.0 ** 13, 4 * abs(offset) + 128)
    for h in range(heads):
        qq, kk, vv, dd = (t[0, :, h].double() for t in (q, k, v, go))
        s = qq @ kk.t()
        p = torch.softmax(s, 1)
        o = p @ vv
        e_p = 4 * U32 * (s.amax(1, keepdim=True) - s) + U32 * (32 + keys / 16) + e_common + (u if u > U32 else 0)
        t_o = (2 * e_p * p) @ vv.abs() + u * o.abs() + tiny
        dp = dd @ vv.t()
        ds = p * (dp - (dd * o).sum(1, keepdim=True))
        e_d = U32 * (D + 4) * (dd.abs() @ vv.abs().t()) + (dd.abs() * (t_o + U32 * (D + 4) * o.abs())).sum(1, keepdim=True)
        e_ds = (2 * e_p + 8 * U32) * ds.abs() + p * e_d
        grow = 1 + U32 * (16 + (queries + keys) / 16)
        want = (o, t_o), (ds @ kk, grow * e_ds @ kk.abs() + U32 * keys / 8 * ds.abs() @ kk.abs()), \
            (ds.t() @ qq, grow * e_ds.t() @ qq.abs() + U32 * queries / 8 * ds.abs().t() @ qq.abs()), \
            (p.t() @ dd, grow * (2 * e_p * p).t() @ dd.abs() + U32 * queries / 8 * p.t() @ dd.abs())
        for name, t, (w, bound) in zip(("output", "dq", "dk", "dv"), got, want):
            t = t[0, :, h].double().cpu()
            bound = bound + u * w.abs() + tiny
            assert torch.isfinite(t).all(), name
            over = (t - w).abs() - bound
            assert over.max() <= 0, f"{name}: {int((over > 0).sum())} of {t.numel()} off, by up to {(t - w).abs().max():.3g}"
