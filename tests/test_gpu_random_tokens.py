"""Drawn sizes, types, layouts and positions of group norm, rotary positions and 4-bit products against their 64-bit forms."""
import random

import pytest
import torch

import tokens_ref as ref
from decoder_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def size(rng, most):
    """From one on, small numbers as often as large ones."""
    return max(1, min(most, int(round(2 ** rng.uniform(0, most.bit_length())))))


def place(rng, x):
    """`x` on the GPU: dense, not aligned, or a part of something larger."""
    form = rng.randrange(3)
    if form == 0 or x.numel() == 0:
        return x.to(DEV)
    if form == 1:
        return torch.empty(x.numel() + 1, device=DEV, dtype=x.dtype)[1:].view(x.shape).copy_(x)
    wide = torch.full((x.shape[0], x.shape[1] + 2, *x.shape[2:-1], x.shape[-1] + 5), float("nan"), device=DEV, dtype=x.dtype)
    part = wide[:, 1:-1, ..., 2:2 + x.shape[-1]]
    return part.copy_(x)


@pytest.mark.parametrize("seed", range(60))
def test_group_norm(seed):
    import medvision_amd.ops as ops
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    groups = rng.choice([1, 1, 2, 3, 4, 7, 8, 16, 32])
    each = rng.choice([1, 2, 3, 4, 5, 6, 8, 10, 16, 24, 33, 64, 150])
    C, B = groups * each, size(rng, 12)
    N = size(rng, max(1, min(40000, 600000 // (B * C))))
    dtype, kind = rng.choice(TYPES), rng.choice([None, "relu", "leaky_relu", "silu", "gelu"])
    wide = rng.random() < 0.5
    middle = rng.choice([0.0, 0.0, 1.0, 30.0])
    x, go = (torch.randn(B, N, C, generator=g) * rng.choice([0.01, 1.0, 20.0]) + middle).to(dtype), torch.randn(B, N, C, generator=g).to(dtype)
    w, b = (torch.randn(C, generator=g).to(torch.float32 if wide else dtype) for _ in range(2))
    w, b = w if rng.random() < 0.8 else None, b if rng.random() < 0.8 else None
    eps, slope = rng.choice([1e-5, 1e-3]), rng.choice([0.01, 0.3])
    want = ref.group_norm(x, groups, w, b, eps, kind, slope, go)
    ins = [place(rng, x).requires_grad_(True), *(None if t is None else t.to(DEV).requires_grad_(True) for t in (w, b))]
    y = ops.group_norm_act(ins[0], groups, ins[1], ins[2], eps, kind, slope)
    grads = torch.autograd.grad(y, [t for t in ins if t is not None], place(rng, go))
    want = [v for v, keep in zip(want, (True, True, w is not None, b is not None)) if keep]
    for n, (got, (value, bound)) in enumerate(zip((y, *grads), want)):
        check(got, value, bound, (n, B, N, C, groups, dtype, kind, middle))


@pytest.mark.parametrize("seed", range(60))
def test_rotary(seed):
    import medvision_amd.ops as ops
    rng, g = random.Random(1000 + seed), torch.Generator().manual_seed(seed)
    B, H, D, A = size(rng, 6), size(rng, 20), size(rng, 160), rng.choice([1, 2, 3, 3, 4, 8])
    P, L = rng.randint(0, D // 2), size(rng, 400)
    dtype, neighbours = rng.choice(TYPES), rng.random() < 0.5
    x, go = torch.randn(B, L, H, D, generator=g).to(dtype), torch.randn(B, L, H, D, generator=g).to(dtype)
    at = rng.choice([1.0, 100.0, 1e5]) * torch.randn(*((B,) if rng.random() < 0.7 else ()), L, A, generator=g)
    at = at.to(rng.choice([torch.float32, torch.float64, torch.int64, torch.int32]))
    f = torch.randn(A, P, generator=g, dtype=rng.choice([torch.float32, torch.float64]))
    a = place(rng, x).requires_grad_(True)
    y = ops.rotary_positions(a, at.to(DEV), f.to(DEV), neighbours)
    dx, = torch.autograd.grad(y, a, place(rng, go))
    full = at.expand(B, L, A)
    what = (B, L, H, D, A, P, dtype, neighbours, at.dtype)
    check(y, *ref.rotary(x, full, f, neighbours), what)
    check(dx, *ref.rotary(go, full, f, neighbours, back=True), what)


@pytest.mark.parametrize("seed", range(80))
def test_group_linear(seed):
    import medvision_amd.ops as ops
    rng, g = random.Random(2000 + seed), torch.Generator().manual_seed(seed)
    M, K = size(rng, 700), size(rng, 9000)
    N = size(rng, max(1, min(1500, 40000000 // (M * K))))
    dtype, group = rng.choice(TYPES[1:]), rng.choice([32, 64, 128])
    x = torch.randn(1, M, K, generator=g).to(dtype)
    w = torch.randn(N, K, generator=g) * torch.exp(2 * torch.randn(N, 1, generator=g))
    bias = torch.randn(N, generator=g).to(dtype) if rng.random() < 0.5 else None
    codes, scales = ops.quantize_groups(w.to(DEV), group)
    want = ref.quantize_groups(w, group)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
    y = ops.group_linear(place(rng, x), codes, scales, None if bias is None else bias.to(DEV))
    check(y[0], *ref.group_linear(x[0], *want, bias), (M, K, N, group, dtype))
