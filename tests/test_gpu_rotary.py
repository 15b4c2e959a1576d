"""Rotary positions on several axes on the GPU against their 64-bit form."""
import pytest
import torch

import tokens_ref as ref
from decoder_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def places(seed, *shape, size=100.0):
    return size * (torch.rand(shape, generator=torch.Generator().manual_seed(seed)) - 0.3)


# batch, rows, heads, channels, axes, pairs
SHAPES = [(1, 1, 8, 32, 3, 15), (2, 50, 3, 64, 3, 30), (2, 7, 2, 13, 2, 6), (1, 300, 1, 2, 1, 1), (3, 33, 6, 40, 2, 18), (1, 5, 64, 128, 4, 64), (2, 3, 2, 1024, 3, 510),
          (1, 70, 4, 20, 1, 10), (2, 9, 5, 96, 8, 33), (1, 2, 100, 100, 2, 50), (2, 17, 2, 16, 3, 3), (1, 4, 1, 1, 1, 0), (4, 1000, 1, 12, 3, 6)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("neighbours", [False, True])
def test_shapes(shape, dtype, neighbours):
    import medvision_amd.ops as ops
    B, L, H, D, A, P = shape
    x, go = rand(1, B, L, H, D, dtype=dtype), rand(2, B, L, H, D, dtype=dtype)
    at, f = places(3, B, L, A), torch.rand(A, P, generator=torch.Generator().manual_seed(4), dtype=torch.float64)
    a = x.to(DEV).requires_grad_(True)
    y = ops.rotary_positions(a, at.to(DEV), f.to(DEV), neighbours)
    g, = torch.autograd.grad(y, a, go.to(DEV))
    check(y, *ref.rotary(x, at, f, neighbours), "y")
    check(g, *ref.rotary(go, at, f, neighbours, back=True), "dx")
    assert torch.equal(y[..., 2 * P:], a[..., 2 * P:]) and torch.equal(g.cpu()[..., 2 * P:], go[..., 2 * P:])
    assert torch.equal(ops.rotary_positions(x.to(DEV), at.to(DEV), f.to(DEV), neighbours), y)
    shared = ops.rotary_positions(a, at[0].to(DEV), f.to(DEV), neighbours)
    check(shared, *ref.rotary(x, at[:1].expand(B, L, A), f, neighbours), "positions for all samples")


@pytest.mark.parametrize("kind", [torch.float64, torch.float32, torch.float16, torch.bfloat16, torch.int64, torch.int32, torch.int16, torch.uint8])
def test_types_of_positions(kind):
    import medvision_amd.ops as ops
    x, f = rand(1, 2, 40, 3, 24), torch.rand(2, 12, generator=torch.Generator().manual_seed(4))
    at = places(3, 2, 40, 2).abs().to(kind)
    y = ops.rotary_positions(x.to(DEV), at.to(DEV), f.to(DEV))
    check(y, *ref.rotary(x, at, f, False), kind)
    assert torch.equal(y, ops.rotary_positions(x.to(DEV), at.double().to(DEV), f.double().to(DEV)))


def test_far_places():
    """Around 1e7 a turn is lost in 32 bits; whole positions beyond 2^31."""
    import medvision_amd.ops as ops
    x, f = rand(1, 1, 64, 2, 16), torch.rand(1, 8, generator=torch.Generator().manual_seed(4), dtype=torch.float64)
    for at in (1e7 + torch.arange(64.).view(64, 1), (2 ** 33 + torch.arange(64)).view(64, 1), -1e6 * torch.rand(64, 1, generator=torch.Generator().manual_seed(5), dtype=torch.float64)):
        check(ops.rotary_positions(x.to(DEV), at.to(DEV), f.to(DEV)), *ref.rotary(x, at, f, False), "far")


def test_quarters_and_whole_turns():
    import math
    import medvision_amd.ops as ops
    x = rand(1, 1, 9, 1, 2)
    at = torch.arange(-4, 5).view(9, 1)
    y = ops.rotary_positions(x.to(DEV), at.to(DEV), torch.tensor([[math.pi / 2]], dtype=torch.float64, device=DEV)).cpu()[0, :, 0]
    a, b = x[0, :, 0].unbind(-1)
    want = torch.stack([torch.stack([(a, -b, -a, b)[n % 4][i], (b, a, -b, -a)[n % 4][i]]) for i, n in enumerate(range(-4, 5))])
    assert (y - want).abs().max() <= 2.0 ** -22 * x.abs().max()
    assert torch.equal(y[4], x[0, 4, 0])   # position zero


def test_products_depend_on_distances():
    import medvision_amd.ops as ops
    q, k = rand(1, 1, 20, 2, 30).double(), rand(2, 1, 20, 2, 30).double()
    f, at = ops.axis_frequencies(30).to(DEV), places(3, 20, 3)
    turned = [ops.rotary_positions(t.float().to(DEV), p.to(DEV), f).double().cpu() for p in (at, at + 32.0) for t in (q, k)]
    one, two = (torch.einsum("bihd,bjhd->bhij", *turned[i:i + 2]) for i in (0, 2))
    assert (one - two).abs().max() <= 1e-4   # positions around 100 are rounded by 4e-6 when they are moved
    plain = torch.einsum("bihd,bjhd->bhij", q, k)
    assert (torch.diagonal(one, 0, 2, 3) - torch.diagonal(plain, 0, 2, 3)).abs().max() <= 1e-4


def test_strides():
    """Keys as one of two heads of a product, positions of a batch that share memory, rows in another order."""
    import medvision_amd.ops as ops
    both = rand(1, 2, 30, 2, 4, 24, dtype=torch.float16).to(DEV)
    key = both.unbind(2)[0]
    f, at = ops.axis_frequencies(24).to(DEV), places(3, 30, 3).to(DEV)
    want = ops.rotary_positions(key.contiguous(), at, f)
    assert torch.equal(ops.rotary_positions(key, at, f), want) and torch.equal(ops.rotary_positions(key, at.expand(2, 30, 3), f), want)
    assert torch.equal(ops.rotary_positions(key, at.t().contiguous().t(), f), want)
    assert torch.equal(ops.rotary_positions(key.transpose(1, 2).contiguous().transpose(1, 2), at, f), want)
    assert torch.equal(ops.rotary_positions(key.transpose(2, 3).contiguous().transpose(2, 3), at, f), want)   # (channels apart: copied)
    assert torch.equal(ops.rotary_positions(key[:1].expand(5, 30, 4, 24), at, f)[4], want[0])
    flat = torch.empty(key.numel() + 1, device=DEV, dtype=torch.float16)[1:].view(key.shape).copy_(key)   # not aligned
    assert torch.equal(ops.rotary_positions(flat, at, f), want) and want.is_contiguous()
    leaf = both.clone().requires_grad_(True)
    g, = torch.autograd.grad(ops.rotary_positions(leaf.unbind(2)[0], at, f), leaf, want)
    assert torch.equal(g[:, :, 1], torch.zeros_like(g[:, :, 1])) and (g[:, :, 0].float() - key.float()).abs().max() <= 2.0 ** -9 * key.abs().max()
    grad = rand(5, 4, 2, 30, 24, dtype=torch.float16).to(DEV).permute(1, 2, 0, 3)   # a gradient in another order
    plain = key.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(ops.rotary_positions(plain, at, f), plain, grad)[0],
                       torch.autograd.grad(ops.rotary_positions(plain, at, f), plain, grad.contiguous())[0])


def test_what_is_not_finite_stays_in_its_row():
    import medvision_amd.ops as ops
    x, f, at = rand(1, 2, 20, 3, 16).to(DEV), torch.rand(2, 8, device=DEV), places(3, 2, 20, 2).to(DEV)
    want = ops.rotary_positions(x, at, f)
    for value in (float("nan"), float("inf")):
        at[1, 7, 0] = value
        y = ops.rotary_positions(x, at, f)
        bad = torch.isnan(y)
        assert bad[1, 7].all() and bad.sum() == 48 and torch.equal(y[~bad], want[~bad])


def test_empty_inputs():
    import medvision_amd.ops as ops
    f = torch.rand(2, 4, device=DEV)
    for shape in ((0, 5, 2, 8), (2, 0, 2, 8), (2, 5, 0, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        y = ops.rotary_positions(x, torch.zeros(shape[1], 2, device=DEV), f)
        assert y.shape == x.shape and torch.autograd.grad(y, x, y)[0].shape == x.shape


def test_both_forms_of_the_node_streams_and_replays():
    import medvision_amd.ops as ops
    from medvision_amd.ops.rotary import RotaryPositionsFunction

    class Python(RotaryPositionsFunction):
        @staticmethod
        def backward(ctx, grad):
            return RotaryPositionsFunction.backward(ctx, grad)

    at, f, go = places(3, 2, 500, 3).to(DEV), ops.axis_frequencies(32).to(DEV), rand(2, 2, 500, 4, 32).to(DEV)
    x = rand(1, 2, 500, 4, 32).to(DEV)

    def step(function, leaf):
        y = function.apply(leaf, at, f, True)
        return (y, *torch.autograd.grad(y, leaf, go))

    want = step(RotaryPositionsFunction, x.clone().requires_grad_(True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(RotaryPositionsFunction, x.clone().requires_grad_(True))
    side.synchronize()
    for a, b, c in zip(want, step(Python, x.clone().requires_grad_(True)), other):
        assert torch.equal(a, b) and torch.equal(a, c)
    leaf, graph = x.clone().requires_grad_(True), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(RotaryPositionsFunction, leaf)
    for n in range(3):
        with torch.no_grad():
            leaf.copy_(rand(10 + n, 2, 500, 4, 32))
            at.add_(1.5)
        graph.replay()
        for a, b in zip(out, step(RotaryPositionsFunction, leaf.detach().clone().requires_grad_(True))):
            assert torch.equal(a, b)
    with torch.no_grad():
        traced = torch.jit.trace(lambda t: ops.rotary_positions(t, at, f), (x,))
        assert torch.equal(traced(x + 1), ops.rotary_positions(x + 1, at, f))


def test_refusals():
    import medvision_amd.ops as ops
    x, at, f = torch.zeros(2, 5, 3, 16, device=DEV), torch.zeros(2, 5, 2, device=DEV), torch.zeros(2, 8, device=DEV)
    for call, text in [(lambda: ops.rotary_positions(x[0], at, f), "batch, rows, heads, channels"), (lambda: ops.rotary_positions(x, at[:1], f), "positions have shape"),
                       (lambda: ops.rotary_positions(x, at[:, :4], f), "positions have shape"), (lambda: ops.rotary_positions(x, at[..., :1], f), "positions have shape"),
                       (lambda: ops.rotary_positions(x, at, torch.zeros(2, 9, device=DEV)), "frequencies have shape"), (lambda: ops.rotary_positions(x, at, f[0]), "frequencies have shape"),
                       (lambda: ops.rotary_positions(x, torch.zeros(2, 5, 9, device=DEV), torch.zeros(9, 8, device=DEV)), "frequencies have shape"),
                       (lambda: ops.rotary_positions(x, at, f.half()), "frequencies have to be"), (lambda: ops.rotary_positions(x, at.bool(), f), "positions have to be"),
                       (lambda: ops.rotary_positions(x.double(), at, f), "float32, float16 or bfloat16"), (lambda: ops.rotary_positions(x, at.cpu(), f), "positions is on cpu"),
                       (lambda: ops.rotary_positions(x, at, f.cpu()), "frequencies is on cpu"), (lambda: ops.rotary_positions(x, at.requires_grad_(True), f), "no gradient for positions"),
                       (lambda: ops.rotary_positions(x, at.detach(), f.requires_grad_(True)), "no gradient for positions"),
                       (lambda: ops.rotary_positions(torch.zeros(1, 5, 1, 1026, device=DEV), at[0].detach(), f.detach()), "1 to 1024")]:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_offsets_past_32_bits():
    import medvision_amd.ops as ops
    B, L, H, D = 3, 700000, 16, 68
    x = torch.zeros(B, L, H, D, device=DEV, dtype=torch.float16)
    last = torch.randn(L, H, D, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV, dtype=torch.float16)
    x[2] = last
    at, f = 100 * torch.rand(L, 3, device=DEV), ops.axis_frequencies(D).to(DEV)
    y = ops.rotary_positions(x, at, f)
    assert torch.equal(y[2:], ops.rotary_positions(last[None], at, f)) and (y[:2] == 0).all()
