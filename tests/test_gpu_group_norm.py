"""Group norm with an activation on the GPU against its 64-bit form."""
import pytest
import torch

import tokens_ref as ref
from decoder_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
KINDS = [None, "relu", "leaky_relu", "silu", "gelu"]
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def compare(x, groups, w, b, kind, grad, eps=1e-5, slope=0.01):
    import medvision_amd.ops as ops
    want = ref.group_norm(x, groups, w, b, eps, kind, slope, grad)
    ins = [None if t is None else t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = ops.group_norm_act(ins[0], groups, ins[1], ins[2], eps, kind, slope)
    grads = torch.autograd.grad(y, [t for t in ins if t is not None], grad.to(DEV))
    plain = ops.group_norm_act(x.to(DEV), groups, None if w is None else w.to(DEV), None if b is None else b.to(DEV), eps, kind, slope)
    assert torch.equal(plain, y) and y.dtype == x.dtype
    names = ["y", "dx"] + ["dw"] * (w is not None) + ["db"] * (b is not None)
    want = [v for v, keep in zip(want, (True, True, w is not None, b is not None)) if keep]
    for name, got, (value, bound) in zip(names, (y, *grads), want):
        check(got, value, bound, name)


SHAPES = [(1, 343, 256, 32), (2, 1, 16, 4), (3, 5, 6, 6), (2, 37, 60, 6), (1, 100, 2, 1), (2, 257, 20, 5), (1, 1000, 33, 3), (2, 50, 2056, 8), (1, 9, 2500, 1),
          (4, 777, 8, 8), (2, 3, 40, 1), (1, 5000, 12, 2), (2, 30000, 16, 4), (1, 2, 4096, 32), (5, 64, 1, 1), (1, 6000, 128, 1), (70, 3, 8, 2)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_shapes(shape, dtype):
    B, N, C, G = shape
    kind = KINDS[sum(shape) % 5]
    compare(rand(1, B, N, C, dtype=dtype), G, rand(2, C, dtype=dtype), rand(3, C, dtype=dtype), kind, rand(4, B, N, C, dtype=dtype))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
def test_activations(kind, dtype):
    x, w, b, go = rand(1, 2, 130, 24, dtype=dtype), rand(2, 24) * 3, rand(3, 24) * 3, rand(4, 2, 130, 24, dtype=dtype)
    compare(x, 4, w, b, kind, go, slope=0.2)
    compare(x.view(2, 13, 10, 24), 8, w.to(dtype), None, kind, go.view(2, 13, 10, 24), eps=1e-3)
    compare(x, 24, None, b.to(dtype), kind, go)
    compare(x, 1, None, None, kind, go)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 500, 16, 4), (1, 20000, 16, 4)])
def test_means_far_from_zero(dtype, shape):
    """Values around 1000, where the mean of squares loses the variance in 32 bits; the first cells are zeros."""
    B, N, C, G = shape
    x = 1000 + 8 * rand(1, B, N, C)
    x[:, :3] = 0
    compare(x.to(dtype), G, rand(2, C), rand(3, C), None, rand(4, B, N, C, dtype=dtype))


def test_constant_cells():
    import medvision_amd.ops as ops
    x = torch.full((2, 300, 16), 7.25, device=DEV, requires_grad=True)
    b = rand(1, 16).to(DEV)
    y = ops.group_norm_act(x, 4, None, b)
    assert torch.equal(y, b.expand_as(y))
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert (g == 0).all()


@pytest.mark.parametrize("N", [200, 40000])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_in_its_group(N, value):
    import medvision_amd.ops as ops
    x = rand(1, 2, N, 24)
    want = ops.group_norm_act(x.to(DEV), 4, activation="silu")
    x[1, N // 2, 7] = value   # group 1 of sample 1
    y = ops.group_norm_act(x.to(DEV), 4, activation="silu")
    bad = torch.isnan(y)
    assert bad[1, :, 6:12].all() and bad.sum() == N * 6
    assert torch.equal(y[~bad], want[~bad])


def test_empty_inputs():
    import medvision_amd.ops as ops
    w = torch.ones(8, device=DEV, requires_grad=True)
    for shape in ((0, 5, 8), (2, 0, 8), (2, 3, 0, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        y = ops.group_norm_act(x, 2, w, w, activation="gelu")
        assert y.shape == x.shape
        gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert gx.shape == x.shape and (gw == 0).all()
    x = rand(1, 3, 8).to(DEV)   # a cell per sample
    assert torch.allclose(ops.group_norm_act(x, 2), torch.nn.functional.group_norm(x, 2), atol=1e-5)


@pytest.mark.parametrize("N", [1, 3])
def test_large_batches(N):
    """More samples than a grid's third dimension has places; the same as a part of them."""
    import medvision_amd.ops as ops
    B, C = 70000, 40
    x, go, w = rand(1, B, N, C).to(DEV).requires_grad_(True), rand(2, B, N, C).to(DEV), rand(3, C).to(DEV).requires_grad_(True)
    y = ops.group_norm_act(x, 4, w, None, activation="silu")
    gx, gw = torch.autograd.grad(y, (x, w), go)
    part = x.detach()[-100:].requires_grad_(True)
    want = ops.group_norm_act(part, 4, w, None, activation="silu")
    wx, = torch.autograd.grad(want, part, go[-100:])
    assert torch.equal(y[-100:], want) and torch.equal(gx[-100:], wx)
    _, _, (dw, bound), _ = ref.group_norm(x, 4, w, None, 1e-5, "silu", grad=go)
    check(gw, dw, bound, "dw")


def test_values_whose_squares_are_too_large():
    """A variance that 32 bits do not hold: its group's cells are the bias, as the formula has it for an infinite variance."""
    import medvision_amd.ops as ops
    for N in (100, 20000):
        x = 1e25 * rand(1, 1, N, 16)
        y = ops.group_norm_act(x.to(DEV), 2, None, rand(2, 16).to(DEV))
        assert torch.isfinite(y).all()


def test_maps_in_either_order():
    """Tokens of a map: in channels-last order they are read as they are, others are copied; the same bits."""
    import medvision_amd.ops as ops
    m = ops.GroupNormAct(4, 32, activation="silu").to(DEV)
    maps = rand(1, 2, 32, 5, 6, 7).to(DEV)
    grads = []
    for order in (torch.contiguous_format, torch.channels_last_3d):
        f = maps.clone(memory_format=order).requires_grad_(True)
        y = m(ops.map_tokens(f))
        g, = torch.autograd.grad(y, f, torch.ones_like(y).cumsum(1))
        grads.append((y, g))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])
    view = torch.zeros(2, 50, 64, device=DEV, dtype=torch.float16)[:, 3:40, 5:29]   # rows that start anywhere
    view.copy_(rand(2, 2, 37, 24))
    assert torch.equal(ops.group_norm_act(view, 3), ops.group_norm_act(view.contiguous(), 3))
    flat = rand(5, 2 * 37 * 24 + 1, dtype=torch.float16).to(DEV)[1:].view(2, 37, 24)   # dense, not aligned
    assert torch.equal(ops.group_norm_act(flat, 3), ops.group_norm_act(flat.clone(), 3))


@pytest.mark.parametrize("kind,cells", [(None, 90), ("gelu", 90), ("silu", 7000)])
def test_gradients_of_some_inputs_and_both_forms_of_the_node(kind, cells):
    from medvision_amd.ops.group_norm import GroupNormActFunction

    class Python(GroupNormActFunction):
        @staticmethod
        def backward(ctx, grad):
            return GroupNormActFunction.backward(ctx, grad)

    tensors, go = (rand(1, 3, cells, 20), rand(2, 20), rand(3, 20)), rand(4, 3, cells, 20).to(DEV)

    def grads(function, wanted):
        ins = [t.to(DEV).requires_grad_(w) for t, w in zip(tensors, wanted)]
        y = function.apply(ins[0], 5, ins[1], ins[2], 1e-5, kind, 0.01)
        y.backward(go)
        return [y, *(t.grad for t in ins)]

    want = grads(GroupNormActFunction, (True, True, True))
    for function in (GroupNormActFunction, Python):
        for n in range(1, 8):
            wanted = tuple(bool(n >> i & 1) for i in range(3))
            got = grads(function, wanted)
            assert torch.equal(got[0], want[0])
            for a, b, w in zip(got[1:], want[1:], wanted):
                assert torch.equal(a, b) if w else a is None
    x = tensors[0].to(DEV)
    for weight, bias in ((None, tensors[2].to(DEV).requires_grad_(True)), (tensors[1].to(DEV).requires_grad_(True), None)):
        one = GroupNormActFunction.apply(x, 5, weight, bias, 1e-5, kind, 0.01)
        two = Python.apply(x, 5, weight, bias, 1e-5, kind, 0.01)
        leaf = weight if bias is None else bias
        assert torch.equal(one, two) and torch.equal(torch.autograd.grad(one, leaf, go)[0], torch.autograd.grad(two, leaf, go)[0])


def test_the_same_bits_each_time_and_on_another_stream():
    import medvision_amd.ops as ops
    x, w, go = rand(1, 2, 50000, 24, dtype=torch.float16).to(DEV).requires_grad_(True), rand(2, 24).to(DEV).requires_grad_(True), rand(3, 2, 50000, 24).half().to(DEV)

    def once():
        y = ops.group_norm_act(x, 6, w, w, activation="silu")
        return (y, *torch.autograd.grad(y, (x, w), go))

    want = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = once()
    side.synchronize()
    for a, b, c in zip(want, once(), other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_and_replayed():
    import medvision_amd.ops as ops
    x, w, go = (t.to(DEV) for t in (rand(1, 2, 9000, 24, dtype=torch.float16), rand(2, 24), rand(3, 2, 9000, 24, dtype=torch.float16)))

    def step(leaves):
        y = ops.group_norm_act(leaves[0], 6, leaves[1], leaves[1], activation="gelu")
        return (y, *torch.autograd.grad(y, leaves, go))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(2):
            step([x.clone().requires_grad_(True), w.clone().requires_grad_(True)])
    side.synchronize()
    leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    graphs = []
    for _ in range(2):   # two that share nothing
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(leaves)
        graphs.append((graph, out))
    for n in range(4):
        with torch.no_grad():
            leaves[0].copy_(rand(10 + n, 2, 9000, 24))
        for graph, out in graphs:
            graph.replay()
        want = step([t.detach().clone().requires_grad_(True) for t in leaves])
        torch.cuda.synchronize()
        for graph, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_refusals():
    import medvision_amd.ops as ops
    x, w = torch.zeros(2, 5, 12, device=DEV), torch.ones(12, device=DEV)
    for call, text in [(lambda: ops.group_norm_act(x, 5), "12 channels in 5 groups"), (lambda: ops.group_norm_act(x, 0), "in 0 groups"),
                       (lambda: ops.group_norm_act(x, 3, w[:6]), "weight has shape"), (lambda: ops.group_norm_act(x, 3, w, w.half()), "one dtype|bias has dtype"),
                       (lambda: ops.group_norm_act(x, 3, w.half()), "weight has dtype"), (lambda: ops.group_norm_act(x.double(), 3), "float32, float16 or bfloat16"),
                       (lambda: ops.group_norm_act(x, 3, w.cpu()), "weight is on cpu"), (lambda: ops.group_norm_act(x[0, 0], 3), "batch, ..., channels"),
                       (lambda: ops.group_norm_act(x, 3, activation="elu"), "activation 'elu'"),
                       (lambda: ops.group_norm_act(torch.zeros(65536, 6000, 1, device=DEV, dtype=torch.float16), 1), "a batch of 65536")]:
        with pytest.raises(RuntimeError, match=text):
            call()
    y = ops.group_norm_act(x.requires_grad_(True), 3)
    g, = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda t: ops.group_norm_act(t, 3), (x.detach(),), (torch.ones_like(x),))


def test_traced():
    import medvision_amd.ops as ops
    x = rand(1, 2, 30, 12).to(DEV)
    with torch.no_grad():
        traced = torch.jit.trace(lambda t: ops.group_norm_act(t, 3, None, None, 1e-5, "silu"), (x,))
        assert torch.equal(traced(x * 2 + 1), ops.group_norm_act(x * 2 + 1, 3, activation="silu"))


def test_offsets_past_32_bits():
    """2.2e9 elements: the last sample is the same as by itself."""
    import medvision_amd.ops as ops
    B, N, C = 3, 11500000, 64
    x = torch.zeros(B, N, C, device=DEV, dtype=torch.float16)
    last = torch.randn(N, C, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV, dtype=torch.float16)
    x[2] = last
    w = rand(2, C).to(DEV)
    ins = [x.requires_grad_(True), w.requires_grad_(True)]
    y = ops.group_norm_act(ins[0], 8, ins[1], None, activation="silu")
    go = torch.zeros_like(x)
    go[2] = last.flip(0)
    gx, gw = torch.autograd.grad(y, ins, go)
    alone = last[None].clone().requires_grad_(True)
    want = ops.group_norm_act(alone, 8, ins[1], None, activation="silu")
    wx, ww = torch.autograd.grad(want, (alone, ins[1]), last.flip(0)[None])
    # (the cells are shared out to workgroups in other ways: sums in another order)
    assert (y[2].float() - want[0].float()).abs().max() <= 2.0 ** -10 * 8 and (y[:2] == 0).all()
    assert (gx[2].float() - wx[0].float()).abs().max() <= 2.0 ** -10 * 8 and (gx[:2] == 0).all()
    assert (gw - ww).norm() <= 1e-4 * ww.norm()
