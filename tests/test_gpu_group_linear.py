"""Products with 4-bit weights on the GPU against their 64-bit form, and the quantiser bit for bit."""
import pytest
import torch

import tokens_ref as ref
from decoder_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (5, 128), (3, 200), (17, 33), (130, 1000), (2, 127), (1, 4097)])
def test_quantiser(group, dtype, shape):
    import medvision_amd.ops as ops
    w = rand(1, *shape, dtype=dtype)
    w[0, 0] = 0
    codes, scales = ops.quantize_groups(w.to(DEV), group)
    want, want_scales = ref.quantize_groups(w, group)
    assert torch.equal(codes.cpu(), want) and torch.equal(scales.cpu(), want_scales)


def test_quantiser_at_halves_and_extremes():
    import medvision_amd.ops as ops
    w = torch.tensor([0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5] + [0.] * 16).repeat(9, 4)
    w[1] *= 2.0 ** -120    # scales at and below 2^-126
    w[2] *= 2.0 ** -140
    w[3] = 0
    w[4, 37] = float("nan")
    w[5, 69] = float("inf")
    w[6] *= 2.0 ** 120
    codes, scales = ops.quantize_groups(w.to(DEV))
    want, want_scales = ref.quantize_groups(w, 32)
    fine = torch.tensor([0, 1, 2, 3, 6, 7, 8])
    assert torch.equal(codes.cpu()[fine], want[fine]) and torch.equal(scales.cpu()[fine], want_scales[fine])
    assert torch.isnan(scales[4, 1]) and torch.isinf(scales[5, 2]) and torch.isfinite(scales[4, 0]) and torch.isfinite(scales[5, 3])
    y = ops.group_linear(torch.ones(1, 128, device=DEV, dtype=torch.bfloat16), codes, scales).cpu()[0]
    assert torch.isnan(y[4]) and torch.isnan(y[5]) and torch.isfinite(y[fine]).all()
    empty = ops.quantize_groups(torch.zeros(0, 70, device=DEV))
    assert empty[0].shape == (0, 64) and empty[1].shape == (0, 4)


# rows, inputs, outputs
SHAPES = [(1, 256, 1024), (1, 1, 1), (2, 7, 17), (5, 31, 64), (16, 128, 65), (17, 129, 33), (13, 1000, 130), (33, 640, 16), (64, 200, 100), (65, 2048, 70), (130, 384, 200),
          (300, 1111, 257), (1, 20000, 40), (3, 8192, 300), (200, 64, 8), (1000, 512, 512), (2, 4096, 2), (31, 12544, 48)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_products(shape, dtype, group):
    import medvision_amd.ops as ops
    M, K, N = shape
    x, bias = rand(1, M, K, dtype=dtype), rand(2, N, dtype=dtype) if (M + group) % 3 else None
    codes, scales = ref.quantize_groups(rand(3, N, K) * torch.exp(rand(4, N, 1)), group)
    got = ops.group_linear(x.to(DEV), codes.to(DEV), scales.to(DEV), None if bias is None else bias.to(DEV))
    assert got.dtype == dtype
    check(got, *ref.group_linear(x, codes, scales, bias), shape)
    again = ops.group_linear(x.to(DEV), codes.to(DEV), scales.to(DEV), None if bias is None else bias.to(DEV))
    assert torch.equal(got, again)


@pytest.mark.parametrize("shape", [(1000, 20011), (1024, 16384), (640, 50000), (500, 33333), (384, 40002), (200, 70001), (128, 66000)])
@pytest.mark.parametrize("rows", [1, 2, 13, 20, 64])
def test_many_outputs_of_short_rows(rows, shape):
    import medvision_amd.ops as ops
    K, N = shape
    dtype, group = (torch.float16, torch.bfloat16)[K % 3 % 2], (32, 64, 128)[(K + rows) % 3]
    x, bias = rand(1, rows, K, dtype=dtype), rand(2, N, dtype=dtype)
    codes, scales = (t.cpu() for t in ops.quantize_groups(rand(3, N, K).to(DEV), group))
    got = ops.group_linear(x.to(DEV), codes.to(DEV), scales.to(DEV), bias.to(DEV))
    check(got, *ref.group_linear(x, codes, scales, bias), shape)


def test_every_code_and_place():
    """A row of x with a single one picks a column; every column of a block, with all sixteen codes."""
    import medvision_amd.ops as ops
    for dtype in (torch.float16, torch.bfloat16):
        for group in (32, 64, 128):
            codes = torch.randint(0, 256, (48, 128), generator=torch.Generator().manual_seed(1), dtype=torch.uint8)
            scales = 0.5 + torch.rand(48, 256 // group, generator=torch.Generator().manual_seed(2))
            scales = scales.to(dtype).float()   # (products with codes of up to three bits round once)
            x = torch.eye(256, dtype=dtype)
            y = ops.group_linear(x.to(DEV), codes.to(DEV), scales.to(DEV))
            assert torch.equal(y.cpu(), ref.group_values(codes, scales, 256).t().to(dtype))


@pytest.mark.parametrize("rows", [1, 3, 20, 200])
@pytest.mark.parametrize("inputs", [90, 100, 127, 1000, 1003])
def test_what_is_not_finite_stays_in_its_row(rows, inputs):
    """Rows end anywhere: what the next one holds is not read into them, nor is what stands behind the last one."""
    import medvision_amd.ops as ops
    codes, scales = ref.quantize_groups(rand(3, 70, inputs), 32)
    codes, scales = codes.to(DEV), scales.to(DEV)
    x = rand(1, rows, inputs, dtype=torch.float16).to(DEV)
    want = ops.group_linear(x, codes, scales)
    space = torch.full((rows * inputs + 200,), float("nan"), device=DEV, dtype=torch.float16)
    inside = space[7:7 + rows * inputs].view(rows, inputs).copy_(x)   # not aligned, NaN on both sides
    assert torch.equal(ops.group_linear(inside, codes, scales), want)
    x[rows // 2] = float("nan")
    y = ops.group_linear(x, codes, scales)
    assert torch.isnan(y[rows // 2]).all()
    keep = torch.arange(rows, device=DEV) != rows // 2
    assert torch.equal(y[keep], want[keep])


@pytest.mark.parametrize("rows", [1, 2, 13, 40, 200])
def test_small_values(rows):
    """float16 below its least normal value counts in full: whole multiples of 2^-24, and sums that are exact in 32 bits."""
    import medvision_amd.ops as ops
    codes, scales = ref.quantize_groups(rand(3, 70, 200), 32)
    scales = torch.full_like(scales, 2.0 ** 12)
    x = torch.randint(-15, 16, (rows, 200), generator=torch.Generator().manual_seed(5)).double() * 2.0 ** -24
    y = ops.group_linear(x.half().to(DEV), codes.to(DEV), scales.to(DEV))
    assert torch.equal(y.cpu(), (x @ ref.group_values(codes, scales, 200).t()).half())


def test_layouts():
    import medvision_amd.ops as ops
    codes, scales = (t.to(DEV) for t in ref.quantize_groups(rand(3, 70, 300), 64))
    x = rand(1, 4, 5, 300, dtype=torch.bfloat16).to(DEV)
    want = ops.group_linear(x.flatten(0, 1), codes, scales).view(4, 5, 70)
    assert torch.equal(ops.group_linear(x, codes, scales), want)
    assert torch.equal(ops.group_linear(x.transpose(0, 1).contiguous().transpose(0, 1), codes, scales), want)
    moved = torch.empty(codes.numel() + 1, device=DEV, dtype=torch.uint8)[1:].view(codes.shape).copy_(codes)   # not aligned: copied
    assert torch.equal(ops.group_linear(x, moved, scales), want)
    assert torch.equal(ops.group_linear(x, codes.t().contiguous().t(), scales.t().contiguous().t()), want)
    assert torch.equal(ops.group_linear(x[0, 0], codes, scales), ops.group_linear(x[0, :1], codes, scales)[0])
    for shape in ((0, 300), (3, 0, 300)):
        assert ops.group_linear(torch.zeros(shape, device=DEV, dtype=torch.float16), codes, scales).shape == (*shape[:-1], 70)
    assert ops.group_linear(x, codes[:0], scales[:0]).shape == (4, 5, 0)


def test_without_a_workspace():
    """The same product in one piece."""
    from medvision_amd import _lib
    lib = _lib.load()
    M, K, N = 3, 20000, 50
    codes, scales = ref.quantize_groups(rand(3, N, K), 128)
    x, bias = rand(1, M, K, dtype=torch.float16), rand(2, N, dtype=torch.float16)
    assert lib.mv_group_linear_workspace_bytes(M, K, N) > 0
    t = [v.to(DEV) for v in (x, codes, scales, bias)]
    y = torch.full((M, N), 7.0, device=DEV, dtype=torch.float16)
    assert lib.mv_group_linear(*(v.data_ptr() for v in t), y.data_ptr(), M, K, N, 128, _lib.MV_F16, None, 0, torch.cuda.current_stream().cuda_stream) == 0
    check(y, *ref.group_linear(x, codes, scales, bias), "no workspace")


def test_streams_and_replays():
    import medvision_amd.ops as ops
    sizes = [(1, 9000, 64), (40, 2048, 256), (300, 512, 128), (200, 4099, 100)]
    layers = [tuple(t.to(DEV) for t in ref.quantize_groups(rand(n, size[2], size[1]), 32)) for n, size in enumerate(sizes)]
    xs = [rand(9 + n, size[0], size[1], dtype=torch.float16).to(DEV) for n, size in enumerate(sizes)]
    step = lambda: [ops.group_linear(x, *w) for x, w in zip(xs, layers)]   # noqa: E731
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for n in range(3):
        for x in xs:
            x.mul_(1.25)
        for graph, _ in graphs:
            graph.replay()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    import medvision_amd.ops as ops
    x, w, s = torch.zeros(2, 200, device=DEV, dtype=torch.float16), torch.zeros(8, 128, device=DEV, dtype=torch.uint8), torch.ones(8, 8, device=DEV)
    for call, text in [(lambda: ops.group_linear(x.float(), w, s), "float16 or bfloat16"), (lambda: ops.group_linear(x, w.short(), s), "uint8 and float32"),
                       (lambda: ops.group_linear(x, w, s.half()), "uint8 and float32"), (lambda: ops.group_linear(x[:, :100], w, s), "weight has shape"),
                       (lambda: ops.group_linear(x, w[:, :64], s), "weight has shape"), (lambda: ops.group_linear(x, w, s[:, :3]), "scales have shape"),
                       (lambda: ops.group_linear(x, w, s[:7]), "scales have shape"), (lambda: ops.group_linear(x, w, s, s[0, :7]), "bias has shape"),
                       (lambda: ops.group_linear(x, w.cpu(), s), "weight is on cpu"), (lambda: ops.group_linear(x, w, s.cpu()), "scales is on cpu"),
                       (lambda: ops.group_linear(x.requires_grad_(True), w, s), "no gradient"), (lambda: ops.quantize_groups(s, 16), "groups of 16"),
                       (lambda: ops.quantize_groups(s[0]), "takes a matrix"), (lambda: ops.quantize_groups(s.double()), "float32, float16 or bfloat16"),
                       (lambda: ops.quantize_groups(s.clone().requires_grad_(True)), "no gradient")]:
        with pytest.raises(RuntimeError, match=text):
            call()
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda t: ops.group_linear(t, w, s), (x.detach(),), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: ops.group_linear(t, w, s))(x.detach()[None])


def test_module():
    import medvision_amd.ops as ops
    linear = torch.nn.Linear(200, 70).to(DEV)
    for group, dtype in ((32, torch.bfloat16), (128, torch.float16)):
        layer = ops.GroupScaledLinear.from_linear(linear, group, dtype)
        x = rand(1, 3, 200).to(DEV)
        y = layer(x)
        assert y.dtype == dtype
        check(y, *ref.group_linear(x.to(dtype), layer.weight, layer.scales, linear.bias.detach()), "module")
        other = ops.GroupScaledLinear(200, 70, group=group, dtype=dtype).to(DEV)
        other.load_state_dict(layer.state_dict())
        assert torch.equal(other.half()(x.to(dtype)), y)


def test_weights_past_32_bits():
    """2.2e9 bytes of weights: the last outputs are the same as by themselves."""
    import medvision_amd.ops as ops
    K, N = 87808, 50000
    codes = torch.randint(0, 256, (N, K // 2), device=DEV, dtype=torch.uint8, generator=torch.Generator(device=DEV).manual_seed(1))
    scales = torch.rand(N, K // 128, device=DEV)
    for rows in (1, 40):
        x = rand(2, rows, K, dtype=torch.bfloat16).to(DEV)
        y = ops.group_linear(x, codes, scales)[:, -100:]
        alone, bound = ref.group_linear(x.cpu()[:1], codes[-100:], scales[-100:], None)
        check(y[:1], alone, bound, "last outputs")
