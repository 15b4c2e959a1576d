"""Traces of the operators and layers without a gradient: on other inputs they give what the calls give."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def compare(call, *inputs):
    """`call` traced with `inputs` and run on others, what memory held in between overwritten."""
    with torch.no_grad():
        traced = torch.jit.trace(call, inputs, check_trace=False)
        for n in range(2):
            other = tuple(t * (2.0 + n) + 0.5 if t.is_floating_point() else t for t in inputs)
            want = call(*other)
            junk = [torch.full((1 << 20,), float("nan"), device=DEV) for _ in range(8)]
            del junk
            got = traced(*other)
            for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                assert a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("rows", [1, 20, 200])
def test_4_bit_products(rows, group):
    import medvision_amd.ops as ops
    layer = ops.GroupScaledLinear.from_linear(torch.nn.Linear(300, 70).to(DEV), group, torch.float16)
    compare(layer, rand(1, rows, 300))
    compare(lambda w: ops.quantize_groups(w, group), rand(2, rows, 300))


def test_8_bit_products():
    import medvision_amd.ops as ops
    layer = ops.BlockScaledLinear.from_linear(torch.nn.Linear(300, 70).to(DEV), torch.float16)
    compare(layer, rand(1, 20, 300))
    compare(lambda w: ops.quantize_blocks(w, 128), rand(2, 200, 300))
    w = rand(3, 300)
    compare(lambda x: ops.add_rms_norm_quantized(x, None, w)[:2], rand(4, 20, 300))
    compare(lambda x, r: ops.add_rms_norm_quantized(x, r, w), rand(4, 20, 300), rand(5, 20, 300))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("axes", [0, 3])
def test_layers_for_inference(bits, axes):
    import medvision_amd.ops as ops
    torch.manual_seed(1)
    layer = ops.RegionDecoderLayer(96, 6, hidden=200, key_heads=3, axes=axes).to(DEV).for_inference(torch.float16, bits=bits)
    regions, residual, tokens = (rand(n, 2, rows, 96, dtype=torch.float16) for n, rows in ((2, 33), (3, 33), (4, 50)))
    if axes:
        compare(lambda r, h, t, p, c: layer(r, t, h, region_positions=p, token_positions=c), regions, residual, tokens, rand(5, 2, 33, 3), rand(6, 50, 3))
    else:
        compare(lambda r, h, t: layer(r, t, h), regions, residual, tokens)
        compare(lambda r, t: layer(r, t), regions, tokens)   # (the first layer: no residual)


def test_resampling():
    import medvision_amd.ops as ops
    image, volume = rand(1, 2, 3, 20, 24), rand(2, 1, 2, 10, 12, 14)
    rois2 = torch.tensor([[0, 10., 9., 12., 10., 0.3], [1, 12., 10., 20., 16., 0.0]], device=DEV)
    rois3 = torch.tensor([[0, 6., 5., 5., 8., 8., 6., 0.1, 0.2, 0.0]], device=DEV)
    compare(lambda t: ops.affine_2d(t, rois2, (9, 11), 1.0), image)
    compare(lambda t: ops.affine_3d(t, rois3, (5, 6, 7), 1.0, order=3), volume)
    move2, move3 = rand(3, 2, 2, 20, 24), rand(4, 1, 3, 10, 12, 14)
    compare(lambda t: ops.apply_offset_2d(t, move2), image)
    compare(lambda t: ops.apply_offset_3d(t, move3), volume)
