"""The decoder layer where types meet: autocast with regions in float32, serving of float32 regions."""
import pytest
import torch

from test_gpu_region_decoder import case, plain_layer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("carried", [True, False])
def test_layers_under_autocast(dtype, carried):
    """Learned queries in float32 through two layers.  Of a layer's six products one after the other each rounds both operands and its
    result to 16 bits; all of a pair of layers adding up: 36 unit roundoffs, and twice that for the gradients."""
    layer, regions, tokens, residual, lengths, keep = case(torch.float32)
    residual = residual if carried else None
    ins = [t.double().requires_grad_(True) for t in (regions, tokens)]
    layer = layer.double()
    want = plain_layer(layer, *plain_layer(layer, *ins, None if residual is None else residual.double(), keep)[:1], ins[1], ins[0], keep)
    grads = [torch.randn_like(t) for t in want]
    want_grads = torch.autograd.grad(want, [*ins, *layer.parameters()], grads)
    layer = layer.float().to(DEV)
    got_ins = [t.to(DEV).requires_grad_(True) for t in (regions, tokens)]
    with torch.autocast("cuda", dtype=dtype):
        first = layer(*got_ins, None if residual is None else residual.to(DEV), key_lengths=lengths.to(DEV))
        assert first[1].dtype == torch.float32
        got = layer(first[0], got_ins[1], got_ins[0], key_lengths=lengths.to(DEV))
    assert got[1].dtype == torch.float32
    unit = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    for a, b in zip(got, want):
        assert (a.double().cpu() - b).norm() <= 36 * unit * b.norm()
    got_grads = torch.autograd.grad(got, [*got_ins, *layer.parameters()], [g.to(a.dtype).to(DEV) for g, a in zip(grads, got)])
    for a, b in zip(got_grads, want_grads):
        assert a.dtype == torch.float32 and (a.double().cpu() - b).norm() <= 72 * unit * b.norm()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_float32_regions_are_served(dtype):
    """The sum that is carried stays in float32; five products in 8 bits on the longest way, 3.7 % each."""
    layer, regions, tokens, residual, lengths, keep = case(torch.float32)
    with torch.no_grad():
        want = sum(plain_layer(layer.double(), regions.double(), tokens.double(), residual.double(), keep))
        fast = layer.float().to(DEV).for_inference(dtype)
        for given in (residual.to(DEV), None):
            y, carried = fast(regions.to(DEV), tokens.to(DEV), given, key_lengths=lengths.to(DEV))
            assert y.dtype == dtype and carried.dtype == torch.float32
            if given is not None:
                assert ((y + carried).double().cpu() - want).norm() <= 5 * 0.037 * want.norm()
        again, carried = fast(y, tokens.to(DEV), carried, key_lengths=lengths.to(DEV))
        assert carried.dtype == torch.float32 and torch.isfinite(again).all()


def test_layers_of_16_bits_are_served():
    layer, regions, tokens, residual, lengths, _ = case(torch.bfloat16)
    with torch.no_grad():
        whole = layer.to(DEV).bfloat16()
        out = whole.for_inference(torch.bfloat16)(*(t.to(DEV).bfloat16() for t in (regions, tokens, residual)), key_lengths=lengths.to(DEV))
    assert all(t.dtype == torch.bfloat16 and torch.isfinite(t).all() for t in out)
    assert whole.norm_query.weight.dtype == torch.bfloat16


def test_hooks_stay_with_their_layer():
    """Hooks that are registered on the layer or on its form for inference run for that one alone; buffers are each one's own."""
    layer, regions, tokens, *_ = case(torch.float32)
    layer = layer.to(DEV)
    before, after = [], []
    layer.register_forward_hook(lambda *_: before.append(1))
    with torch.no_grad():
        fast = layer.for_inference(torch.float16)
        fast.register_forward_hook(lambda *_: after.append("fast"))
        layer.register_forward_pre_hook(lambda *_: after.append("layer"))
        fast.register_buffer("extra", torch.zeros(1))
        layer(regions.to(DEV), tokens.to(DEV))
        assert after == ["layer"]
        fast(regions.to(DEV).half(), tokens.to(DEV).half())
        assert after == ["layer", "fast"] and len(before) == 2   # (what was registered before goes along)
    assert "extra" not in dict(layer.named_buffers()) and layer.training and not fast.training
