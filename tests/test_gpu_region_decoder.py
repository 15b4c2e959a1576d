"""The decoder layer that runs the operators together, and the example that uses it."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def plain_layer(layer, regions, tokens, residual, keep):
    """The layer in elementary operations."""
    norm = lambda m, x: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + m.eps) * m.weight.to(x)   # noqa: E731
    linear = lambda m, x: x @ m.weight.to(x).t() + (0 if m.bias is None else m.bias.to(x))   # noqa: E731
    h = regions if residual is None else regions + residual
    q = linear(layer.query, norm(layer.norm_query, h)).unflatten(-1, (layer.heads, -1)).transpose(1, 2)
    kv = linear(layer.key_value, tokens).unflatten(-1, (2, layer.key_heads, -1)).permute(2, 0, 3, 1, 4)
    k, v = (t.repeat_interleave(layer.heads // layer.key_heads, 1) for t in kv)
    s = q @ k.transpose(-1, -2) * layer.head_channels ** -0.5
    p = torch.softmax(s.masked_fill(~keep[:, None, None], float("-inf")), -1)
    h = linear(layer.out, (p @ v).transpose(1, 2).flatten(2)) + h
    return linear(layer.down, torch.relu(linear(layer.up, norm(layer.norm_hidden, h)))), h


def case(dtype, channels=96, heads=6, key_heads=3):
    import medvision_amd.ops as ops
    torch.manual_seed(1)
    layer = ops.RegionDecoderLayer(channels, heads, hidden=200, key_heads=key_heads)
    regions, tokens, residual = torch.randn(2, 33, channels), torch.randn(2, 140, channels), torch.randn(2, 33, channels)
    lengths = torch.tensor([140, 57])
    keep = torch.arange(140) < lengths[:, None]
    return layer, regions, tokens, residual, lengths, keep


def test_layer_and_its_gradients():
    layer, regions, tokens, residual, lengths, keep = case(torch.float32)
    ins = [t.double().requires_grad_(True) for t in (regions, tokens, residual)]
    layer = layer.double()
    want = plain_layer(layer, *ins, keep)
    grads = [torch.randn_like(t) for t in want]
    want_grads = torch.autograd.grad(want, [*ins, *layer.parameters()], grads)
    layer = layer.float().to(DEV)
    got_ins = [t.to(DEV).requires_grad_(True) for t in (regions, tokens, residual)]
    got = layer(*got_ins, key_lengths=lengths.to(DEV))
    got_grads = torch.autograd.grad(got, [*got_ins, *layer.parameters()], [g.float().to(DEV) for g in grads])
    for a, b in zip((*got, *got_grads), (*want, *want_grads)):   # float32 sums of up to 200 terms, six in a row
        assert (a.double().cpu() - b).norm() <= 2e-5 * b.norm()


def test_inference_in_8_bits_stays_near():
    """Each of the five products rounds both operands to four bits: 2.6 % of its size each, root of two for the pair, 3.7 % a
    layer; five of them on the longest way, all adding up."""
    layer, regions, tokens, residual, lengths, keep = case(torch.bfloat16)
    with torch.no_grad():
        want = sum(plain_layer(layer.double(), regions.double(), tokens.double(), residual.double(), keep))
        fast = layer.float().to(DEV).for_inference()
        out = sum(fast(*(t.to(DEV).bfloat16() for t in (regions, tokens)), residual.to(DEV).bfloat16(), key_lengths=lengths.to(DEV)))
    assert out.dtype == torch.bfloat16 and (out.double().cpu() - want).norm() <= 5 * 0.037 * want.norm()
    assert layer.query.weight.dtype == torch.float32   # the layer itself has stayed


def test_example_trains_and_serves():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
    import region_decoder
    losses, right, agree = region_decoder.main(30)
    assert losses[-1] < 0.5 * losses[0] and right > 0.8 and agree > 0.9
