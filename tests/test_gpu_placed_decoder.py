"""Group norm in front of the tokens, positions in the decoder layer, its linear layers in 4 bits: run together."""
import copy

import pytest
import torch

import tokens_ref as ref
from test_gpu_region_decoder import plain_layer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def case(channels=96, heads=6, key_heads=3):
    import medvision_amd.ops as ops
    torch.manual_seed(1)
    norm = ops.GroupNormAct(8, channels, activation="gelu")
    torch.nn.init.normal_(norm.bias)
    layer = ops.RegionDecoderLayer(channels, heads, hidden=200, key_heads=key_heads, axes=3)
    regions, residual = torch.randn(2, 33, channels), torch.randn(2, 33, channels)
    features = torch.randn(2, channels, 4, 5, 7)
    cells = torch.stack(torch.meshgrid(*(torch.arange(n) + 0.5 for n in (4, 5, 7)), indexing="ij"), -1).reshape(-1, 3)
    return norm, layer, regions, residual, features, 5 * torch.rand(2, 33, 3), cells


def plain(layer, regions, residual, tokens, region_positions, token_positions):
    """The layer in elementary operations and the type of its inputs."""
    f = layer.place.frequencies
    rms = lambda m, x: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + m.eps) * m.weight.to(x)   # noqa: E731
    linear = lambda m, x: x @ m.weight.to(x).t() + (0 if m.bias is None else m.bias.to(x))   # noqa: E731
    h = regions + residual
    q = linear(layer.query, rms(layer.norm_query, h)).unflatten(-1, (layer.heads, -1))
    k, v = linear(layer.key_value, tokens).unflatten(-1, (2, layer.key_heads, -1)).unbind(2)
    q, k = turned(q, region_positions, f), turned(k, token_positions, f)
    k, v = (t.repeat_interleave(layer.heads // layer.key_heads, 2).transpose(1, 2) for t in (k, v))
    p = torch.softmax(q.transpose(1, 2) @ k.transpose(-1, -2) * layer.head_channels ** -0.5, -1)
    h = linear(layer.out, (p @ v).transpose(1, 2).flatten(2)) + h
    return linear(layer.down, torch.relu(linear(layer.up, rms(layer.norm_hidden, h)))), h


def turned(x, positions, f):
    angle = (positions.double() @ f.double()).unsqueeze(-2).to(x)
    n = f.shape[1]
    a, b = x[..., :n], x[..., n:2 * n]
    return torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), x[..., 2 * n:]), -1)


def plain_tokens(norm, features):
    x = features.flatten(2).transpose(1, 2)
    y = torch.nn.functional.group_norm(x.transpose(1, 2), norm.groups, norm.weight.to(x), norm.bias.to(x), norm.eps).transpose(1, 2)
    return torch.nn.functional.gelu(y)


def test_together_with_gradients():
    import medvision_amd.ops as ops
    norm, layer, regions, residual, features, at, cells = case()
    ins = [t.double().requires_grad_(True) for t in (regions, residual, features)]
    params = [*norm.double().parameters(), *layer.double().parameters()]
    want = plain(layer, ins[0], ins[1], plain_tokens(norm, ins[2]), at, cells)
    grads = [torch.randn_like(t) for t in want]
    want_grads = torch.autograd.grad(want, [*ins, *params], grads)
    norm, layer = norm.float().to(DEV), layer.float().to(DEV)
    got_ins = [t.to(DEV).requires_grad_(True) for t in (regions, residual, features)]
    got = layer(got_ins[0], norm(ops.map_tokens(got_ins[2])), got_ins[1], region_positions=at.to(DEV), token_positions=cells.to(DEV))
    got_grads = torch.autograd.grad(got, [*got_ins, *norm.parameters(), *layer.parameters()], [g.float().to(DEV) for g in grads])
    for a, b in zip((*got, *got_grads), (*want, *want_grads)):   # float32 sums of up to 280 terms, seven in a row
        assert (a.double().cpu() - b).norm() <= 2e-5 * b.norm()
    assert all(torch.isfinite(g).all() for g in got_grads)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_under_autocast(dtype):
    """Regions in float32, queries in 16 bits.  Seven products and norms one after the other, each of which rounds operands and
    results: 42 unit roundoffs."""
    import medvision_amd.ops as ops
    norm, layer, regions, residual, features, at, cells = case()
    with torch.no_grad():
        want = plain(copy.deepcopy(layer).double(), regions.double(), residual.double(), plain_tokens(copy.deepcopy(norm).double(), features.double()), at, cells)
    norm, layer = norm.to(DEV), layer.to(DEV)
    with torch.autocast("cuda", dtype=dtype):
        got = layer(regions.to(DEV), norm(ops.map_tokens(features.to(DEV))), residual.to(DEV), region_positions=at.to(DEV), token_positions=cells.to(DEV))
        sum(t.float().sum() for t in got).backward()
    unit = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    for a, b in zip(got, want):
        assert (a.double().cpu() - b).norm() <= 42 * unit * b.norm()
    assert all(torch.isfinite(p.grad).all() for m in (norm, layer) for p in m.parameters())


@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_served_in_4_bits(group, dtype):
    """The same as the layer whose weights are the values of the codes, in 64 bits: 36 unit roundoffs as under autocast; the
    layer itself stays."""
    import medvision_amd.ops as ops
    _, layer, regions, residual, features, at, cells = case()
    tokens = ops.map_tokens(features)
    before = {k: v.clone() for k, v in layer.state_dict().items()}
    fast = layer.to(DEV).for_inference(dtype, bits=4, group=group)
    assert isinstance(fast.up, ops.GroupScaledLinear) and fast.place is not layer.place
    with torch.no_grad():
        stand = copy.deepcopy(layer).cpu().double()
        for name in ("query", "key_value", "out", "up", "down"):
            m = getattr(fast, name)
            getattr(stand, name).weight.copy_(ref.group_values(m.weight, m.scales, m.in_features))
        want = plain(stand, regions.double(), residual.double(), tokens.double(), at, cells)
        for regions_type in (dtype, torch.float32):   # float32 regions: the sum that is carried keeps its type
            got = fast(regions.to(DEV, regions_type), tokens.to(DEV, dtype), residual.to(DEV, regions_type), region_positions=at.to(DEV), token_positions=cells.to(DEV))
            assert got[0].dtype == dtype and got[1].dtype == regions_type
            unit = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
            for a, b in zip(got, want):
                assert (a.double().cpu() - b).norm() <= 36 * unit * b.norm()
    assert all(torch.equal(v.cpu(), before[k]) for k, v in layer.state_dict().items())


def test_layers_without_axes_are_as_they_were():
    import medvision_amd.ops as ops
    from test_gpu_region_decoder import case as old_case
    layer, regions, tokens, residual, lengths, keep = old_case(torch.float32)
    want = plain_layer(layer.double(), regions.double(), tokens.double(), residual.double(), keep)
    layer = layer.float().to(DEV)
    got = layer(regions.to(DEV), tokens.to(DEV), residual.to(DEV), key_lengths=lengths.to(DEV))
    for a, b in zip(got, want):
        assert (a.double().cpu() - b).norm() <= 2e-5 * b.norm()
    with pytest.raises(ValueError, match="given"):
        layer(regions.to(DEV), tokens.to(DEV), region_positions=torch.zeros(33, 3, device=DEV))
    with torch.no_grad():
        eight, four = layer.for_inference(torch.float16), layer.for_inference(torch.float16, bits=4)
        assert isinstance(eight.up, ops.BlockScaledLinear) and isinstance(four.up, ops.GroupScaledLinear)
        y, h = four(regions.to(DEV).half(), tokens.to(DEV).half(), key_lengths=lengths.to(DEV))
    assert torch.isfinite(y).all() and torch.isfinite(h).all()
