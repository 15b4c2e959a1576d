"""Host side of the decoder layer."""
import pytest
import torch


def test_layer_refuses_what_does_not_divide():
    import medvision_amd.ops as ops
    with pytest.raises(ValueError, match="heads"):
        ops.RegionDecoderLayer(100, 3)
    with pytest.raises(ValueError, match="heads"):
        ops.RegionDecoderLayer(96, 6, key_heads=4)
    layer = ops.RegionDecoderLayer(96, 6, key_heads=2)
    assert layer.key_value.weight.shape == (64, 96) and layer.up.weight.shape == (384, 96)
    with pytest.raises(RuntimeError, match="not implemented on CPU"):
        layer(torch.zeros(1, 2, 96), torch.zeros(1, 3, 96))


def test_tokens_of_a_map():
    import medvision_amd.ops as ops
    x = torch.arange(2 * 3 * 2 * 2 * 2).view(2, 3, 2, 2, 2)
    t = ops.map_tokens(x)
    assert t.shape == (2, 8, 3) and torch.equal(t[1, 5], x[1, :, 1, 0, 1])
