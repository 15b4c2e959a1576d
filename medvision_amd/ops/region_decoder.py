"""A decoder layer for the regions of a head: they look at the tokens of a feature map and go through two linear layers.

``RegionDecoderLayer`` is for training, ``RegionDecoderLayer.for_inference`` gives the same layer with its linear layers in
8 bits: the norms then write what those read.  No counterpart in the reference."""
import copy

import torch
from torch import nn

from .block_linear import BlockScaledLinear
from .cross_attention import cross_attention
from .rms_norm import AddRMSNorm


def map_tokens(features):
    """The cells of a feature map ``[batch, channels, *spatial]`` as tokens ``[batch, cells, channels]``."""
    return features.flatten(2).transpose(1, 2)


class RegionDecoderLayer(nn.Module):
    """Norm, cross attention to the tokens, norm, two linear layers; the sum of all that passes by the layers is carried
    beside what the last one gave, and each norm adds the two.

    Args:
        channels (int): of regions and tokens
        heads (int): of the queries; ``channels // heads`` channels each, at most 128
        hidden (int): channels between the two linear layers, four times ``channels`` by default
        key_heads (int): of keys and values, ``heads`` by default; ``heads`` is a multiple of it
        eps (float): of the norms
    """

    def __init__(self, channels, heads, hidden=None, key_heads=None, eps=1e-6):
        super().__init__()
        key_heads = heads if key_heads is None else key_heads
        if channels % heads or heads % key_heads:
            raise ValueError(f"{channels} channels in {heads} heads over {key_heads} heads of keys")
        self.heads, self.key_heads, self.head_channels = heads, key_heads, channels // heads
        hidden = 4 * channels if hidden is None else hidden
        self.norm_query, self.norm_hidden = AddRMSNorm(channels, eps), AddRMSNorm(channels, eps)
        self.query = nn.Linear(channels, channels, bias=False)
        self.key_value = nn.Linear(channels, 2 * key_heads * self.head_channels, bias=False)
        self.out = nn.Linear(channels, channels)
        self.up, self.down = nn.Linear(channels, hidden), nn.Linear(hidden, channels)

    def for_inference(self, dtype=torch.bfloat16):
        """This layer, on the GPU, for inference: linear layers in 8 bits, their results in ``dtype``.  The norms' weights are
        float32, which goes with regions of any type."""
        layer = copy.copy(self)
        for name, value in vars(self).items():   # hooks, parameters, buffers and modules of its own
            if isinstance(value, (dict, set)):
                setattr(layer, name, value.copy())
        for name in ("query", "key_value", "out", "up", "down"):
            layer._modules[name] = BlockScaledLinear.from_linear(getattr(self, name), dtype)
        for name in ("norm_query", "norm_hidden"):
            layer._modules[name] = copy.deepcopy(getattr(self, name)).float().requires_grad_(False)
        return layer.eval()

    def _normed(self, norm, x, residual):
        if residual is not None:   # the sum that is carried keeps its type: float32 regions under autocast, or in front of 8-bit layers
            x = x.to(residual.dtype)
        if isinstance(self.query, BlockScaledLinear):   # straight to 8 bits
            return norm.quantized(x, residual)
        return norm(x, residual)

    def forward(self, regions, tokens, residual=None, key_mask=None, key_lengths=None):
        """``regions [batch, regions, channels]``, ``residual`` like them or None, ``tokens [batch, cells, channels]`` of
        which ``key_mask`` and ``key_lengths`` may leave some out: ``(regions, residual)`` for the next layer.  After the last
        one the result is their sum.  The residual has the type of the one that was given, or of the regions."""
        y, residual = self._normed(self.norm_query, regions, residual)
        q = self.query(y).unflatten(-1, (self.heads, self.head_channels))
        k, v = self.key_value(tokens).unflatten(-1, (2, self.key_heads, self.head_channels)).unbind(2)
        seen = cross_attention(q, k, v, key_mask, key_lengths).flatten(2)
        y, residual = self._normed(self.norm_hidden, self.out(seen), residual)
        return self.down(torch.relu(self.up(y))), residual
