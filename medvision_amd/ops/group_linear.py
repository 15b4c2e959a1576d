"""Linear layers with weights in 4 bits (e2m1) and a scale for each group of a row, for inference.  No counterpart in the
reference."""
import torch

from .._lib import native
from ._function import RecordedFunction, tracing
from ._module import KeepsTypes


class QuantizeGroupsFunction(RecordedFunction):
    refuses = 'quantize_groups'

    @staticmethod
    def native(weight, group):
        return native.quantize_groups(weight, group)


class GroupLinearFunction(RecordedFunction):
    refuses = 'group_linear'

    @staticmethod
    def native(x, weight, scales, bias):
        return native.group_linear(x, weight, scales, bias)


def quantize_groups(weight, group=32):
    """A matrix ``[outputs, inputs]`` in 4 bits: ``(codes, scales)``.

    ``scales [outputs, groups]`` is float32, one for each ``group`` (32, 64 or 128) columns of a row, padded with zeros to whole blocks
    of 128: ``scale = max(max|w| / 6, 2 ** -126)``.  A code is ``w * (1 / scale)`` rounded to the nearest of 0, 1/2, 1, 3/2, 2, 3,
    4, 6 (codes 0 .. 7, halves to even codes) or their negatives (8 .. 15).  ``codes [outputs, 64 * blocks]`` is uint8: two codes a
    byte, the first one in its low half; the four bytes of eight neighbouring columns together; of a block's sixteen
    such pieces number ``4 s + g`` at place ``4 g + s``.  No gradient."""
    if tracing() is None:
        return native.quantize_groups(weight, group)
    return QuantizeGroupsFunction.apply(weight, group)


def group_linear(x, weight, scales, bias=None):
    """``x @ values.T + bias`` of float16 or bfloat16 rows ``[..., inputs]`` and the values of weights ``[outputs, inputs]`` as
    ``quantize_groups`` gives them, in the type of ``x``.  Values and products are exact, sums are in 32 bits.  No gradient."""
    if tracing() is None:
        return native.group_linear(x, weight, scales, bias)
    return GroupLinearFunction.apply(x, weight, scales, bias)


class GroupScaledLinear(KeepsTypes):
    """A trained ``nn.Linear`` with its weight in 4 bits.

    Args:
        in_features, out_features (int): sizes of the layer
        bias (bool): whether there is a bias
        group (int): columns that share a scale: 32, 64 or 128
        dtype (torch.dtype): of the products and the results, float16 or bfloat16; rows of other types are rounded to it
    """
    kept = ('scales',)

    def __init__(self, in_features, out_features, bias=True, group=32, dtype=torch.bfloat16, device=None):
        super().__init__()
        if group not in (32, 64, 128):
            raise ValueError(f"groups of {group} columns: 32, 64 or 128 are possible")
        self.in_features, self.out_features, self.group, self.dtype = in_features, out_features, group, dtype
        blocks = -(-in_features // 128)
        self.register_buffer('weight', torch.zeros(out_features, 64 * blocks, dtype=torch.uint8, device=device))
        self.register_buffer('scales', torch.ones(out_features, 128 // group * blocks, device=device))
        self.register_buffer('bias', torch.zeros(out_features, dtype=dtype, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear, group=32, dtype=torch.bfloat16):
        """The layer of a ``nn.Linear`` on the GPU."""
        layer = cls(linear.in_features, linear.out_features, linear.bias is not None, group, dtype, 'meta')
        layer.weight, layer.scales = quantize_groups(linear.weight.detach(), group)
        if linear.bias is not None:
            layer.bias = linear.bias.detach().to(dtype)
        return layer

    def forward(self, x):
        if x.size(-1) != self.in_features:
            raise RuntimeError(f"the input has rows of {x.size(-1)}, expected {self.in_features}")
        return group_linear(x.to(self.dtype), self.weight, self.scales, self.bias)

    def __repr__(self):
        return (f"{self.__class__.__name__}({self.in_features}, {self.out_features}, bias={self.bias is not None}, "
                f"group={self.group}, dtype={self.dtype})")
