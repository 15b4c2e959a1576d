"""Linear layers in 8-bit floating point (e4m3) with a scale for each block of 128, for inference.  No counterpart in the
reference."""
import torch
from torch import nn

from .._lib import native


def quantize_blocks(x, block_rows=1):
    """``x [..., columns]`` in 8 bits: ``(q, scales)``.

    ``q`` is float8_e4m3fn with the columns padded with zeros to whole blocks of 128, ``scales`` float32: one for each row
    and block of 128 columns (activations, ``block_rows=1``) or for each 128 x 128 block of a matrix (weights,
    ``block_rows=128``).  ``scale = max(max|x| / 448, 2 ** -126)``, ``q = e4m3(x * (1 / scale))``.  No gradient."""
    return native.quantize_blocks(x, block_rows)


def block_linear(q, q_scales, weight, weight_scales, bias=None, out_dtype=torch.bfloat16):
    """``(q * q_scales) @ (weight * weight_scales).T + bias`` of 8-bit activations ``[..., inputs]`` and weights
    ``[outputs, inputs]`` as ``quantize_blocks`` gives them (``block_rows`` 1 and 128); float16 or bfloat16
    ``[..., outputs]``.  No gradient."""
    return native.block_linear(q, q_scales, weight, weight_scales, bias, out_dtype)


class BlockScaledLinear(nn.Module):
    """A trained ``nn.Linear`` with its weight in 8 bits.  Takes activations as they are, or ``(q, scales)`` that are in
    8 bits already (``AddRMSNorm.quantized``).

    Args:
        in_features, out_features (int): sizes of the layer
        bias (bool): whether there is a bias
        dtype (torch.dtype): of the results, float16 or bfloat16
    """

    def __init__(self, in_features, out_features, bias=True, dtype=torch.bfloat16, device=None):
        super().__init__()
        self.in_features, self.out_features, self.dtype = in_features, out_features, dtype
        blocks = -(-in_features // 128)
        self.register_buffer('weight', torch.zeros(out_features, 128 * blocks, device=device).to(torch.float8_e4m3fn))
        self.register_buffer('weight_scales', torch.ones(-(-out_features // 128), blocks, device=device))
        self.register_buffer('bias', torch.zeros(out_features, dtype=dtype, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear, dtype=torch.bfloat16):
        """The layer of a ``nn.Linear`` on the GPU."""
        layer = cls(linear.in_features, linear.out_features, linear.bias is not None, dtype, 'meta')
        layer.weight, layer.weight_scales = quantize_blocks(linear.weight.detach(), 128)
        if linear.bias is not None:
            layer.bias = linear.bias.detach().to(dtype)
        return layer

    def _apply(self, fn, recurse=True):
        # .half() and its like leave what is in 8 bits, and its scales, as they are; moves between devices take all
        kept = {name: getattr(self, name) for name in ('weight', 'weight_scales')}
        super()._apply(fn, recurse)
        for name, tensor in kept.items():
            now = getattr(self, name)
            if now.dtype != tensor.dtype:
                setattr(self, name, tensor.to(now.device))
        return self

    def forward(self, x):
        if isinstance(x, tuple):
            q, scales = x
        else:
            if x.size(-1) != self.in_features:
                raise RuntimeError(f"the input has rows of {x.size(-1)}, expected {self.in_features}")
            q, scales = quantize_blocks(x)
        return block_linear(q, scales, self.weight, self.weight_scales, self.bias, self.dtype)

    def __repr__(self):
        return (f"{self.__class__.__name__}({self.in_features}, {self.out_features}, bias={self.bias is not None}, "
                f"dtype={self.dtype})")
