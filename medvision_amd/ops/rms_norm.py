"""RMS norm with the residual's addition, with an output in 8 bits for the layers of ``block_linear.py``.  No counterpart
in the reference."""
import torch
from torch import nn
from torch.autograd.function import once_differentiable

from .._lib import native
from ._function import NativeFunction, RecordedFunction, tracing


class AddRMSNormFunction(NativeFunction):
    @staticmethod
    def native(x, residual, weight, eps=1e-6):
        return native.add_rms_norm(x, residual, weight, eps)

    @staticmethod
    def forward(ctx, x, residual, weight, eps=1e-6):
        y, total = native.add_rms_norm_forward(x, residual, weight, eps)
        ctx.eps, ctx.added = eps, total is not None
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(total if ctx.added else x, weight)
        return (y, total) if ctx.added else (y, x)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_sum):
        if grad_y is None and grad_sum is None:
            return None, None, None, None
        h, weight = ctx.saved_tensors
        for_x, for_residual, for_weight = ctx.needs_input_grad[:3]
        grad_h, grad_weight = native.add_rms_norm_backward(h, weight, grad_y, grad_sum, ctx.eps, for_x or for_residual, for_weight)
        return grad_h if for_x else None, grad_h if for_residual else None, grad_weight, None


class AddRMSNormQuantizedFunction(RecordedFunction):
    refuses = 'add_rms_norm_quantized'

    @staticmethod
    def native(x, residual, weight, eps):
        return native.add_rms_norm_quantized(x, residual, weight, eps)


def add_rms_norm(x, residual, weight, eps=1e-6):
    """``h = x + residual`` and its norm ``y = h / sqrt(mean(h ** 2) + eps) * weight`` over the last dimension: ``(y, h)``.

    ``residual`` is None (``h`` is then ``x``) or like ``x``; ``weight`` has the type of ``x`` or float32.  ``h`` is held in
    the type of ``x``, and the norm is that of what is held.  Gradients flow to ``x``, ``residual`` and ``weight`` from both
    results."""
    return AddRMSNormFunction.apply(x, residual, weight, eps)


def add_rms_norm_quantized(x, residual, weight, eps=1e-6):
    """``add_rms_norm`` whose ``y`` is in 8 bits, as ``quantize_blocks`` gives them: ``(q, scales, h)``.  No gradient."""
    if tracing() is None:
        return native.add_rms_norm_quantized(x, residual, weight, eps)
    return AddRMSNormQuantizedFunction.apply(x, residual, weight, eps)


class AddRMSNorm(nn.Module):
    """``add_rms_norm`` with its weight: ``norm(x, residual)`` gives ``(y, h)``, ``norm.quantized(x, residual)`` gives
    ``((q, scales), h)`` for a ``BlockScaledLinear``."""

    def __init__(self, channels, eps=1e-6):
        super().__init__()
        self.eps = float(eps)
        self.weight = nn.Parameter(torch.ones(channels))

    def forward(self, x, residual=None):
        return add_rms_norm(x, residual, self.weight, self.eps)

    def quantized(self, x, residual=None):
        q, scales, h = add_rms_norm_quantized(x, residual, self.weight, self.eps)
        return (q, scales), h

    def __repr__(self):
        return f"{self.__class__.__name__}({self.weight.numel()}, eps={self.eps})"
