"""Group norm with an activation on cells in channels-last order, as ``map_tokens`` gives them.  No counterpart in the
reference."""
import torch
from torch import nn
from torch.autograd.function import once_differentiable

from .._lib import native
from ._function import NativeFunction


class GroupNormActFunction(NativeFunction):
    @staticmethod
    def native(x, groups, weight=None, bias=None, eps=1e-5, activation=None, slope=0.01):
        return native.group_norm_act(x, groups, weight, bias, eps, activation, slope)

    @staticmethod
    def forward(ctx, x, groups, weight=None, bias=None, eps=1e-5, activation=None, slope=0.01):
        y, stats = native.group_norm_act_forward(x, groups, weight, bias, eps, activation, slope)
        ctx.groups, ctx.activation, ctx.slope = groups, activation, slope
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        x, weight, bias, stats = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        grads = native.group_norm_act_backward(x, ctx.groups, weight, bias, stats, grad_output, ctx.activation, ctx.slope,
                                               wanted[0], wanted[2], wanted[3])
        return grads[0], None, grads[1], grads[2], None, None, None


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, activation=None, slope=0.01):
    """``activation(h * weight + bias)`` with ``h = (x - mean) / sqrt(var + eps)``, mean and variance those of a sample's cells
    and a group's channels.

    Args:
        x (Tensor): ``[batch, ..., channels]``, float32, float16 or bfloat16; the dimensions between are cells.  Tokens of a
            map in ``channels_last`` or ``channels_last_3d`` order are read in place, others are copied into that order
        groups (int): of neighbouring channels, as many in each (as many groups as channels: instance norm)
        weight, bias (Tensor): ``[channels]``, of the type of ``x`` or float32, or None (ones, zeros)
        eps (float): added to the variance
        activation (str): ``'relu'``, ``'leaky_relu'``, ``'silu'``, ``'gelu'`` (the exact form), or None
        slope (float): of ``'leaky_relu'`` below zero

    Gradients flow to ``x``, ``weight`` and ``bias``; at zero the activations with two branches have the lower one's.  Statistics
    and sums are in 32 bits or more, each result is rounded once.  Batches of 65536 and more are taken where a group of a sample
    fits into a workgroup's registers (up to 5000 cells, and about 16384 values of an odd number of channels to 65536 of a
    multiple of four)."""
    return GroupNormActFunction.apply(x, groups, weight, bias, eps, activation, slope)


class GroupNormAct(nn.Module):
    """``group_norm_act`` with its weight and bias.

    Args:
        groups, channels (int): sizes; ``channels`` is a multiple of ``groups``
        eps (float): added to the variance
        activation (str), slope (float): as ``group_norm_act`` takes them
    """

    def __init__(self, groups, channels, eps=1e-5, activation=None, slope=0.01):
        super().__init__()
        if groups < 1 or channels % groups:
            raise ValueError(f"{channels} channels in {groups} groups")
        self.groups, self.eps, self.activation, self.slope = groups, float(eps), activation, float(slope)
        self.weight, self.bias = nn.Parameter(torch.ones(channels)), nn.Parameter(torch.zeros(channels))

    def forward(self, x):
        return group_norm_act(x, self.groups, self.weight, self.bias, self.eps, self.activation, self.slope)

    def __repr__(self):
        return f"{self.__class__.__name__}({self.groups}, {self.weight.numel()}, eps={self.eps}, activation={self.activation!r})"
