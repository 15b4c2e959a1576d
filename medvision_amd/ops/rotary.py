"""Rotary positions on several axes: queries and keys are told where in a volume their regions and cells lie.  No counterpart
in the reference."""
import torch
from torch.autograd.function import once_differentiable

from .._lib import native
from ._function import NativeFunction
from ._module import KeepsTypes


class RotaryPositionsFunction(NativeFunction):
    @staticmethod
    def native(x, positions, frequencies, neighbours=False):
        return native.rotary_positions(x, positions, frequencies, neighbours)

    @staticmethod
    def forward(ctx, x, positions, frequencies, neighbours=False):
        ctx.neighbours, ctx.dtype = neighbours, x.dtype
        ctx.save_for_backward(positions, frequencies)
        return native.rotary_positions_turn(x, positions, frequencies, neighbours, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        positions, frequencies = ctx.saved_tensors
        return native.rotary_positions_turn(grad_output.to(ctx.dtype), positions, frequencies, ctx.neighbours, True), None, None, None


def axis_frequencies(channels, axes=3, theta=100.0, device=None):
    """Frequencies that give each axis a share of a head's pairs: float64 ``[axes, channels // 2]`` for ``rotary_positions``.

    Of the ``channels // 2`` pairs each axis has ``n = channels // 2 // axes``, which turn by ``theta ** (-i / n)``, ``i = 0 .. n - 1``,
    per unit of the position; the pairs that are left over, the last ones, do not turn.  Whole positions over a few hundred cells go
    well with the default ``theta``."""
    each = channels // 2 // axes if axes > 0 else 0
    if each < 1:
        raise ValueError(f"{channels} channels for {axes} axes: at least one pair for each is needed")
    turn = float(theta) ** (-torch.arange(each, dtype=torch.float64, device=device) / each)
    return torch.nn.functional.pad(torch.block_diag(*[turn[None]] * axes), (0, channels // 2 - axes * each))


def rotary_positions(x, positions, frequencies, neighbours=False):
    """Heads turned by their rows' positions: the products of turned queries and keys depend on how far apart they are.

    Args:
        x (Tensor): ``[batch, rows, heads, channels]``, float32, float16 or bfloat16; views are read in place as long as a
            head's channels are neighbours
        positions (Tensor): ``[batch, rows, axes]``, or ``[rows, axes]`` for all samples; whole or floating numbers
        frequencies (Tensor): ``[axes, pairs]``, float64 (or float32), in radians per unit: pair ``p`` of a row at ``positions[a]`` is
            turned by the sum over the axes of ``positions[a] * frequencies[a, p]``, formed in 64 bits
        neighbours (bool): whether pair ``p`` are the channels ``2 p`` and ``2 p + 1``, or ``p`` and ``pairs + p``

    Channels behind the pairs stay as they are.  The gradient flows to ``x``."""
    return RotaryPositionsFunction.apply(x, positions, frequencies, neighbours)


class RotaryPositions(KeepsTypes):
    """``rotary_positions`` with the frequencies of ``axis_frequencies``, for heads of ``channels``."""
    kept = ('frequencies',)

    def __init__(self, channels, axes=3, theta=100.0, neighbours=False):
        super().__init__()
        self.neighbours = neighbours
        self.register_buffer('frequencies', axis_frequencies(channels, axes, theta))

    def forward(self, x, positions):
        return rotary_positions(x, positions, self.frequencies, self.neighbours)

    def __repr__(self):
        return f"{self.__class__.__name__}({tuple(self.frequencies.shape)}, neighbours={self.neighbours})"
