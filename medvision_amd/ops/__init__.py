"""Operator classes with the names and signatures of the reference's ``medvision.ops``
(``medvision/ops/__init__.py:1-24``), restricted to the trilinear-sampling family, and the operators of region decoders
behind a head: cross attention, RMS norm with residual, linear layers in 8 and 4 bits, group norm with an activation, rotary
positions."""
from .roi_align_nd import PreparedFeatures, RoIAlign
from .roi_align_rotated_nd import RoIAlignRotated
from .deform_conv_2d import DeformConv2d, DeformConv2dPack
from .modulated_deform_conv_2d import ModulatedDeformConv2d, ModulatedDeformConv2dPack
from .deform_conv_3d import DeformConv3d, DeformConv3dPack
from .modulated_deform_conv_3d import ModulatedDeformConv3d, ModulatedDeformConv3dPack
from .cuda_fun_tools import affine_2d, affine_3d, apply_offset_2d, apply_offset_3d
from .cross_attention import cross_attention
from .rms_norm import AddRMSNorm, add_rms_norm, add_rms_norm_quantized
from .block_linear import BlockScaledLinear, block_linear, quantize_blocks
from .group_norm import GroupNormAct, group_norm_act
from .rotary import RotaryPositions, axis_frequencies, rotary_positions
from .group_linear import GroupScaledLinear, group_linear, quantize_groups
from .region_decoder import RegionDecoderLayer, map_tokens

__all__ = [
    'RoIAlign',
    'PreparedFeatures',
    'RoIAlignRotated',
    'DeformConv2d',
    'DeformConv2dPack',
    'ModulatedDeformConv2d',
    'ModulatedDeformConv2dPack',
    'DeformConv3d',
    'DeformConv3dPack',
    'ModulatedDeformConv3d',
    'ModulatedDeformConv3dPack',
    'affine_2d', 'affine_3d', 'apply_offset_2d', 'apply_offset_3d',
    'cross_attention',
    'AddRMSNorm', 'add_rms_norm', 'add_rms_norm_quantized',
    'BlockScaledLinear', 'block_linear', 'quantize_blocks',
    'GroupNormAct', 'group_norm_act',
    'RotaryPositions', 'axis_frequencies', 'rotary_positions',
    'GroupScaledLinear', 'group_linear', 'quantize_groups',
    'RegionDecoderLayer', 'map_tokens',
]
