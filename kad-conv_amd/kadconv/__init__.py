"""kadconv -- KAD-Conv with gfx950 (MI355X) HIP kernels behind the reference API.

Public API of the reference (KAD-Conv/kadconv/__init__.py:1-4): ``KADConv``,
``DSC``, ``LCSA``, ``enable_fast_inference``, ``disable_fast_inference``.
Added here: ``deform_conv2d`` (torchvision-compatible DCNv2 on the GPU), the
fused blocks ``Conv1x1SiLU``, ``SqueezeExcitation`` and ``KADDown``, for
training ``group_norm_act`` / ``GroupNormAct`` (group norm and an activation on
channels-last maps, with its gradients) and ``AdamW`` / ``AdamWPlan`` (the step
over a network's tensors in one launch, states in 32 or 8 bits), and the typed
custom operators ``torch.ops.kadconv.deform_conv2d`` / ``layer_fwd`` /
``group_norm_act`` (kadconv.library).
"""
from . import library  # registers the kadconv:: custom operators
from .blocks import Conv1x1SiLU, GroupNormAct, KADDown, SqueezeExcitation
from .fast import disable_fast_inference, enable_fast_inference
from .kad_conv import DSC, LCSA, KADConv
from .ops import deform_conv2d, group_norm_act
from .optim import AdamW, AdamWPlan

__all__ = ['KADConv', 'DSC', 'LCSA', 'enable_fast_inference', 'disable_fast_inference', 'deform_conv2d',
           'Conv1x1SiLU', 'SqueezeExcitation', 'KADDown', 'group_norm_act', 'GroupNormAct', 'AdamW', 'AdamWPlan']
