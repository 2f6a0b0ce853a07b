"""The fast forwards as typed PyTorch custom operators (torch.library).

The reference exposes its native kernels as typed pybind11 functions
(KAD-Conv/kadconv/acceleration/kadc_dcn16.cpp:247-330) and calls
torchvision's registered ``torchvision::deform_conv2d``.  Here the ctypes
calls are wrapped as custom ops with fake (meta) implementations, so
``torch.compile`` and FakeTensor tracing see typed operators with known output
shapes instead of breaking the graph at an opaque Python call:

  kadconv::deform_conv2d(input, offset, weight, bias?, stride_h, stride_w,
                         pad_h, pad_w, dil_h, dil_w, mask?) -> Tensor
      the functional operator (kadconv.ops.deform_conv2d, torchvision's
      argument meaning);
  kadconv::layer_fwd(x, handle) -> Tensor
      the fused forward of one enabled layer (a KADConv / KADC4 / DSC plan):
      ``handle`` names the plan in a process-wide registry, because a plan
      (packed weights, folded BN, streams) is not a tensor argument.  The
      output has x's shape for KAD-Conv layers and [N, Cout, H', W'] for DSCs,
      in x's memory format.
  kadconv::group_norm_act(x, num_groups, weight?, bias?, eps, act?)
        -> (Tensor y, Tensor mean, Tensor rstd)
      kadconv.ops.group_norm_act with the statistics its gradient uses, which are
      constants to autograd; the gradient is the operator
      kadconv::group_norm_act_backward.

The eager implementations run the HIP kernels; nothing here falls back to
another implementation.
"""
import itertools

import torch

_PLANS = {}
_NEXT = itertools.count(1)


def register_plan(plan):
    """Store a plan and return its integer handle for ``kadconv::layer_fwd``."""
    h = next(_NEXT)
    _PLANS[h] = plan
    return h


def release_plan(handle):
    _PLANS.pop(handle, None)


def _memory_format(x):
    if x.dim() == 4 and x.is_contiguous(memory_format=torch.channels_last) and not x.is_contiguous():
        return torch.channels_last
    return torch.contiguous_format


@torch.library.custom_op('kadconv::layer_fwd', mutates_args=())
def layer_fwd(x: torch.Tensor, handle: int) -> torch.Tensor:
    with torch.no_grad():
        return _PLANS[handle].forward(x)


@layer_fwd.register_fake
def _(x, handle):
    plan = _PLANS[handle]
    n, _, h, w = x.shape
    cout, ho, wo = plan.out_shape(h, w)
    return torch.empty((n, cout, ho, wo), dtype=x.dtype, device=x.device, memory_format=_memory_format(x))


@torch.library.custom_op('kadconv::deform_conv2d', mutates_args=())
def deform_conv2d(input: torch.Tensor, offset: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None,
                  stride_h: int, stride_w: int, pad_h: int, pad_w: int, dil_h: int, dil_w: int,
                  mask: torch.Tensor | None) -> torch.Tensor:
    from . import ops
    return ops.deform_conv2d(input, offset, weight, bias, stride=(stride_h, stride_w), padding=(pad_h, pad_w),
                             dilation=(dil_h, dil_w), mask=mask)


@deform_conv2d.register_fake
def _(input, offset, weight, bias, stride_h, stride_w, pad_h, pad_w, dil_h, dil_w, mask):
    n, _, h, w = input.shape
    co, _, kh, kw = weight.shape
    ho = (h + 2 * pad_h - dil_h * (kh - 1) - 1) // stride_h + 1
    wo = (w + 2 * pad_w - dil_w * (kw - 1) - 1) // stride_w + 1
    return input.new_empty((n, co, ho, wo))


@torch.library.custom_op('kadconv::group_norm_act', mutates_args=())
def group_norm_act(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None, bias: torch.Tensor | None, eps: float,
                   act: str | None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    from . import ops
    if not x.is_cuda:
        raise ValueError('kadconv::group_norm_act needs a GPU tensor')
    ops._group_norm_check(x, num_groups, weight, bias, eps, act)
    return ops.group_norm_act_forward(x, num_groups, weight, bias, eps, act)


def _nhwc_empty(x):
    n, c, h, w = x.shape
    return x.new_empty((n, h, w, c)).permute(0, 3, 1, 2)


@group_norm_act.register_fake
def _(x, num_groups, weight, bias, eps, act):
    mean = x.new_empty((x.shape[0], num_groups), dtype=torch.float32)
    return _nhwc_empty(x), mean, torch.empty_like(mean)


@torch.library.custom_op('kadconv::group_norm_act_backward', mutates_args=())
def group_norm_act_backward(dy: torch.Tensor, x: torch.Tensor, num_groups: int, weight: torch.Tensor | None,
                            bias: torch.Tensor | None, mean: torch.Tensor, rstd: torch.Tensor, eps: float,
                            act: str | None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    from . import ops
    dx, dw, db = ops.group_norm_act_backward(dy, x, num_groups, weight, bias, mean, rstd, eps, act)
    none = mean.new_empty(0)
    return dx, none if dw is None else dw, none.clone() if db is None else db


@group_norm_act_backward.register_fake
def _(dy, x, num_groups, weight, bias, mean, rstd, eps, act):
    def like(p):
        return mean.new_empty(0) if p is None else torch.empty_like(p, memory_format=torch.contiguous_format)
    return _nhwc_empty(x), like(weight), like(bias)


def _group_norm_act_context(ctx, inputs, output):
    x, num_groups, weight, bias, eps, act = inputs
    ctx.mark_non_differentiable(output[1], output[2])  # for the gradient's own use
    ctx.save_for_backward(x, weight, bias, output[1], output[2])
    ctx.rest = num_groups, eps, act


def _group_norm_act_grad(ctx, dy, _mean, _rstd):
    x, weight, bias, mean, rstd = ctx.saved_tensors
    num_groups, eps, act = ctx.rest
    dx, dw, db = torch.ops.kadconv.group_norm_act_backward(dy, x, num_groups, weight, bias, mean, rstd, eps, act)
    return dx, None, None if weight is None else dw, None if bias is None else db, None, None


group_norm_act.register_autograd(_group_norm_act_grad, setup_context=_group_norm_act_context)
