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
  kadconv::layer_norm(x, weight?, bias?, eps, dim) -> (Tensor y, Tensor mean, Tensor rstd)
      kadconv.ops.layer_norm, likewise, with kadconv::layer_norm_backward.
  kadconv::linear8(x, weight, bias?, act?, dim) -> Tensor
  kadconv::linear8_kept(x, codes, scales, size, bias?, act?, dim) -> Tensor
  kadconv::quantize8(x, dim) -> (Tensor codes, Tensor scales)
  kadconv::matmul8(a_codes, a_scales, b_codes, b_scales, size, bias?, act?, dtype) -> Tensor
      those of kadconv.block8; the first's gradient is kadconv::linear8_backward.
  kadconv::distill_loss(logits, teacher_logits, teacher_index, temperature, reduction, dim)
        -> (Tensor loss, Tensor stats, Tensor share)
      kadconv.ops.distill_loss, likewise, with kadconv::distill_loss_backward.

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


def _rows_empty(x, dim, c=None, dtype=None):
    """A dense result for x's rows (of c values each)."""
    from . import ops
    axis = ops._row_axis(x, dim)
    shape = list(x.shape)
    own = shape.pop(axis)
    return x.new_empty((*shape, own if c is None else c), dtype=dtype or x.dtype).movedim(-1, axis)


@torch.library.custom_op('kadconv::layer_norm', mutates_args=())
def layer_norm(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, eps: float,
               dim: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    from . import ops
    if not x.is_cuda:
        raise ValueError('kadconv::layer_norm needs a GPU tensor')
    return ops.layer_norm_forward(x, weight, bias, eps, dim)


@layer_norm.register_fake
def _(x, weight, bias, eps, dim):
    from . import ops
    mean = x.new_empty((x.numel() // x.shape[ops._row_axis(x, dim)],), dtype=torch.float32)
    return _rows_empty(x, dim), mean, torch.empty_like(mean)


def _or_empty(like, *grads):
    """Gradients as an operator's results: of what is not needed or has no tensor an empty one."""
    return tuple(like.new_empty(0) if g is None else g for g in grads)


@torch.library.custom_op('kadconv::layer_norm_backward', mutates_args=())
def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None,
                        mean: torch.Tensor, rstd: torch.Tensor, eps: float, dim: int, need_x: bool = True, need_weight: bool = True,
                        need_bias: bool = True) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    from . import ops
    return _or_empty(mean, *ops.layer_norm_backward(dy, x, weight, bias, mean, rstd, eps, dim, need_x, need_weight, need_bias))


@layer_norm_backward.register_fake
def _(dy, x, weight, bias, mean, rstd, eps, dim, need_x=True, need_weight=True, need_bias=True):
    def like(need, p):
        return torch.empty_like(p, memory_format=torch.contiguous_format) if need and p is not None else None
    return _or_empty(mean, _rows_empty(x, dim) if need_x else None, like(need_weight, weight), like(need_bias, bias))


def _layer_norm_context(ctx, inputs, output):
    x, weight, bias, eps, dim = inputs
    ctx.mark_non_differentiable(output[1], output[2])  # for the gradient's own use
    ctx.save_for_backward(x, weight, bias, output[1], output[2])
    ctx.rest = eps, dim


def _layer_norm_grad(ctx, dy, _mean, _rstd):
    x, weight, bias, mean, rstd = ctx.saved_tensors
    need = ctx.needs_input_grad[:3]
    grads = torch.ops.kadconv.layer_norm_backward(dy, x, weight, bias, mean, rstd, *ctx.rest, *need)
    return *(g if n else None for g, n in zip(grads, need)), None, None


layer_norm.register_autograd(_layer_norm_grad, setup_context=_layer_norm_context)


@torch.library.custom_op('kadconv::distill_loss', mutates_args=())
def distill_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor, temperature: float,
                 reduction: str, dim: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    from . import ops
    if not logits.is_cuda:
        raise ValueError('kadconv::distill_loss needs a GPU tensor')
    return ops.distill_loss_forward(logits, teacher_logits, teacher_index, temperature, reduction, dim)


@distill_loss.register_fake
def _(logits, teacher_logits, teacher_index, temperature, reduction, dim):
    from . import ops
    axis = ops._row_axis(logits, dim)
    shape = [n for d, n in enumerate(logits.shape) if d != axis]
    rows = logits.numel() // logits.shape[axis]
    loss = logits.new_empty(shape if reduction == 'none' else (), dtype=torch.float32)
    return loss, logits.new_empty((rows, 2), dtype=torch.float32), logits.new_empty((1,), dtype=torch.float32)


@torch.library.custom_op('kadconv::distill_loss_backward', mutates_args=())
def distill_loss_backward(dloss: torch.Tensor, logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor,
                          stats: torch.Tensor, share: torch.Tensor, temperature: float, reduction: str, dim: int) -> torch.Tensor:
    from . import ops
    return ops.distill_loss_backward(dloss, logits, teacher_logits, teacher_index, stats, share, temperature, reduction, dim)


@distill_loss_backward.register_fake
def _(dloss, logits, teacher_logits, teacher_index, stats, share, temperature, reduction, dim):
    return _rows_empty(logits, dim)


def _distill_loss_context(ctx, inputs, output):
    logits, teacher_logits, teacher_index, temperature, reduction, dim = inputs
    ctx.mark_non_differentiable(output[1], output[2])  # for the gradient's own use
    ctx.save_for_backward(logits, teacher_logits, teacher_index, output[1], output[2])
    ctx.rest = temperature, reduction, dim


def _distill_loss_grad(ctx, dloss, _stats, _share):
    dz = torch.ops.kadconv.distill_loss_backward(dloss, *ctx.saved_tensors, *ctx.rest)
    return dz, None, None, None, None, None


distill_loss.register_autograd(_distill_loss_grad, setup_context=_distill_loss_context)


@torch.library.custom_op('kadconv::quantize8', mutates_args=())
def quantize8(x: torch.Tensor, dim: int) -> tuple[torch.Tensor, torch.Tensor]:
    from . import _ext
    return _ext.native().quantize8_forward(x, dim)


@quantize8.register_fake
def _(x, dim):
    from . import ops
    axis = ops._row_axis(x, dim)
    shape = [n for d, n in enumerate(x.shape) if d != axis]
    blocks = -(-x.shape[axis] // 128)
    return (x.new_empty((*shape, blocks * 128), dtype=torch.float8_e4m3fn),
            x.new_empty((*shape, -(-blocks // 4) * 4), dtype=torch.float8_e8m0fnu))


@torch.library.custom_op('kadconv::matmul8', mutates_args=())
def matmul8(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, size: int,
            bias: torch.Tensor | None, act: str | None, dtype: torch.dtype) -> torch.Tensor:
    from . import _ext
    return _ext.native().matmul8_forward(a, a_scales, b, b_scales, size, bias, act, dtype)


@matmul8.register_fake
def _(a, a_scales, b, b_scales, size, bias, act, dtype):
    return a.new_empty((*a.shape[:-1], b.shape[0]), dtype=dtype)


@torch.library.custom_op('kadconv::linear8', mutates_args=())
def linear8(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, act: str | None, dim: int) -> torch.Tensor:
    from . import block8
    return block8.linear8_forward(x, weight, bias, act, dim)


@linear8.register_fake
def _(x, weight, bias, act, dim):
    return _rows_empty(x, dim, weight.shape[0])


@torch.library.custom_op('kadconv::linear8_backward', mutates_args=())
def linear8_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, dim: int, need_x: bool = True,
                     need_weight: bool = True, need_bias: bool = True) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    from . import block8
    return _or_empty(weight, *block8.linear8_backward(dy, x, weight, bias, dim, need_x, need_weight, need_bias))


@linear8_backward.register_fake
def _(dy, x, weight, bias, dim, need_x=True, need_weight=True, need_bias=True):
    def like(need, p):
        return torch.empty_like(p, memory_format=torch.contiguous_format) if need and p is not None else None
    return _or_empty(weight, _rows_empty(x, dim) if need_x else None, like(need_weight, weight), like(need_bias, bias))


def _linear8_context(ctx, inputs, output):
    from . import block8
    x, weight, bias, act, dim = inputs
    if act is not None:
        raise NotImplementedError('kadconv.linear8 with an activation has no gradient')
    block8._gradient_check(x.numel() // weight.shape[1], weight.shape[0], *ctx.needs_input_grad[:3])
    ctx.save_for_backward(x, weight, bias)
    ctx.dim = dim


def _linear8_grad(ctx, dy):
    x, weight, bias = ctx.saved_tensors
    need = ctx.needs_input_grad[:3]
    grads = torch.ops.kadconv.linear8_backward(dy, x, weight, bias, ctx.dim, *need)
    return *(g if n else None for g, n in zip(grads, need)), None, None


linear8.register_autograd(_linear8_grad, setup_context=_linear8_context)


@torch.library.custom_op('kadconv::linear8_kept', mutates_args=())
def linear8_kept(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, size: int, bias: torch.Tensor | None,
                 act: str | None, dim: int) -> torch.Tensor:
    from . import _ext
    return _ext.native().linear8_kept_forward(x, codes, scales, size, bias, act, dim)


@linear8_kept.register_fake
def _(x, codes, scales, size, bias, act, dim):
    return _rows_empty(x, dim, codes.shape[0])
