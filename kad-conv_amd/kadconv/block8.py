"""Matrix products in 8 bits with a scale for each block of 128.

A row of K numbers is cut into blocks of 128, the last one short.  A block is held as e4m3 codes times one power of two,

    x = code * scale,  scale the smallest power of two with max |x| <= 448 * scale  (1 for a block of zeros),

so that dividing by the scale is exact and a number is rounded once, to nearest, ties to even: by 2^-4 of itself at most,
down to 2^-6 of the block's scale.  A power of two is also what the GPU's matrix instruction takes as a scale.  What is
not finite is held as NaN and does not count for its block's scale.

* ``quantize8`` -- rows in 8 bits: a ``Block8``.
* ``matmul8`` -- the product of two of them.
* ``linear8`` -- act(x W^T + b): x is brought to 8 bits on the way; W is a ``Block8``, kept by a program that serves, or
  numbers that are trained.  The gradients are such products too, each in 8 bits along its own sums.
"""
import torch
import torch.nn.functional as F

from . import _ext
from .ops import _ACTS, _check_param, _row_axis

BLOCK = 128


class Block8:
    """Rows of ``size`` numbers in 8 bits.

    ``codes``   float8_e4m3fn [..., size rounded up to 128], zeros behind the last number
    ``scales``  float8_e8m0fnu [..., blocks rounded up to 4], ones behind the last block
    """

    def __init__(self, codes, scales, size):
        size = int(size)
        blocks = -(-size // BLOCK)
        if codes.dtype != torch.float8_e4m3fn or scales.dtype != torch.float8_e8m0fnu:
            raise TypeError(f'codes must be torch.float8_e4m3fn and scales torch.float8_e8m0fnu, got {codes.dtype} and {scales.dtype}')
        if size < 1 or codes.dim() < 1 or codes.shape[:-1] != scales.shape[:-1] or codes.device != scales.device or \
                (codes.shape[-1], scales.shape[-1]) != (blocks * BLOCK, -(-blocks // 4) * 4):
            raise ValueError(f'codes [..., {blocks * BLOCK}] and scales [..., {-(-blocks // 4) * 4}] of one device expected for rows of '
                             f'{size}, got {tuple(codes.shape)} and {tuple(scales.shape)}')
        self.codes, self.scales, self.size = codes.contiguous(), scales.contiguous(), size

    @property
    def shape(self):
        return torch.Size((*self.codes.shape[:-1], self.size))

    @property
    def device(self):
        return self.codes.device

    def to(self, device):
        return Block8(self.codes.to(device), self.scales.to(device), self.size)

    def dequantize(self, dtype=torch.float32):
        """The numbers held."""
        scales = self.scales.to(torch.float64)[..., :self.codes.shape[-1] // BLOCK]
        v = self.codes.to(torch.float32).to(torch.float64).unflatten(-1, (-1, BLOCK)) * scales[..., None]
        return v.flatten(-2)[..., :self.size].to(dtype)

    def __repr__(self):
        return f'Block8({tuple(self.shape)}, device={self.device})'


def _quantize_cpu(rows):
    """(codes, scales) of rows [..., K]."""
    k = rows.shape[-1]
    blocks = -(-k // BLOCK)
    v = F.pad(rows.to(torch.float32), (0, blocks * BLOCK - k)).unflatten(-1, (blocks, BLOCK))
    most = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(-1)
    bits = most.view(torch.int32)
    power = ((bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=-127)  # 448 is 1.75 * 2^8
    power = torch.where(bits == 0, torch.zeros_like(power), power)
    y = v * ((127 - power) << 23).view(torch.float32)[..., None]
    codes = torch.where(torch.isfinite(y), y, torch.full_like(y, float('nan'))).to(torch.float8_e4m3fn).flatten(-2)
    scales = F.pad((power + 127).to(torch.uint8), (0, -blocks % 4), value=127)
    return codes, scales.view(torch.float8_e8m0fnu)


def _quantize_check(x, dim):
    axis = _row_axis(x, dim)
    if not 1 <= x.shape[axis] <= _ext.QUANT8_MOST:
        raise ValueError(f'rows of 1 to {_ext.QUANT8_MOST} values expected, got {x.shape[axis]}')
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f'unsupported dtype {x.dtype}; expected float32, float16 or bfloat16')
    return axis


def quantize8(input, dim=-1):
    """``input`` [..., K] (fp32, fp16 or bf16; with ``dim=1`` the channels of each pixel of a map [N, C, H, W], whose codes
    are [N, H, W, ...]) as a ``Block8``.  Not differentiable: the result is constants."""
    axis = _quantize_check(input, dim)
    if input.is_cuda:
        held = None if torch.compiler.is_compiling() else _ext.native().quantize8(input, dim)
        codes, scales = held or torch.ops.kadconv.quantize8(input.detach(), dim)
    else:
        codes, scales = _quantize_cpu(input.detach().movedim(axis, -1))
    return Block8(codes, scales, input.shape[axis])


def _act_cpu(z, act):
    return {None: lambda t: t, 'relu': F.relu, 'silu': F.silu}[act](z)


def _check_act(act):
    if act not in _ACTS:
        raise ValueError(f"act {act!r} is none of None, 'relu', 'silu'")


def matmul8(a, b, bias=None, act=None, dtype=torch.bfloat16):
    """act(a b^T + bias) for a ``Block8`` a [..., K] and b [N, K]: [..., N] of ``dtype`` (fp32, fp16 or bf16).

    Sums are 32-bit.  A result in fp32 is a sum of exact products; for one in 16 bits the matrix instruction cuts the
    products of eight consecutive k to 2^-13 of the largest of them, which comes to 1e-5 to 5e-5 of the result.
    Inference only."""
    if not isinstance(a, Block8) or not isinstance(b, Block8):
        raise TypeError('a and b must be Block8')
    if len(b.shape) != 2 or a.size != b.size:
        raise ValueError(f'a [..., K] and b [N, K] expected, got {tuple(a.shape)} and {tuple(b.shape)}')
    if a.device != b.device or (bias is not None and bias.device != a.device):
        raise ValueError('a, b and bias must be on one device')
    if bias is not None and tuple(bias.shape) != (b.shape[0],):
        raise ValueError(f'bias must have shape ({b.shape[0]},), got {tuple(bias.shape)}')
    if bias is not None and torch.is_grad_enabled() and bias.requires_grad:
        raise NotImplementedError('kadconv.matmul8 has no gradient')
    _check_act(act)
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f'unsupported dtype {dtype}; expected float32, float16 or bfloat16')
    if a.codes.is_cuda:
        args = a.codes, a.scales, b.codes, b.scales, a.size, bias, act, dtype
        y = None if torch.compiler.is_compiling() else _ext.native().matmul8(*args)
        return torch.ops.kadconv.matmul8(*args) if y is None else y
    z = F.linear(a.dequantize(torch.float64), b.dequantize(torch.float64), None if bias is None else bias.double())
    return _act_cpu(z, act).to(dtype)


def _gradient_check(rows, outputs, need_x, need_weight, need_bias):
    """The limits of gradients on the GPU: sums over the rows, and over the outputs."""
    if need_weight and rows > _ext.GEMM8_MOST:
        raise ValueError(f'a weight has a gradient of up to {_ext.GEMM8_MOST} rows, got {rows}')
    in_memory = need_weight or need_bias or (need_x and rows > _ext.GEMM8_FEW)
    most = _ext.QUANT8_MOST if in_memory else _ext.GEMM8_MOST if need_x else outputs
    if rows and outputs > most:
        raise ValueError(f'gradients of up to {most} outputs expected, got {outputs}')


def _linear8_check(x, weight, bias, act, dim):
    axis = _quantize_check(x, dim)
    kept = isinstance(weight, Block8)
    if len(weight.shape) != 2 or weight.shape[0] < 1:
        raise ValueError(f'weight [N, K] expected, got {tuple(weight.shape)}')
    if x.shape[axis] != weight.shape[1]:
        raise ValueError(f'rows of {weight.shape[1]} values expected, got {x.shape[axis]}')
    if weight.device != x.device:
        raise ValueError('input and weight must be on one device')
    if not kept and weight.dtype not in (torch.float32, x.dtype):
        raise TypeError(f'weight must be float32 or {x.dtype}, got {weight.dtype}')
    _check_param(bias, x, weight.shape[0], 'bias')
    _check_act(act)
    if torch.is_grad_enabled():
        grad = x.requires_grad or (bias is not None and bias.requires_grad)
        if kept and grad:
            raise NotImplementedError('kadconv.linear8 with a weight in 8 bits has no gradient')
        if act is not None and not kept and (grad or weight.requires_grad):
            raise NotImplementedError('kadconv.linear8 with an activation has no gradient')
        if x.is_cuda and not kept:
            _gradient_check(x.numel() // x.shape[axis], weight.shape[0], x.requires_grad, weight.requires_grad,
                            bias is not None and bias.requires_grad)
    return axis


def _rounded(rows):
    """The numbers, in 64 bits, that rows [..., K] are held as."""
    return Block8(*_quantize_cpu(rows), rows.shape[-1]).dequantize(torch.float64)


class _Linear8CPU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(x, weight)
        ctx.bias = None if bias is None else bias.dtype
        z = F.linear(_rounded(x), _rounded(weight), None if bias is None else bias.double())
        return z.to(x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        rows = dy.reshape(-1, dy.shape[-1])
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = (_rounded(dy) @ _rounded(weight.t()).t()).to(x.dtype)
        if ctx.needs_input_grad[1]:
            dw = torch.zeros_like(weight) if not rows.shape[0] else \
                (_rounded(rows.t()) @ _rounded(x.reshape(-1, x.shape[-1]).t()).t()).to(weight.dtype)
        if ctx.needs_input_grad[2]:
            db = rows.double().sum(0).to(ctx.bias)
        return dx, dw, db


def _linear8_cpu(x, weight, bias, act, axis):
    rows = x.movedim(axis, -1)
    if isinstance(weight, Block8):
        z = F.linear(_rounded(rows.detach()), weight.dequantize(torch.float64), None if bias is None else bias.detach().double())
        return _act_cpu(z, act).to(x.dtype).movedim(-1, axis)
    if act is None:
        return _Linear8CPU.apply(rows, weight, bias).movedim(-1, axis)
    z = F.linear(_rounded(rows.detach()), _rounded(weight.detach()), None if bias is None else bias.detach().double())
    return _act_cpu(z, act).to(x.dtype).movedim(-1, axis)


def linear8_forward(x, weight, bias, act, dim):
    """linear8 without a graph of gradients."""
    if isinstance(weight, Block8):
        return _ext.native().linear8_kept_forward(x, weight.codes, weight.scales, weight.size, bias, act, dim)
    return _ext.native().linear8_forward(x, weight, bias, act, dim)


def linear8_backward(dy, x, weight, bias, dim, need_x=True, need_weight=True, need_bias=True):
    """(dx, dweight, dbias) of linear8; None for what is not needed or has no tensor."""
    return _ext.native().linear8_backward(dy, x, weight, bias, dim, need_x, need_weight, need_bias)


def linear8(input, weight, bias=None, act=None, dim=-1):
    """act(x W^T + bias) with x and W in 8 bits along K: ``input`` x [..., K], or with ``dim=1`` the channels of each pixel
    of a map [N, K, H, W] (a 1 x 1 convolution); ``weight`` W [N, K] a ``Block8`` that is kept, or numbers (float32 or
    input's dtype) that are brought to 8 bits in the call; ``bias`` [N] (float32 or input's dtype); ``act`` None, 'relu'
    or 'silu'.  The result has input's dtype; its sums are those of ``matmul8``.

    With numbers as weight and no ``act`` it is differentiable once.  Gradients pass the rounding as if it were not there,
    and are products in 8 bits themselves: that of x is dy W, both along N, that of W is dy^T x, both along the rows; that
    of the bias is the sum of dy.  For them x and W are kept in 8 bits, not as they are: later changes of either are not
    seen.  On the GPU the gradient of W takes up to 2^22 rows, and gradients up to 2^20 outputs N (that of x alone, of up to 32
    rows, 2^22).

    GPU tensors (fp32, fp16, bf16) run the gfx950 HIP kernels; rows that lie a fixed distance apart are read where they
    are.  Up to 32 rows, and short ones (up to 512 values), take one launch, their numbers brought to 8 bits by the product's
    own threads.  The result is
    dense (a map's: channels-last).  CPU tensors run the plain composition."""
    kept = isinstance(weight, Block8)
    if input.is_cuda and not torch.compiler.is_compiling():
        native = _ext.native()  # with the same checks
        y = native.linear8_kept(input, weight.codes, weight.scales, weight.size, bias, act, dim) if kept else \
            native.linear8(input, weight, bias, act, dim)
        if y is not None:  # not traced, and no tensor a fake one
            return y
    axis = _linear8_check(input, weight, bias, act, dim)
    if input.is_cuda:
        if kept:
            return torch.ops.kadconv.linear8_kept(input, weight.codes, weight.scales, weight.size, bias, act, dim)
        return torch.ops.kadconv.linear8(input, weight, bias, act, dim)
    return _linear8_cpu(input, weight, bias, act, axis)
