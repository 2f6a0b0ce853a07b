"""The other fused blocks on the north-star path.

* ``Conv1x1SiLU`` -- KAD-CNet's ``Conv`` (1x1 conv + BN + SiLU) after Conv-BN
  fusion (KAD-CNet/models/common.py:43-57, utils/torch_utils.py:244-265):
  SiLU(W x + b) as one MFMA GEMM with a fused epilogue.
* ``SqueezeExcitation`` -- the channel attention KADConv applies per branch
  (KAD-Conv/kadconv/kad_conv.py:105-109,117), as a standalone block with a
  reduction ratio: GAP -> Linear -> ReLU -> Linear -> sigmoid -> channel scale.
* ``KADDown`` -- stride-2 multi-branch downsampling with a learnable softmax
  over branches and a per-channel sigmoid selection gate.  The reference has
  no such operator; it is defined here from KADConv's branch structure
  (kad_conv.py:112-121) as
      y = sigmoid(gate) * sum_i softmax(alpha)_i * up(conv1x1_i(avgpool(x, 2^(i+1))))
  with up = bilinear (align_corners=False) to (H // 2, W // 2).
* ``GroupNormAct`` -- group norm and an activation on channels-last maps, for
  layers trained at a batch too small for batch statistics.
* ``LayerNorm`` -- layer norm of rows or of each pixel's channels.
* ``Linear8`` -- a linear layer or 1 x 1 convolution whose products are in 8 bits.

The first three: eval-mode GPU inputs run the HIP kernels (no fallback: a missing library
raises); training mode or CPU inputs run the plain torch composition.
``GroupNormAct``, ``LayerNorm`` and ``Linear8`` run them in training mode too: their kernels have a backward.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _ext, block8, ops


def _use_hip(module, x):
    return (not module.training and x.is_cuda and x.dim() == 4
            and x.dtype in (torch.float32, torch.float16, torch.bfloat16))


class Conv1x1SiLU(nn.Module):
    def __init__(self, c1, c2):
        super().__init__()
        self.conv = nn.Conv2d(c1, c2, 1, bias=True)
        self._packed = {}

    @classmethod
    def from_conv_bn(cls, conv, bn):
        """Fold a bias-free 1x1 Conv2d followed by BatchNorm2d (eval statistics)."""
        m = cls(conv.in_channels, conv.out_channels)
        with torch.no_grad():
            a = bn.weight / torch.sqrt(bn.running_var + bn.eps)
            m.conv.weight.copy_(conv.weight * a.view(-1, 1, 1, 1))
            b = conv.bias if conv.bias is not None else torch.zeros_like(bn.bias)
            m.conv.bias.copy_((b - bn.running_mean) * a + bn.bias)
        return m.to(conv.weight.device)

    def forward(self, x):
        if _use_hip(self, x):
            # packed weights and the fp32 bias are cached per parameter version
            key = (x.dtype, self.conv.weight._version, self.conv.weight.data_ptr(), self.conv.bias._version,
                   self.conv.bias.data_ptr())
            if key not in self._packed:
                self._packed = {key: (_ext.gemm_pack_weights(self.conv.weight, x.dtype),
                                      self.conv.bias.detach().float().contiguous())}
            wpack, bias = self._packed[key]
            with torch.no_grad():
                return ops.conv1x1(x, self.conv.weight, bias, act='silu', wpack=wpack)
        return F.silu(self.conv(x))


class SqueezeExcitation(nn.Module):
    def __init__(self, c, reduction=16, min_hidden=1):
        super().__init__()
        hid = max(min_hidden, c // reduction)
        self.fc = nn.Sequential(nn.Linear(c, hid), nn.ReLU(), nn.Linear(hid, c), nn.Sigmoid())
        self._f32 = {}

    def forward(self, x):
        if _use_hip(self, x):
            # fp32 copies of the MLP parameters, cached per parameter version
            ps = (self.fc[0].weight, self.fc[0].bias, self.fc[2].weight, self.fc[2].bias)
            key = tuple((p._version, p.data_ptr()) for p in ps)
            if key not in self._f32:
                self._f32 = {key: tuple(p.detach().float().contiguous() for p in ps)}
            with torch.no_grad():
                return ops.squeeze_excitation(x, *self._f32[key])
        return x * self.fc(x.mean(dim=(2, 3))).view(x.shape[0], -1, 1, 1)


class KADDown(nn.Module):
    def __init__(self, c1, c2, n=3):
        super().__init__()
        self.n = n
        self.proj = nn.ModuleList(nn.Conv2d(c1, c2, 1) for _ in range(n))
        self.alpha = nn.Parameter(torch.zeros(n))
        self.gate = nn.Parameter(torch.zeros(c2))
        self._packed = {}

    def _plain(self, x):
        ho, wo = x.shape[2] // 2, x.shape[3] // 2
        a = torch.softmax(self.alpha, dim=0)
        z = 0
        for i in range(self.n):
            b = self.proj[i](F.avg_pool2d(x, kernel_size=2 ** (i + 1)))
            if b.shape[2:] != (ho, wo):
                b = F.interpolate(b, size=(ho, wo), mode='bilinear', align_corners=False)
            z = z + a[i] * b
        return z * torch.sigmoid(self.gate).view(1, -1, 1, 1)

    # kad_kaddown_prep keeps a plane's 2x2, 4x4 and 8x8 means in LDS as fp32 (160 KB per CU)
    _PREP_LDS = 160 * 1024

    def _hip_eligible(self, x):
        H, W = x.shape[2:]
        pools = (H // 2) * (W // 2) + (H // 4) * (W // 4) + (H // 8) * (W // 8)
        return (_use_hip(self, x) and 1 <= self.n <= 3 and H >= 2 ** self.n and W >= 2 ** self.n
                and 4 * pools <= self._PREP_LDS)

    def forward(self, x):
        # inputs the one-pass kernel does not cover (n > 3 branches, planes whose pools exceed
        # its LDS staging, images smaller than the deepest pool) take the plain composition
        if not self._hip_eligible(x):
            return self._plain(x)
        with torch.no_grad():
            return self._fast(x)

    def _fast(self, x):
        """One input pass (kad_kaddown_prep: the pooled inputs of every branch at
        (H/2, W/2), stacked along channels) and one 1x1 GEMM over them with the
        branch projections stacked along Cin; softmax(alpha) and sigmoid(gate)
        are folded into the packed weights and bias.  A 1x1 projection commutes
        with the bilinear resize (its weights sum to 1), so this equals the
        per-branch form of ``_plain``."""
        N, C, H, W = x.shape
        c2 = self.proj[0].weight.shape[0]
        dtype = x.dtype
        # folded weights are cached per parameter version (no per-call host work)
        params = [p.weight for p in self.proj] + [p.bias for p in self.proj] + [self.alpha, self.gate]
        key = (dtype,) + tuple((p._version, p.data_ptr()) for p in params)
        if key not in self._packed:
            a = torch.softmax(self.alpha.detach().float(), dim=0)
            g = torch.sigmoid(self.gate.detach().float())
            w = torch.cat([a[i] * self.proj[i].weight.detach().float().reshape(c2, C) for i in range(self.n)], dim=1)
            b = sum(a[i] * self.proj[i].bias.detach().float() for i in range(self.n))
            self._packed = {key: (_ext.gemm_pack_weights(w * g[:, None], dtype), (g * b).contiguous())}
        wpack, bias = self._packed[key]
        if N == 0:  # nothing to compute: the empty result
            return torch.empty(N, c2, H // 2, W // 2, dtype=dtype, device=x.device)
        u = torch.empty(N, self.n * C, H // 2, W // 2, dtype=dtype, device=x.device)
        _ext.kaddown_prep(x.contiguous(), u, self.n)
        out = torch.empty(N, c2, H // 2, W // 2, dtype=dtype, device=x.device)
        _ext.gemm1x1_fwd(u, _ext.KAD_NCHW, self.n * C, wpack, c2, out, _ext.KAD_NCHW, bias=bias)
        if x.is_contiguous(memory_format=torch.channels_last) and not x.is_contiguous():
            out = out.contiguous(memory_format=torch.channels_last)
        return out


class GroupNormAct(nn.Module):
    """act(group_norm(x)); parameters as torch.nn.GroupNorm's, so its state dicts load."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, act='silu'):
        super().__init__()
        if num_groups < 1 or num_channels % num_groups:
            raise ValueError(f'{num_groups} groups do not divide {num_channels} channels')
        if act not in (None, 'relu', 'silu'):
            raise ValueError(f"act {act!r} is none of None, 'relu', 'silu'")
        self.num_groups, self.num_channels, self.eps, self.act = num_groups, num_channels, eps, act
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def forward(self, x):
        return ops.group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.act)

    def extra_repr(self):
        return f'{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.weight is not None}, act={self.act!r}'


class LayerNorm(nn.Module):
    """Layer norm of rows of ``num_channels`` values, along the last axis or, with ``dim=1``, of each pixel of a map
    [N, C, H, W]; parameters as torch.nn.LayerNorm's, so its state dicts load."""

    def __init__(self, num_channels, eps=1e-5, affine=True, dim=-1):
        super().__init__()
        if num_channels < 1:
            raise ValueError(f'at least one channel expected, got {num_channels}')
        if dim not in (-1, 1):
            raise ValueError(f'dim must be -1 or 1, got {dim}')
        self.num_channels, self.eps, self.dim = num_channels, eps, dim
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def forward(self, x):
        if x.shape[ops._row_axis(x, self.dim)] != self.num_channels:
            raise ValueError(f'rows of {self.num_channels} values expected, got {tuple(x.shape)} along axis {self.dim}')
        return ops.layer_norm(x, self.weight, self.bias, self.eps, self.dim)

    def extra_repr(self):
        return f'{self.num_channels}, eps={self.eps}, affine={self.weight is not None}, dim={self.dim}'


class Linear8(nn.Module):
    """x W^T + b along the last axis or, with ``dim=1``, of each pixel of a map [N, C, H, W] (a 1 x 1 convolution), the
    products in 8 bits (``kadconv.linear8``); parameters as torch.nn.Linear's, so its state dicts load.

    Every call brings W to 8 bits as it is then.  A program that serves spares that: ``keep()`` makes a copy in 8 bits, by which
    the calls go that follow in eval mode, where nothing is differentiated; ``act`` is part of such a call's launch.  The
    copy is dropped where W is seen to have changed (another tensor or version of it, ``train()``); writes that no version
    tells, through ``.data`` or by the replay of a graph, need another ``keep()``.  Traced calls, and ones that are captured into
    a graph, go by W itself, and so do their replays.  (For a graph that reads W in 8 bits only, capture ``kadconv.linear8``
    with ``kadconv.quantize8(W)``.)"""

    def __init__(self, in_features, out_features, bias=True, act=None, dim=-1):
        super().__init__()
        if in_features < 1 or out_features < 1:
            raise ValueError(f'positive sizes expected, got {in_features} and {out_features}')
        if act not in (None, 'relu', 'silu'):
            raise ValueError(f"act {act!r} is none of None, 'relu', 'silu'")
        if dim not in (-1, 1):
            raise ValueError(f'dim must be -1 or 1, got {dim}')
        self.in_features, self.out_features, self.act, self.dim = in_features, out_features, act, dim
        like = nn.Linear(in_features, out_features, bias)
        self.weight, self.bias = like.weight, like.bias
        self._kept = None  # (W, what it is known by, the copy, the stream that it was made on, and when)

    def __getstate__(self):
        return {**self.__dict__, '_kept': None}  # a copy of the module makes its own

    def train(self, mode=True):
        if mode:
            self._kept = None
        return super().train(mode)

    def _known_by(self):
        w = self.weight
        return w.data_ptr(), w.shape, w.stride(), w.dtype, 0 if w.is_inference() else w._version

    def keep(self, on=True):
        """Makes the copy of W in 8 bits that calls in eval mode go by (on=False: drops it); returns the module."""
        self._kept = None
        if not on:
            return self
        w = self.weight.detach()  # held, so that its address is no other's
        if self.training or not w.is_cuda or type(self.weight) is not nn.Parameter:
            raise RuntimeError('keep() is for eval mode and a parameter on a GPU')
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError('keep() cannot be captured into a graph')
        stream = torch.cuda.current_stream(w.device)
        copy = block8.quantize8(w)
        self._kept = w, self._known_by(), copy, stream, stream.record_event()
        return self

    def _weight8(self):
        """The copy, for the current stream; None where there is none of W as it is."""
        if self._kept is None:
            return None
        w, known_by, copy, made_on, made = self._kept
        if known_by != self._known_by():
            self._kept = None
            return None
        stream = torch.cuda.current_stream(w.device)
        if stream != made_on:
            stream.wait_event(made)
            copy.codes.record_stream(stream)
            copy.scales.record_stream(stream)
        return copy

    def forward(self, x):
        grad = torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in self.parameters()))
        if grad and self.act is not None:
            return {'relu': F.relu, 'silu': F.silu}[self.act](block8.linear8(x, self.weight, self.bias, None, self.dim))
        weight = self.weight
        if not (grad or self.training or torch.compiler.is_compiling()) and self._kept is not None and x.is_cuda and \
                type(weight) is nn.Parameter and not _ext.native().observed(x, weight) and \
                not torch.cuda.is_current_stream_capturing():
            copy = self._weight8()
            weight = weight if copy is None else copy
        return block8.linear8(x, weight, self.bias, self.act, self.dim)

    def extra_repr(self):
        return f'{self.in_features}, {self.out_features}, bias={self.bias is not None}, act={self.act!r}, dim={self.dim}'
