"""Operators on rows without a GPU: their refusals, the plain compositions of CPU tensors, and the C entries' checks."""
import ctypes

import pytest
import torch

import kadconv
from kadconv import _ext


def test_layer_norm_plain():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 6, 4, 5, generator=g, dtype=torch.float64)
    m = kadconv.LayerNorm(6, dim=1).double()
    want = torch.nn.functional.layer_norm(x.permute(0, 2, 3, 1), (6,)).permute(0, 3, 1, 2)
    assert torch.allclose(m(x), want, atol=1e-12)
    ref = torch.nn.LayerNorm(5).double()
    mine = kadconv.LayerNorm(5).double()
    mine.load_state_dict(ref.state_dict())
    assert torch.equal(mine(x), ref(x))
    assert kadconv.layer_norm(x.bfloat16()).dtype == torch.bfloat16


def test_layer_norm_refusals():
    x = torch.randn(2, 6, 4, 5)
    for dim in (0, 2, 4, -2, -4):
        with pytest.raises(ValueError, match='dim must be'):
            kadconv.layer_norm(x, dim=dim)
    with pytest.raises(ValueError, match='dim must be'):
        kadconv.layer_norm(x[0], dim=1)
    with pytest.raises(ValueError, match='one axis'):
        kadconv.layer_norm(torch.tensor(1.0))
    with pytest.raises(ValueError, match='at least one value'):
        kadconv.layer_norm(x[..., :0])
    with pytest.raises(ValueError, match='weight must have shape'):
        kadconv.layer_norm(x, torch.ones(6))
    with pytest.raises(ValueError, match='eps'):
        kadconv.layer_norm(x, eps=-1.0)
    with pytest.raises(TypeError):
        kadconv.layer_norm(x, torch.ones(5).half())
    with pytest.raises(TypeError, match='share'):
        kadconv.layer_norm(x.half(), torch.ones(5).half(), torch.ones(5))
    with pytest.raises(ValueError):
        kadconv.LayerNorm(0)
    with pytest.raises(ValueError):
        kadconv.LayerNorm(4, dim=2)
    with pytest.raises(ValueError, match='rows of 4'):
        kadconv.LayerNorm(4)(x)
    with pytest.raises(ValueError, match='needs a GPU'):
        torch.ops.kadconv.layer_norm(x, None, None, 1e-5, -1)
    native = _ext.native()
    for call in (lambda: native.layer_norm(x, None, None, 1e-5, -1), lambda: native.layer_norm_forward(x, None, None, 1e-5, -1)):
        with pytest.raises(ValueError, match='GPU'):
            call()


def _ln_args(**kw):
    a = _ext.LayerNormArgs()
    for f in ('x', 'dy', 'out', 'weight', 'bias', 'mean', 'rstd', 'dweight', 'dbias', 'work'):
        setattr(a, f, 4096)
    a.rows, a.c, a.x_rs, a.dy_rs, a.eps, a.dtype, a.param_dtype = 3, 8, 8, 8, 1e-5, _ext.KAD_F16, _ext.KAD_F32
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize('kw', [dict(x=None), dict(rows=0), dict(rows=(1 << 40) + 1), dict(c=0), dict(c=16385), dict(x_rs=7),
                                dict(x_rs=1 << 31), dict(eps=-1.0), dict(dtype=9), dict(param_dtype=_ext.KAD_BF16), dict(out=None),
                                dict(mean=None)], ids=str)
def test_layer_norm_c_refuses(kw):
    lib = _ext.load()
    assert lib.kad_layer_norm_fwd(ctypes.byref(_ln_args(**kw)), None) == -1
    assert b'kad_layer_norm_fwd' in lib.kad_last_error()


@pytest.mark.parametrize('kw', [dict(dy=None), dict(dy_rs=7), dict(work=None), dict(mean=None, rstd=None)], ids=str)
def test_layer_norm_backward_c_refuses(kw):
    assert _ext.load().kad_layer_norm_bwd(ctypes.byref(_ln_args(**kw)), None) == -1


def test_layer_norm_work():
    lib = _ext.load()
    a = _ln_args(rows=1, c=5)
    assert lib.kad_layer_norm_work_elems(ctypes.byref(a)) == 2 * 5          # one block's dw and db
    a = _ln_args(rows=1 << 40, c=16384, x_rs=16384, dy_rs=16384)
    assert 0 < lib.kad_layer_norm_work_elems(ctypes.byref(a)) <= 1024 * 2 * 16384
    assert lib.kad_layer_norm_work_elems(ctypes.byref(_ln_args(c=0))) == -1
