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
    with pytest.raises(ValueError, match='dim must'):
        kadconv.LayerNorm(4, dim=1)(x[0])
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


# ---------------------------------------------------------------------------- distillation
def _logits(dim=-1):
    g = torch.Generator().manual_seed(1)
    shape = (3, 6, 5) if dim == -1 else (3, 5, 2, 3)
    z = torch.randn(shape, generator=g, dtype=torch.float64)
    top = torch.topk(torch.randn(shape, generator=g, dtype=torch.float64), 3, dim=dim)
    return z, top.values, top.indices


@pytest.mark.parametrize('dim', [-1, 1])
def test_distill_plain(dim):
    from tests._distill_ref import reference
    z, t, i = _logits(dim)
    i.movedim(dim, -1)[0] = -1
    z.movedim(dim, -1)[0] = float('nan')
    zs = z.clone().requires_grad_(True)
    rows = [a.movedim(dim, -1).reshape(-1, a.shape[dim]) for a in (z, t, i)]
    loss = kadconv.distill_loss(zs, t, i, 2.0, 'none', dim)
    g = torch.rand(loss.shape, dtype=torch.float64)
    ref = reference(*rows, 2.0, g.reshape(-1))
    assert torch.allclose(loss.reshape(-1), ref['loss'], atol=1e-12)
    dz, = torch.autograd.grad(loss, zs, g)
    assert torch.allclose(dz.movedim(dim, -1).reshape(-1, z.shape[dim]), ref['dz'], atol=1e-12)
    mean = kadconv.distill_loss(z, t, i, 2.0, 'mean', dim)
    assert torch.allclose(mean, ref['loss'].sum() / ref['live'].sum(), atol=1e-12)
    full = torch.topk(torch.randn(4, 6, dtype=torch.float64), 6, dim=1)  # all classes: the divergence itself
    z = torch.randn(4, 6, dtype=torch.float64)
    p = torch.zeros(4, 6, dtype=torch.float64).scatter(1, full.indices, torch.softmax(full.values, 1))
    want = torch.nn.functional.kl_div(torch.log_softmax(z, 1), p, reduction='batchmean')
    assert torch.allclose(kadconv.distill_loss(z, full.values, full.indices), want, atol=1e-12)


def test_distill_refusals():
    z, t, i = _logits()
    for args, match in (((z[..., :0], t, i), 'class'), ((z, t[0], i[0]), 'one shape'), ((z, t, i[..., :2]), 'one shape'),
                        ((z[:2], t, i), 'shape of logits'), ((z, t[..., :0], i[..., :0]), 'entries')):
        with pytest.raises(ValueError, match=match):
            kadconv.distill_loss(*args)
    for temperature in (0.0, -1.0, 9e-7, 1.1e6, float('inf'), float('nan')):
        with pytest.raises(ValueError, match='temperature'):
            kadconv.distill_loss(z, t, i, temperature)
    with pytest.raises(ValueError, match='reduction'):
        kadconv.distill_loss(z, t, i, reduction='max')
    with pytest.raises(ValueError, match='dim must'):
        kadconv.distill_loss(z, t, i, dim=1)
    with pytest.raises(TypeError, match='int32'):
        kadconv.distill_loss(z, t, i.short())
    with pytest.raises(TypeError, match='floating'):
        kadconv.distill_loss(z.long(), t, i)
    with pytest.raises(ValueError, match='GPU'):
        _ext.native().distill_loss(z.float(), t.float(), i, 1.0, 'mean', -1)
    with pytest.raises(ValueError, match='needs a GPU'):
        torch.ops.kadconv.distill_loss(z, t, i, 1.0, 'mean', -1)


def _distill_args(**kw):
    a = _ext.DistillArgs()
    for f in ('logits', 'teacher', 'index', 'dloss', 'dlogits', 'stats', 'loss', 'share', 'work'):
        setattr(a, f, 4096)
    a.rows, a.v, a.z_rs, a.inner, a.k, a.temperature, a.reduction = 3, 8, 8, 3, 2, 1.0, 2
    a.t_sp = a.i_sp = 2
    a.t_sk = a.i_sk = 1
    a.dtype = a.teacher_dtype = _ext.KAD_F16
    a.index_bits = 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize('kw', [dict(logits=None), dict(teacher=None), dict(index=None), dict(loss=None), dict(work=None), dict(rows=0),
                                dict(rows=1 << 31), dict(v=0), dict(v=(1 << 30) + 1), dict(k=0), dict(k=1025), dict(z_rs=7),
                                dict(z_rs=1 << 31), dict(inner=0), dict(t_sk=-1), dict(i_sn=-1), dict(t_sp=1 << 32), dict(i_sk=1 << 32), dict(temperature=0.0), dict(temperature=1e7), dict(reduction=3),
                                dict(dtype=9), dict(teacher_dtype=-1), dict(index_bits=16)], ids=str)
def test_distill_c_refuses(kw):
    lib = _ext.load()
    assert lib.kad_distill_fwd(ctypes.byref(_distill_args(**kw)), None) == -1
    assert b'kad_distill' in lib.kad_last_error()


@pytest.mark.parametrize('kw', [dict(dloss=None), dict(dlogits=None), dict(stats=None), dict(share=None)], ids=str)
def test_distill_backward_c_refuses(kw):
    assert _ext.load().kad_distill_bwd(ctypes.byref(_distill_args(**kw)), None) == -1


def test_distill_work():
    """Two floats for each block that has losses, and for each part of a row."""
    lib = _ext.load()
    def work(**kw):
        return lib.kad_distill_work_elems(ctypes.byref(_distill_args(**kw)))
    assert work(reduction=0) == 0 and work() == 2
    for v in list(range(8192, 8400)) + list(range(100000, 100100)) + [1 << 30]:
        for rows in (1, 2, 7, 511, 512):
            for dtype in (0, 1):
                n = work(rows=rows, v=v, z_rs=v, dtype=dtype)
                assert 2 * rows <= n <= 2 * rows + 2 * rows * 256


# ---------------------------------------------------------------------------- products in 8 bits
def test_quantize8_plain():
    from tests._block8_ref import held, numbers
    g = torch.Generator().manual_seed(2)
    for k in (1, 100, 128, 129, 700):
        x = torch.randn(5, k, generator=g) * torch.exp(3 * torch.randn(5, k, generator=g))
        x[0, 0] = float('nan')
        x[1] = 0
        q = kadconv.quantize8(x)
        codes, powers = held(x)
        assert q.shape == (5, k) and q.codes.shape[1] == -(-k // 128) * 128 and q.scales.shape[1] % 4 == 0
        got = q.codes[:, :k].float().double()
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(codes)) and torch.equal(torch.isnan(got), torch.isnan(codes))
        assert torch.equal(q.scales.view(torch.uint8)[:, :powers.shape[1]].int() - 127, powers.int())
        assert torch.equal(torch.nan_to_num(q.dequantize(torch.float64)), torch.nan_to_num(numbers(x)))


def test_linear8_plain():
    from tests._block8_ref import numbers
    g = torch.Generator().manual_seed(3)
    x, w, b, dy = (torch.randn(*s, generator=g) for s in ((2, 6, 3, 4), (5, 6), (5,), (2, 5, 3, 4)))
    rows, drows = x.permute(0, 2, 3, 1).reshape(-1, 6), dy.permute(0, 2, 3, 1).reshape(-1, 5)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = kadconv.linear8(*leaves, dim=1)
    want = numbers(rows) @ numbers(w).t() + b.double()
    assert torch.allclose(y.permute(0, 2, 3, 1).reshape(-1, 5).double(), want, atol=1e-5)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.allclose(dx.permute(0, 2, 3, 1).reshape(-1, 6).double(), numbers(drows) @ numbers(w.t()).t(), atol=1e-5)
    assert torch.allclose(dw.double(), numbers(drows.t()) @ numbers(rows.t()).t(), atol=1e-5)
    assert torch.allclose(db, drows.sum(0), atol=1e-5)
    kept = kadconv.quantize8(w)
    served = kadconv.linear8(x, kept, b, 'silu', dim=1)
    assert torch.allclose(served, torch.nn.functional.silu(y.detach()), atol=1e-5)
    assert torch.equal(kadconv.linear8(x, w, b, 'silu', dim=1), served)
    z = kadconv.matmul8(kadconv.quantize8(x, dim=1), kept, b, 'relu', torch.float32)
    assert torch.allclose(z.permute(0, 3, 1, 2), y.detach().clamp(min=0), atol=1e-5)
    m = kadconv.Linear8(6, 5, act='silu', dim=1)
    m.load_state_dict(torch.nn.Linear(6, 5).state_dict())
    m(x).sum().backward()
    assert m.weight.grad.shape == (5, 6)
    m.eval()
    with torch.no_grad():
        assert m(x).shape == (2, 5, 3, 4)
    x0 = torch.empty(0, 6, requires_grad=True)
    assert not torch.autograd.grad(kadconv.linear8(x0, leaves[1]).sum(), leaves[1])[0].any()


def test_block8_refusals():
    x, w = torch.randn(3, 40), torch.randn(5, 40)
    q = kadconv.quantize8(w)
    for args in ((q.codes, q.scales, 129), (q.codes, q.scales, 0), (q.codes[:4], q.scales, 40), (q.codes, q.scales[:, :1], 40)):
        with pytest.raises(ValueError):
            kadconv.Block8(*args)
    with pytest.raises(TypeError):
        kadconv.Block8(q.codes.view(torch.uint8), q.scales, 40)
    for bad in (x.double(), x.long()):
        with pytest.raises(TypeError):
            kadconv.quantize8(bad)
        with pytest.raises(TypeError):
            kadconv.linear8(bad, q)
    with pytest.raises(ValueError):
        kadconv.quantize8(x[:, :0])
    with pytest.raises(ValueError, match='dim must'):
        kadconv.quantize8(x, dim=0)
    for args, match in (((x[:, :39], w), 'rows of 40'), ((x, w[0]), 'weight'), ((x, w, torch.zeros(4)), 'bias'),
                        ((x, w, None, 'gelu'), 'act')):
        with pytest.raises(ValueError, match=match):
            kadconv.linear8(*args)
    with pytest.raises(TypeError, match='weight'):
        kadconv.linear8(x, w.half())
    with pytest.raises(NotImplementedError, match='8 bits'):
        kadconv.linear8(x.requires_grad_(True), q)
    with pytest.raises(NotImplementedError, match='activation'):
        kadconv.linear8(x, w, act='relu')
    x = x.detach()
    with pytest.raises(TypeError, match='Block8'):
        kadconv.matmul8(x, q)
    with pytest.raises(ValueError, match='expected'):
        kadconv.matmul8(kadconv.quantize8(x[:, :39]), q)
    with pytest.raises(TypeError, match='dtype'):
        kadconv.matmul8(kadconv.quantize8(x), q, dtype=torch.float64)
    with pytest.raises(ValueError, match='bias'):
        kadconv.matmul8(kadconv.quantize8(x), q, torch.zeros(4))
    for args in ((0, 4), (4, 0), (4, 4, True, 'tanh'), (4, 4, True, None, 2)):
        with pytest.raises(ValueError):
            kadconv.Linear8(*args)
    with pytest.raises(ValueError, match='GPU'):
        _ext.native().linear8(x, w, None, None, -1)
    with pytest.raises(ValueError, match='GPU'):
        _ext.native().quantize8(x, -1)


def _quant_args(**kw):
    a = _ext.Quant8Args()
    for f in ('x', 'codes', 'scales', 't_codes', 't_scales', 'sums', 'work'):
        setattr(a, f, 4096)
    a.rows, a.x_rs, a.c, a.dtype, a.sums_dtype = 3, 8, 8, 1, 0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize('kw', [dict(x=None), dict(codes=None), dict(scales=None), dict(t_codes=None), dict(codes=4104), dict(work=None),
                                dict(rows=0), dict(rows=1 << 31), dict(c=0), dict(c=(1 << 20) + 1), dict(x_rs=7), dict(x_rs=1 << 31),
                                dict(dtype=3), dict(sums_dtype=3), dict(rows=1 << 30, c=1 << 20, x_rs=1 << 20),
                                dict(codes=None, scales=None, t_codes=None, t_scales=None, sums=None)], ids=str)
def test_quant8_c_refuses(kw):
    lib = _ext.load()
    assert lib.kad_quant8(ctypes.byref(_quant_args(**kw)), None) == -1
    assert b'kad_quant8' in lib.kad_last_error()


def _gemm_args(**kw):
    a = _ext.Gemm8Args()
    for f in ('a', 'a_scales', 'b', 'b_scales', 'bias', 'out', 'work'):
        setattr(a, f, 4096)
    a.a_rs, a.m, a.n, a.k, a.dtype = 8, 3, 4, 8, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize('kw', [dict(a=None), dict(b=None), dict(b_scales=None), dict(out=None), dict(m=0), dict(n=0), dict(k=0),
                                dict(k=(1 << 22) + 1), dict(m=(1 << 31) - 100), dict(m=1, n=1 << 26), dict(act=7), dict(dtype=5), dict(bias_dtype=-1),
                                dict(a_scales=None, m=65), dict(a_scales=None, a_rs=7), dict(a_scales=None, a_dtype=4), dict(b=4104),
                                dict(a=4104), dict(b_scales=4098), dict(a_scales=4098), dict(m=1 << 20, n=1 << 20),
                                dict(m=100, k=100000, work=None)], ids=str)
def test_gemm8_c_refuses(kw):
    lib = _ext.load()
    assert lib.kad_gemm8(ctypes.byref(_gemm_args(**kw)), None) == -1
    assert b'kad_gemm8' in lib.kad_last_error()


def test_gemm8_takes_values():
    lib = _ext.load()
    takes = lambda **kw: lib.kad_gemm8_takes_values(ctypes.byref(_gemm_args(**{**dict(m=1000, n=64, k=300, a_dtype=1), **kw})))
    assert lib.kad_gemm8_takes_values(None) == 0
    assert takes() == takes(n=128, k=512) == takes(m=1 << 24) == takes(n=1024, k=512) == takes(m=64, n=10000) == takes(n=1 << 20, k=256) == 1
    assert takes(a_dtype=0) == takes(k=513) == takes(m=40000, n=1025) == takes(a_dtype=9, m=3) == 0
    f32 = dict(dtype=0, a_dtype=0)
    assert takes(**f32) == takes(m=40000, n=256, k=512, **f32) == takes(n=1024, **f32) == 1
    assert takes(m=40000, n=257, **f32) == takes(k=513, **f32) == 0
    assert takes(m=32, n=1 << 20, k=1 << 20, a_dtype=0) == 1


def test_gemm8_parts_cover_k():
    """Floats of scratch: none, or one matrix for each part of k."""
    lib = _ext.load()
    for m in (1, 64, 65, 1000, 70000):
        for n in (1, 300, 5000):
            for k in (1, 128, 1000, 20000, 1 << 22):
                for dtype in (0, 1):
                    w = lib.kad_gemm8_work_elems(ctypes.byref(_gemm_args(m=m, n=n, k=k, dtype=dtype)))
                    assert w >= 0 and w % (m * n) == 0 and w // (m * n) != 1 and w // (m * n) <= 512


def test_fake_tensors():
    """Calls on fake GPU tensors give fake results of the right shapes and types, and launch nothing."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(), torch.device('cuda'):
        x, w = torch.empty(5, 70), torch.empty(9, 70)
        held, kept = kadconv.quantize8(x), kadconv.quantize8(w)
        assert held.codes.shape == (5, 128) and held.scales.shape == (5, 4) and held.shape == (5, 70)
        y = kadconv.matmul8(held, kept, dtype=torch.float16)
        assert y.shape == (5, 9) and y.dtype == torch.float16
        assert kadconv.linear8(x, kept, act='relu').shape == kadconv.linear8(x, w).shape == (5, 9)
        m = kadconv.Linear8(70, 9).eval()
        with torch.no_grad():
            assert m(x).shape == m(x).shape == (5, 9) and m._kept is None
        assert kadconv.LayerNorm(70)(x).shape == (5, 70)
        t, i = torch.empty(5, 3), torch.empty(5, 3, dtype=torch.int64)
        assert kadconv.distill_loss(x, t, i).shape == () and kadconv.distill_loss(x, t, i, reduction='none').shape == (5,)
