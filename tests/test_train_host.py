"""The training operators without a GPU: refusals, the CPU composition, the chunk table, the C ABI's checks
and the layout of its structs."""
import ctypes
import importlib.util
import os
import shutil
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import kadconv
from kadconv import _ext
from tests._norm_ref import assert_within, reference
from tests.conftest import ROOT


@pytest.mark.parametrize('act', [None, 'relu', 'silu'])
def test_group_norm_act_cpu(act):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 12, 5, 7, generator=g, dtype=torch.float64)
    w, b = torch.randn(12, generator=g).double(), torch.randn(12, generator=g).double()
    dy = torch.randn(2, 12, 5, 7, generator=g, dtype=torch.float64)
    xs, ws, bs = (t.clone().requires_grad_(True) for t in (x, w, b))
    y = kadconv.group_norm_act(xs, 4, ws, bs, 1e-5, act)
    ref = reference(x, 4, w, b, 1e-5, act, dy)
    assert_within(y, ref['y'], ref['tol_y'], 'y')
    dx, dw, db = torch.autograd.grad(y, (xs, ws, bs), dy)
    assert_within(dx, ref['dx'], ref['tol_dx'], 'dx')
    assert_within(dw, ref['dw'], ref['tol_dw'], 'dw')
    assert_within(db, ref['db'], ref['tol_db'], 'db')


def test_reference_gradient_is_the_formulas():
    """The tests' own formulas against automatic differentiation of the definition, in 64 bits."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 10, 4, 3, generator=g, dtype=torch.float64).requires_grad_(True)
    w = torch.randn(10, generator=g, dtype=torch.float64).requires_grad_(True)
    b = torch.randn(10, generator=g, dtype=torch.float64).requires_grad_(True)
    dy = torch.randn(3, 10, 4, 3, generator=g, dtype=torch.float64)
    for act, f in ((None, lambda t: t), ('relu', torch.relu), ('silu', torch.nn.functional.silu)):
        y = f(torch.nn.functional.group_norm(x, 5, w, b, 1e-3))
        ref = reference(x, 5, w, b, 1e-3, act, dy)
        for got, want in zip((y, *torch.autograd.grad(y, (x, w, b), dy)), (ref['y'], ref['dx'], ref['dw'], ref['db'])):
            torch.testing.assert_close(got.detach(), want, rtol=1e-10, atol=1e-12)


def test_group_norm_act_refusals():
    x = torch.randn(2, 12, 3, 3)
    with pytest.raises(ValueError, match='N, C, H, W'):
        kadconv.group_norm_act(x[0], 3)
    with pytest.raises(ValueError, match='divide'):
        kadconv.group_norm_act(x, 5)
    with pytest.raises(ValueError, match='divide'):
        kadconv.group_norm_act(x, 0)
    with pytest.raises(ValueError, match='act'):
        kadconv.group_norm_act(x, 3, act='gelu')
    with pytest.raises(ValueError, match='shape'):
        kadconv.group_norm_act(x, 3, torch.ones(11))
    with pytest.raises(ValueError, match='eps'):
        kadconv.group_norm_act(x, 3, eps=-1.0)
    with pytest.raises(TypeError):
        kadconv.group_norm_act(x.half(), 3, torch.ones(12, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match='divide'):
        kadconv.GroupNormAct(5, 12)
    with pytest.raises(ValueError, match='act'):
        kadconv.GroupNormAct(3, 12, act='gelu')


def test_group_norm_act_module_loads_torch_state():
    ref = torch.nn.GroupNorm(3, 12)
    with torch.no_grad():
        ref.weight.normal_()
        ref.bias.normal_()
    m = kadconv.GroupNormAct(3, 12, act='silu')
    m.load_state_dict(ref.state_dict())
    x = torch.randn(2, 12, 4, 5)
    torch.testing.assert_close(m(x), torch.nn.functional.silu(ref(x)), rtol=1e-5, atol=1e-6)
    assert not list(kadconv.GroupNormAct(3, 12, affine=False).parameters())


def test_group_norm_act_fake():
    with FakeTensorMode():
        x = torch.empty(2, 12, 5, 7, dtype=torch.float16)
        w = torch.empty(12)
        y, mean, rstd = torch.ops.kadconv.group_norm_act(x, 4, w, None, 1e-5, 'silu')
        assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous(memory_format=torch.channels_last)
        assert tuple(mean.shape) == tuple(rstd.shape) == (2, 4) and mean.dtype == torch.float32
        dx, dw, db = torch.ops.kadconv.group_norm_act_backward(y, x, 4, w, None, mean, rstd, 1e-5, 'silu')
        assert dx.shape == x.shape and dw.shape == w.shape and db.numel() == 0


def test_group_norm_statistics_have_no_gradient():
    """mean and rstd of the operator are constants to autograd: a loss of them alone is refused, not taken for one of y."""
    with FakeTensorMode():
        x, w = torch.empty(2, 12, 5, 7).requires_grad_(True), torch.empty(12, requires_grad=True)
        y, mean, rstd = torch.ops.kadconv.group_norm_act(x, 4, w, None, 1e-5, 'silu')
        assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad
        for t in (mean, rstd):
            with pytest.raises(RuntimeError, match='does not require grad'):
                t.sum().backward()
        dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
        assert dx.shape == x.shape and dw.shape == w.shape


def test_group_norm_act_of_fake_gpu_maps():
    """The public function on tensors without values, in their mode and outside of it: shapes, and nothing run."""
    with FakeTensorMode():
        x = torch.empty(2, 12, 5, 7, dtype=torch.float16, device='cuda').requires_grad_(True)
        w = torch.empty(12, device='cuda', requires_grad=True)
        y = kadconv.group_norm_act(x, 4, w, act='silu')
        assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous(memory_format=torch.channels_last)
        with pytest.raises(ValueError, match='divide'):
            kadconv.group_norm_act(x, 5, w)
    assert type(kadconv.group_norm_act(x.detach(), 4)) is type(x)


@pytest.mark.parametrize('backward', [False, True], ids=['forward', 'backward'])
def test_group_norm_entries_check_weight_and_bias(backward):
    """The functions below the autograd one, and the gradient's operator: what they are given is checked before
    anything is allocated or launched (here: before the map is found to be on the CPU)."""
    x, stat = torch.zeros(2, 12, 3, 3, dtype=torch.float16), torch.zeros(2, 3)
    ok = torch.ones(12)

    def call(w, b, x=x, groups=3, eps=1e-5):
        if backward:
            kadconv.ops.group_norm_act_backward(x, x, groups, w, b, stat, stat, eps, 'silu')
        else:
            kadconv.ops.group_norm_act_forward(x, groups, w, b, eps, 'silu')
    for w, b, error, words in ((torch.ones(11), None, ValueError, 'shape'), (ok, torch.ones(1, 12), ValueError, 'shape'),
                               (None, torch.ones(13), ValueError, 'shape'), (ok, ok.half(), TypeError, 'share'),
                               (ok.half(), ok, TypeError, 'share'), (ok.bfloat16(), None, TypeError, 'float32'),
                               (ok.to('meta'), None, ValueError, 'one device'), (ok, ok, ValueError, 'GPU')):
        with pytest.raises(error, match=words):
            call(w, b)
        if backward and words not in ('GPU', 'one device'):  # (a meta tensor goes to the operator's shapes)
            with pytest.raises(error, match=words):
                torch.ops.kadconv.group_norm_act_backward(x, x, 3, w, b, stat, stat, 1e-5, 'silu')
    for kw, words in ((dict(x=x[0]), 'N, C, H, W'), (dict(groups=5), 'divide'), (dict(groups=0), 'divide'), (dict(eps=-1.0), 'eps')):
        with pytest.raises(ValueError, match=words):
            call(ok, ok, **kw)


def _gn_args(**kw):
    a = _ext.GroupNormArgs()
    a.x = a.dy = a.out = a.mean = a.rstd = a.work = 256   # never dereferenced: rejected first
    a.n, a.c, a.groups, a.h, a.w, a.x_cs, a.dy_cs, a.eps = 2, 16, 4, 5, 5, 16, 16, 1e-5
    a.dtype = _ext.KAD_F16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize('kw', [dict(n=0), dict(c=0), dict(h=0), dict(w=-1), dict(groups=3), dict(groups=0), dict(dtype=5),
                                dict(param_dtype=_ext.KAD_BF16), dict(act=7), dict(eps=-1.0), dict(eps=float('nan')),
                                dict(x=None), dict(mean=None), dict(x_cs=8), dict(c=12, x_cs=24),
                                dict(n=70000), dict(h=1 << 20, w=1 << 20)], ids=str)
def test_group_norm_c_refusals(kw):
    lib = _ext.load()
    a = _gn_args(**kw)
    assert lib.kad_group_norm_fwd(ctypes.byref(a), None) == -1
    assert lib.kad_group_norm_bwd(ctypes.byref(a), None) == -1
    assert lib.kad_last_error()
    assert lib.kad_group_norm_fwd(None, None) == -1


def test_group_norm_c_refusals_of_one_direction():
    lib = _ext.load()
    for kw in (dict(dy=None), dict(dy_cs=8)):
        assert lib.kad_group_norm_bwd(ctypes.byref(_gn_args(**kw)), None) == -1
    assert lib.kad_group_norm_fwd(ctypes.byref(_gn_args(out=None)), None) == -1
    assert lib.kad_group_norm_work_elems(ctypes.byref(_gn_args(groups=3)), 0) == -1
    big = _gn_args(c=256, groups=32, h=200, w=200, x_cs=256, dy_cs=256, work=None)
    if lib.kad_group_norm_work_elems(ctypes.byref(big), 1):
        assert lib.kad_group_norm_bwd(ctypes.byref(big), None) == -1


def test_group_norm_groups_are_numbered_in_32_bits():
    lib = _ext.load()
    for backward in (0, 1):
        most = _gn_args(n=1 << 10, c=1 << 20, groups=1 << 20, h=1, w=1)
        assert lib.kad_group_norm_work_elems(ctypes.byref(most), backward) >= 0
        most.n += 1
        assert lib.kad_group_norm_work_elems(ctypes.byref(most), backward) == -1


def test_group_norm_small_maps_of_many_images_fit_a_grid():
    """More (image, set of groups) pairs than layers of a grid hold go to the kernels that take a batch by rows."""
    lib = _ext.load()
    few = _gn_args(n=65535, c=512, groups=64, h=2, w=2, x_cs=512, dy_cs=512)
    many = _gn_args(n=65535, c=1024, groups=128, h=2, w=2, x_cs=1024, dy_cs=1024)
    assert lib.kad_group_norm_work_elems(ctypes.byref(few), 0) == 0
    assert lib.kad_group_norm_work_elems(ctypes.byref(many), 0) > 0


def _table(host):
    n = host.numel() // ctypes.sizeof(_ext.AdamwChunk)
    return list((_ext.AdamwChunk * n).from_buffer_copy(bytes(host.numpy().tobytes())))


def test_adamw_chunks_cover_every_value_once():
    numels = [1, 255, 256, 257, 0, 4095, 4096, 4097, 20000, 3]
    params = [1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20, 6 << 20, 7 << 20, 8 << 20, 9 << 20, 10 << 20]
    grads = [p + (1 << 30) for p in params]
    grads[3] = 0   # no gradient: a place among the states, no chunk
    host, elems = _ext.adamw_chunks(params, grads, numels, 2)
    offset, want = 0, {}
    for p, g, n in zip(params, grads, numels):
        assert offset % _ext.ADAMW_SEG == 0
        for i in range(n if g else 0):
            want[p + 2 * i] = (g + 2 * i, offset + i)
        offset += -(-n // 256) * 256
    assert elems == offset
    got = {}
    for c in _table(host):
        assert 1 <= c.count <= 4096 and c.offset % 256 == 0 and c.offset + c.count <= elems
        for i in range(c.count):
            assert c.param + 2 * i not in got
            got[c.param + 2 * i] = (c.grad + 2 * i, c.offset + i)
    assert got == want


def test_adamw_chunks_of_one_tensor_past_32_bits():
    n = (1 << 32) + 5
    lib = _ext.load()
    one = [(ctypes.c_int64 * 1)(v) for v in (4096, 8192, n)]
    elems = ctypes.c_int64()
    assert lib.kad_adamw_chunks(*one, 1, 4, None, ctypes.byref(elems)) == -(-n // 4096)
    assert elems.value == -(-n // 256) * 256
    assert lib.kad_adamw_chunks(None, None, None, 1, 4, None, None) == -1
    assert lib.kad_adamw_chunks(*one, 1, 3, None, None) == -1
    assert lib.kad_adamw_chunks(*one, -1, 4, None, None) == -1
    one[2][0] = -1
    assert lib.kad_adamw_chunks(*one, 1, 4, None, None) == -1


def test_adamw_chunks_refuse_addresses_a_kernel_cannot_use():
    """A table is read by the kernel as it is: no null or misaligned address gets into one, and no count that runs over."""
    for params, grads, bytes_ in (([0], [4096], 4), ([4098], [8192], 4), ([4096], [8193], 2), ([4096, 2], [8192, 8196], 4)):
        with pytest.raises(RuntimeError, match='addresses'):
            _ext.adamw_chunks(params, grads, [5] * len(params), bytes_)
    # without a gradient or without values there is no chunk
    table, elems = _ext.adamw_chunks([0, 4096, 0], [0, 8192, 16], [5, 5, 0], 4)
    assert len(_table(table)) == 1 and elems == 512
    n = 3
    most = [(ctypes.c_int64 * n)(*[v] * n) for v in (4096, 0, 1 << 47)]
    assert _ext.load().kad_adamw_chunks(*most, 2, 4, None, None) == 0
    assert _ext.load().kad_adamw_chunks(*most, n, 4, None, None) == -1 and b'too many' in _ext.load().kad_last_error()


@pytest.mark.parametrize('kw', [dict(dtype=9), dict(state_bits=16), dict(chunks=None), dict(exp_avg=None), dict(step=0),
                                dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(lr=float('nan')),
                                dict(weight_decay=-1.0), dict(state_bits=8), dict(master=256, dtype=_ext.KAD_F32),
                                dict(nchunks=-1), dict(nchunks=1 << 31)], ids=str)
def test_adamw_c_refusals(kw):
    lib = _ext.load()
    a = _ext.AdamwArgs()
    a.chunks = a.exp_avg = a.exp_avg_sq = 256   # never dereferenced: rejected first
    a.lr, a.beta1, a.beta2, a.eps, a.weight_decay = 1e-3, 0.9, 0.999, 1e-8, 1e-2
    a.step, a.nchunks, a.dtype, a.state_bits = 1, 1, _ext.KAD_F16, 32
    for k, v in kw.items():
        setattr(a, k, v)
    assert lib.kad_adamw_step(ctypes.byref(a), None) == -1 and lib.kad_last_error()
    assert lib.kad_adamw_step(None, None) == -1
    assert lib.kad_adamw_hyper(ctypes.byref(a), None, None, None, None) == -1


def test_adamw_refusals():
    p = torch.zeros(4)
    with pytest.raises(ValueError, match='GPU'):
        kadconv.AdamWPlan([p], [p.clone()])
    with pytest.raises(ValueError, match='state_bits'):
        kadconv.AdamWPlan([p], [p.clone()], state_bits=4)
    with pytest.raises(ValueError, match='at least one'):
        kadconv.AdamWPlan([], [])
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-1.0),
               dict(state_bits=16), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            kadconv.AdamW([torch.nn.Parameter(p)], **kw)
    opt = kadconv.AdamW([torch.nn.Parameter(p)])
    assert opt.step() is None                      # no gradient: nothing to do
    q = torch.nn.Parameter(p.clone())
    q.grad = torch.ones(4)
    with pytest.raises(ValueError, match='GPU'):
        kadconv.AdamW([q]).step()


def test_adamw_refuses_another_optimizers_state():
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    other = torch.optim.AdamW([p], lr=0.5)
    other.step()
    opt = kadconv.AdamW([p], lr=1e-2)
    with pytest.raises(ValueError, match='another optimizer'):
        opt.load_state_dict(other.state_dict())
    assert opt.param_groups[0]['lr'] == 1e-2 and opt.param_groups[0]['step'] == 0 and not opt.state


def test_adamw_loads_a_group_without_parameters():
    p = torch.nn.Parameter(torch.zeros(4))
    for lr in (1e-2, torch.tensor(1e-2)):
        a, b = (kadconv.AdamW([dict(params=[]), dict(params=[p])], lr=v, capturable=True) for v in (lr, 1e-3))
        for opt in (a, b):
            opt.load_state_dict(a.state_dict())
            assert [float(group['lr']) for group in opt.param_groups] == [pytest.approx(1e-2)] * 2


@pytest.mark.parametrize('nchunks', [1 << 24, 1 << 40])
def test_adamw_c_refuses_more_blocks_than_a_grid_holds(nchunks):
    lib = _ext.load()
    a = _ext.AdamwArgs()
    a.chunks = a.exp_avg = a.exp_avg_sq = 256   # never dereferenced: rejected first
    a.beta1, a.beta2, a.step, a.nchunks, a.dtype, a.state_bits = 0.9, 0.99, 1, nchunks, _ext.KAD_F16, 32
    assert lib.kad_adamw_step(ctypes.byref(a), None) == -1 and b'too many chunks' in lib.kad_last_error()


STRUCTS = {'kad_group_norm_args': _ext.GroupNormArgs, 'kad_adamw_args': _ext.AdamwArgs, 'kad_adamw_chunk': _ext.AdamwChunk}


@pytest.mark.skipif(shutil.which('gcc') is None, reason='needs gcc')
def test_structs_match_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "kadconv_hip.h"', 'int main(void) {']
    expect = []
    for cname, cls in STRUCTS.items():
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        expect.append(ctypes.sizeof(cls))
        for field in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({cname}, {field[0]}));')
            expect.append(getattr(cls, field[0]).offset)
    lines += ['  printf("%zu\\n%d\\n", sizeof(kad_adamw_scalars), KAD_ADAMW_SEG);', '  return 0;', '}']
    expect += [4 * _ext.ADAMW_SCALARS, _ext.ADAMW_SEG]
    src, exe = tmp_path / 'layout.c', tmp_path / 'layout'
    src.write_text('\n'.join(lines) + '\n')
    subprocess.run(['gcc', '-std=c11', '-I', os.path.join(ROOT, 'include'), str(src), '-o', str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == expect


@pytest.mark.parametrize('name', ['exp_avg', 'exp_avg_sq', 'master'])
def test_adamw_c_alignment(name):
    lib = _ext.load()
    a = _ext.AdamwArgs()
    a.chunks = a.exp_avg = a.exp_avg_sq = a.master = 256   # never dereferenced: rejected first
    a.beta1, a.beta2, a.step, a.nchunks, a.dtype, a.state_bits = 0.9, 0.99, 1, 1, _ext.KAD_F16, 32
    setattr(a, name, 264)
    assert lib.kad_adamw_step(ctypes.byref(a), None) == -1 and b'16 bytes' in lib.kad_last_error()


def test_group_norm_c_refuses_far_pixels():
    lib = _ext.load()
    for kw in (dict(x_cs=(1 << 20) + 8), dict(dy_cs=(1 << 20) + 8)):
        assert lib.kad_group_norm_bwd(ctypes.byref(_gn_args(**kw)), None) == -1


def test_binding_is_built_again_for_another_torch(tmp_path, monkeypatch):
    """The object of the binding is used again for the same sources, torch, Python and command, and for no other."""
    spec = importlib.util.spec_from_file_location('kad_build', os.path.join(ROOT, 'kad-conv_amd', 'build.py'))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    ran = []

    def run(cmd, **_):
        ran.append(cmd)
        open(cmd[cmd.index('-o') + 1], 'w').close()
        return subprocess.CompletedProcess(cmd, 0, '', '')

    monkeypatch.setattr(build, 'OBJ', str(tmp_path))
    monkeypatch.setattr(build.subprocess, 'run', run)

    def compiles(n):
        assert build._compile_native(False) == (str(tmp_path / 'kad_torch.cpp.o'), None)
        assert len(ran) == n
    compiles(1)
    compiles(1)
    monkeypatch.setattr(torch, '__version__', '9.0')
    compiles(2)
    compiles(2)
    monkeypatch.setattr(torch.version, 'hip', '9.0')
    compiles(3)
    monkeypatch.setattr(build, 'INCLUDE', str(tmp_path / '..' / 'include'))
    monkeypatch.setattr(build, '_deps', lambda: [])
    compiles(4)
    compiles(4)
