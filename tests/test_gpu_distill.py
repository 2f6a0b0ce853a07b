"""distill_loss on the GPU, with its gradient, against the formulas in 64 bits."""
import pytest
import torch

import kadconv
from kadconv import ops
from tests._distill_ref import EPS32, reference
from tests._norm_ref import assert_within

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = pytest.mark.parametrize('dtype', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
DEV, INF, NAN = 'cuda', float('inf'), float('nan')


def make(rows, v, k, dtype, seed=0, index=torch.int64, holes=True):
    """Logits near a teacher's, and that one's k best; some entries left out, some rows without any."""
    g = torch.Generator().manual_seed(seed)
    teacher = 2 * torch.randn(rows, v, generator=g)
    z = (0.7 * teacher + torch.randn(rows, v, generator=g)).to(dtype)
    top = torch.topk(teacher, min(k, v), dim=1)
    t, i = top.values.to(dtype), top.indices
    if k > v:  # more entries than classes: some come again
        t, i = t.repeat(1, -(-k // v))[:, :k].contiguous(), i.repeat(1, -(-k // v))[:, :k].contiguous()
    if holes and rows > 1:
        out = torch.rand(rows, k, generator=g) < 0.1
        out |= torch.rand(rows, 1, generator=g) < 0.15
        i = torch.where(out, -1, i)
    return z.to(DEV), t.to(DEV), i.to(index).to(DEV)


def rows_of(x, dim):
    return x.movedim(dim, -1).reshape(-1, x.shape[dim])


def check(z, t, i, temperature=2.0, dim=-1, seed=5):
    zs = z.detach().requires_grad_(True)
    n = rows_of(z, dim).shape[0]
    g = torch.rand(n, generator=torch.Generator().manual_seed(seed)).to(DEV)
    ref = reference(rows_of(z, dim), rows_of(t, dim), rows_of(i, dim), temperature, g, z.dtype)
    loss = kadconv.distill_loss(zs, t, i, temperature, 'none', dim)
    shape = list(z.shape)
    shape.pop(dim)
    assert loss.dtype == F32 and list(loss.shape) == shape
    with torch.no_grad():
        assert torch.equal(kadconv.distill_loss(zs, t, i, temperature, 'none', dim), loss)
    assert_within(loss.reshape(-1), ref['loss'], ref['tol_loss'], 'loss')
    dz, = torch.autograd.grad(loss, zs, g.view(shape))
    assert dz.dtype == z.dtype and dz.shape == z.shape and dz.movedim(dim, -1).is_contiguous()
    assert_within(rows_of(dz, dim), ref['dz'], ref['tol_dz'], 'dz')
    for reduction in ('sum', 'mean'):
        live = max(1, int(ref['live'].sum())) if reduction == 'mean' else 1
        ones = torch.full((n,), 3.0 / live, dtype=torch.float64)
        ref2 = reference(rows_of(z, dim), rows_of(t, dim), rows_of(i, dim), temperature, ones, z.dtype)
        loss = kadconv.distill_loss(zs, t, i, temperature, reduction, dim)
        want = ref['loss'].sum() / live
        tol = (ref['tol_loss'].sum() + (64 + n / 2048) * EPS32 * ref['loss'].abs().sum()) / live + 1e-36
        assert loss.shape == () and abs(loss.double().cpu() - want) <= tol, (loss.item(), want.item(), tol.item())
        dz, = torch.autograd.grad(loss, zs, torch.tensor(3.0, device=DEV))
        # the gradient's factor is a product of three, one of them rounded
        assert_within(rows_of(dz, dim), ref2['dz'], ref2['tol_dz'] + 4 * EPS32 * ref2['dz'].abs(), 'dz of ' + reduction)


SHAPES = [  # rows, classes, entries: values a lane, a wave's rows, a block's, parts of rows; their borders
    (1, 1, 1), (3, 2, 1), (40, 3, 2), (7, 5, 5), (300, 7, 3), (33, 8, 8), (65, 9, 4), (129, 16, 16), (90, 17, 2), (400, 20, 4),
    (50, 64, 10), (21, 80, 80), (5, 100, 7), (9, 511, 64), (6, 513, 1), (4, 1000, 300), (5, 1023, 33), (6, 1024, 256), (5, 1025, 16),
    (4, 1027, 100), (3, 2000, 1024), (70, 4097, 20), (1, 8192, 50), (3, 8203, 64), (600, 8200, 9), (2, 33001, 256), (1, 150001, 1000),
    (2100, 1030, 5), (5000, 10, 3), (3, 4, 40), (2, 300, 900)]


@DTYPES
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(map(str, s)))
def test_loss_and_gradient(shape, dtype):
    rows, v, k = shape
    check(*make(rows, v, k, dtype, seed=v, index=torch.int32 if v % 2 else torch.int64))


@DTYPES
@pytest.mark.parametrize('shape', [(1024, 1025, 3), (1025, 2047, 64), (1101, 3000, 256), (1030, 8192, 20), (1027, 1500, 257),
                                   (1024, 8193, 30), (1500, 513, 12), (1026, 1024, 40), (1024, 600, 900)], ids=lambda s: 'x'.join(map(str, s)))
def test_many_rows(shape, dtype):
    """Rows of a wave each, and at the borders of that form, with rows that are unlike each other side by side."""
    rows, v, k = shape
    z, t, i = make(rows, v, k, dtype, seed=v)
    i[0] = -1
    i[1] = i[1].max()
    t[2] = -INF
    i[5, k // 2:] = i[5, 0]
    i[-1, 1:] = v
    z[6, ::3] = torch.where(torch.isin(torch.arange(0, v, 3, device=DEV), i[6]), z[6, ::3], -INF)
    check(z, t, i, 1.5)
    bad = z.clone()
    bad[7, 11], bad[8, -1], bad[9] = NAN, INF, -INF
    some = [r for r in range(rows) if r not in (7, 8, 9)]
    for zs in (z, bad):
        zs.requires_grad_(True)
        loss = kadconv.distill_loss(zs, t, i, 1.5, 'none')
        dz, = torch.autograd.grad(loss, zs, torch.ones_like(loss))
        if zs is z:
            want, want_dz = loss.detach(), dz
    assert torch.equal(loss[some], want[some]) and torch.equal(dz[some], want_dz[some])
    counts = ((i[7:10] >= 0) & (i[7:10] < v)).any(1)
    assert torch.equal(loss[7:10].isnan(), counts) and torch.equal(dz[7:10].isnan().all(1), counts)


@DTYPES
@pytest.mark.parametrize('layout', ['cl', 'nchw', 'slice'])
@pytest.mark.parametrize('shape', [(2, 20, 5, 7, 4), (1, 16, 20, 20, 16), (3, 9, 1, 4, 2), (2, 1100, 3, 2, 10), (2, 6, 4, 1, 3)],
                         ids=lambda s: 'x'.join(map(str, s)))
def test_maps(shape, layout, dtype):
    n, v, h, w, k = shape
    z, t, i = (a.view(n, h, w, -1).permute(0, 3, 1, 2) for a in make(n * h * w, v, k, dtype, 3))
    if layout == 'nchw':
        z, t, i = z.contiguous(), t.contiguous(), i.contiguous()
    if layout == 'slice':
        wide = torch.full((n, h, w, v + 5), 7.0, dtype=dtype, device=DEV)
        wide[..., 3:3 + v] = z.permute(0, 2, 3, 1)
        z = wide[..., 3:3 + v].permute(0, 3, 1, 2)
        t = t.contiguous()
    check(z, t, i, dim=1)


@DTYPES
def test_rows_in_other_places(dtype):
    z, t, i = make(12, 40, 6, dtype, 6)
    wide = torch.zeros(12, 51, dtype=dtype, device=DEV)
    wide[:, 3:43] = z
    check(wide[:, 3:43], t, i)
    check(z[::2], t[::2], i[::2])
    check(z, t.t().contiguous().t(), i.flip(1).t().contiguous().t().flip(1))
    check(z.view(2, 3, 2, 40), t.view(2, 3, 2, 6), i.view(2, 3, 2, 6))
    check(z.view(2, 6, 40).transpose(0, 1), t.view(2, 6, 6).transpose(0, 1), i.view(2, 6, 6).transpose(0, 1))
    check(z, t[:1].expand(12, 6), i[:1].expand(12, 6))
    check(z[3], t[3], i[3])
    check(z[:, ::2], t, (i // 2).clamp(min=-1))


def test_types_of_the_teacher():
    z, t, i = make(30, 50, 8, F32, 7)
    for zt in (F32, F16, BF16):
        for tt in (F32, F16, BF16):
            check(z.to(zt), t.to(tt), i)


def test_temperatures():
    for v in (30, 3000):
        z, t, i = make(9, v, 8, F32, 8)
        for temperature in (0.05, 0.7, 1.0, 3.0, 20.0):
            check(z, t, i, temperature)


@DTYPES
@pytest.mark.parametrize('v', [12, 700, 3000, 20000])
def test_entries_that_do_not_count(v, dtype):
    """Indexes outside, far outside and of -infinity logits, in every form; rows left without any."""
    z, t, i = make(6, v, 6, dtype, 9, holes=False)
    i[0] = -1
    i[1, 0], i[1, 1], i[1, 2] = v, -7, (1 << 32) + 3
    t[2] = -INF
    t[3, 1:] = -INF
    i[4, :5] = -(1 << 40)
    check(z, t, i)
    ref = kadconv.distill_loss(z, t, i, reduction='none')
    assert ref[0] == 0 and ref[2] == 0 and (ref[[1, 3, 4, 5]] != 0).all()
    none = torch.full_like(i, -1)
    zs = z.clone().requires_grad_(True)
    for reduction in ('none', 'sum', 'mean'):
        loss = kadconv.distill_loss(zs, t, none, reduction=reduction)
        assert not loss.any()
        assert not torch.autograd.grad(loss.sum(), zs)[0].any()


@DTYPES
@pytest.mark.parametrize('v', [12, 700, 3000, 20000])
def test_an_index_that_comes_again(v, dtype):
    z, t, i = make(4, v, 12, dtype, 10, holes=False) if v >= 12 else make(4, 12, 12, dtype, 10, holes=False)
    i[0] = i[0, 0]
    i[1, 3] = i[1, 0]
    i[2, 4:9] = i[2, 4:5]
    check(z, t, i)


@pytest.mark.parametrize('v', [12, 700, 3000, 20000])
def test_masked_logits(v):
    """Classes of -infinity: no weight and no gradient; of the type's lowest value likewise; all of the lowest value:
    all alike.  An entry at a class without weight: an infinite loss, and a finite gradient."""
    for dtype, lowest in ((F32, -INF), (F16, -INF), (F32, torch.finfo(F32).min), (BF16, torch.finfo(BF16).min)):
        z, t, i = make(5, v, 4, dtype, 11, holes=False)
        away = torch.ones(5, v, dtype=torch.bool, device=DEV).scatter_(1, i, False)
        away[:, ::3] = False
        z[away] = lowest
        if lowest == -INF:
            check(z, t, i, 1.0)
        zs = z.clone().requires_grad_(True)
        dz, = torch.autograd.grad(kadconv.distill_loss(zs, t, i, 1.0), zs)
        assert not dz[away].any() and torch.isfinite(dz).all()
    z = torch.full((2, v), torch.finfo(F32).min, device=DEV).requires_grad_(True)
    dz, = torch.autograd.grad(kadconv.distill_loss(z, t[:2].float(), i[:2], 1.0, 'sum'), z)
    others = torch.ones(2, v, dtype=torch.bool, device=DEV).scatter_(1, i[:2], False)
    torch.testing.assert_close(dz[others], torch.full_like(dz[others], 1 / v), rtol=(64 + v / 256) * EPS32, atol=0)
    z, t, i = make(3, v, 4, F32, 12, holes=False)
    z[1, i[1, 2]] = -INF
    zs = z.requires_grad_(True)
    loss = kadconv.distill_loss(zs, t, i, reduction='none')
    dz, = torch.autograd.grad(loss, zs, torch.ones_like(loss))
    assert loss[1] == INF and torch.isfinite(loss[[0, 2]]).all() and torch.isfinite(dz).all() and dz[1, i[1, 2]] < 0


@pytest.mark.parametrize('v', [5, 12, 700, 3000, 20000])
def test_not_finite_stays_in_its_row(v):
    z, t, i = make(6, v, 4, F32, 13, holes=False)
    z[1, v - 1] = NAN
    z[2] = -INF
    t[3, 1] = NAN
    z[4, 0] = INF
    i[5] = -1
    z[5] = NAN
    zs = z.requires_grad_(True)
    loss = kadconv.distill_loss(zs, t, i, reduction='none')
    dz, = torch.autograd.grad(loss, zs, torch.ones_like(loss))
    assert torch.isfinite(loss[0]) and torch.isfinite(dz[0]).all()
    for r in (1, 2, 3, 4):
        assert torch.isnan(loss[r]) and torch.isnan(dz[r]).any(), r
    for r in (2, 3):
        assert torch.isnan(dz[r]).all(), r
    assert loss[5] == 0 and not dz[5].any()  # no entries: whatever the logits are


def test_empty():
    for shape, dim in (((0, 8), -1), ((3, 0, 8), -1), ((0, 8, 4, 4), 1), ((2, 8, 0, 4), 1)):
        z = torch.empty(shape, device=DEV, requires_grad=True)
        k = list(shape)
        k[dim] = 3
        t, i = torch.empty(k, device=DEV), torch.empty(k, dtype=torch.int64, device=DEV)
        for reduction in ('none', 'sum', 'mean'):
            loss = kadconv.distill_loss(z, t, i, reduction=reduction, dim=dim)
            assert not loss.any()
            assert torch.autograd.grad(loss.sum(), z)[0].shape == z.shape


@pytest.mark.parametrize('v', [9, 4000])
def test_gradient_against_differences(v):
    """(f(z + h d) - f(z - h d)) / 2h of the 64-bit loss equals <dz, d>, off by its third derivative times h^2."""
    z, t, i = make(5, v, 4, F32, 14, holes=False)
    i[2, 1] = i[2, 0]
    zs = z.clone().requires_grad_(True)
    dz, = torch.autograd.grad(kadconv.distill_loss(zs, t, i, 2.0, 'sum'), zs)
    d = torch.randn(z.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    h = 1e-4
    f = [reference(z.double().cpu() + s * d, t, i, 2.0)['loss'].sum() for s in (h, -h)]
    want, got = ((f[0] - f[1]) / (2 * h)).item(), (dz.double().cpu() * d).sum().item()
    assert abs(got - want) <= 2e-5 * (dz.double().cpu() * d).abs().sum().item()


@pytest.mark.parametrize('shape', [(3000, 60, 30), (50, 5000, 64), (3, 40000, 200)], ids=['small', 'large', 'parts'])
def test_same_result_every_time(shape):
    z, t, i = make(*shape, BF16, 15)
    i[:, 1:5] = i[:, 0:1]
    zs = z.requires_grad_(True)
    first = None
    for _ in range(3):
        loss = kadconv.distill_loss(zs, t, i)
        got = (loss, *torch.autograd.grad(loss, zs))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_other_stream():
    z, t, i = make(300, 64, 5, F16, 16)
    want = kadconv.distill_loss(z, t, i)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kadconv.distill_loss(z * 1, t * 1, i * 1)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize('shape', [(300, 60, 30), (50, 5000, 64), (3, 40000, 200)], ids=['small', 'large', 'parts'])
@pytest.mark.parametrize('reduction', ['none', 'mean'])
def test_captured(shape, reduction):
    """Forward and backward captured into one graph; every replay is checked, with eager work between."""
    g = torch.full((shape[0],) if reduction == 'none' else (), 0.5, device=DEV)

    def both(z, t, i):
        loss, stats, share = ops.distill_loss_forward(z, t, i, 2.0, reduction, -1)
        return loss, ops.distill_loss_backward(g, z, t, i, stats, share, 2.0, reduction, -1)

    state = make(*shape, F16, 17)
    both(*state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(*state)
    for n in range(4):
        new = make(*shape, F16, 30 + n)
        for a, b in zip(state, new):
            a.copy_(b)
        graph.replay()
        want = both(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), n


def test_more_than_2_31_values():
    """Offsets that pass 32 bits: the last rows' results equal those of these rows alone."""
    rows, v = 66_000, 33_000
    free, _ = torch.cuda.mem_get_info()
    if free < 30 << 30:
        pytest.skip('needs 30 GiB of GPU memory')
    assert rows * v > 2 ** 31
    z = torch.empty(rows, v, dtype=F16, device=DEV).normal_()
    t = torch.empty(rows, 4, dtype=F16, device=DEV).normal_()
    i = torch.randint(0, v, (rows, 4), device=DEV)
    g = torch.ones(rows, device=DEV)
    last = slice(rows - 2048, rows)
    loss, stats, share = ops.distill_loss_forward(z, t, i, 1.0, 'none', -1)
    dz = ops.distill_loss_backward(g, z, t, i, stats, share, 1.0, 'none', -1)
    la, sa, ha = ops.distill_loss_forward(z[last], t[last], i[last], 1.0, 'none', -1)
    assert torch.equal(loss[last], la)
    assert torch.equal(dz[last], ops.distill_loss_backward(g[last], z[last], t[last], i[last], sa, ha, 1.0, 'none', -1))


def test_compiled():
    for dim, shape in ((-1, None), (1, (2, 5, 4))):
        z, t, i = make(40, 12, 3, F32, 18)
        if shape:
            z, t, i = (a.view(*shape, -1).permute(0, 3, 1, 2) for a in (z, t, i))
        for reduction in ('none', 'mean'):
            def f(z):
                return kadconv.distill_loss(z, t, i, 2.0, reduction, dim).sum()
            zs = z.clone().requires_grad_(True)
            want = torch.autograd.grad(f(zs), zs)[0]
            got = torch.autograd.grad(torch.compile(f, fullgraph=True, backend='aot_eager')(zs), zs)[0]
            assert torch.equal(want, got)


def test_refusals():
    z, t, i = make(3, 8, 2, F32)
    with pytest.raises(TypeError):
        kadconv.distill_loss(z.double(), t, i)
    with pytest.raises(TypeError, match='int32'):
        kadconv.distill_loss(z, t, i.short())
    with pytest.raises(ValueError, match='one device'):
        kadconv.distill_loss(z, t.cpu(), i)
    with pytest.raises(ValueError, match='reduction'):
        kadconv.distill_loss(z, t, i, reduction='batchmean')
    with pytest.raises(ValueError, match='temperature'):
        kadconv.distill_loss(z, t, i, temperature=1e-60)
    with pytest.raises(ValueError, match='1024'):
        kadconv.distill_loss(z, t[:, :1].expand(3, 1025), i[:, :1].expand(3, 1025))
    loss, stats, share = ops.distill_loss_forward(z, t, i, 1.0, 'none', -1)
    with pytest.raises(ValueError, match='stats and share'):
        ops.distill_loss_backward(loss, z, t, i, stats[:2], share, 1.0, 'none', -1)
    with pytest.raises(ValueError, match='dloss'):
        ops.distill_loss_backward(loss[:2], z, t, i, stats, share, 1.0, 'none', -1)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        zs = z.clone().requires_grad_(True)
        g, = torch.autograd.grad(kadconv.distill_loss(zs, t, i), zs, create_graph=True)
        g.sum().backward()
    ts = t.clone().requires_grad_(True)
    assert not kadconv.distill_loss(z, ts, i).requires_grad  # the teacher is a constant
