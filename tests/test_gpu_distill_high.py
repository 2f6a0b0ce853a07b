"""distill_loss at temperatures above 8, which are computed in 64 bits: the layouts, types, masks and lengths of the other form."""
import pytest
import torch

import kadconv
from kadconv import ops
from tests.test_gpu_distill import DEV, DTYPES, F16, F32, INF, NAN, check, make

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize('shape', [(1, 1, 1), (40, 3, 2), (33, 8, 8), (17, 16, 16), (300, 256, 64), (301, 257, 64), (65, 200, 65), (9, 4096, 256),
                                   (7, 4097, 20), (6, 4000, 257), (3, 50, 1024), (2, 33001, 256), (1, 150001, 1000), (40000, 10, 3),
                                   (8200, 300, 5), (2100, 5000, 2)], ids=lambda s: 'x'.join(map(str, s)))
def test_loss_and_gradient(shape, dtype):
    rows, v, k = shape
    check(*make(rows, v, k, dtype, seed=v, index=torch.int32 if v % 2 else torch.int64), 20.0)


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
        z, t = wide[..., 3:3 + v].permute(0, 3, 1, 2), t.contiguous()
    check(z, t, i, 12.0, dim=1)


def test_rows_in_other_places():
    z, t, i = make(12, 40, 6, F32, 6)
    check(z[::2], t[::2], i[::2], 12.0)
    check(z, t.t().contiguous().t(), i.flip(1).t().contiguous().t().flip(1), 12.0)
    check(z.view(2, 6, 40).transpose(0, 1), t.view(2, 6, 6).transpose(0, 1), i.view(2, 6, 6).transpose(0, 1), 12.0)
    check(z, t[:1].expand(12, 6), i[:1].expand(12, 6), 12.0)
    check(z, t.bfloat16(), i, 12.0)


@DTYPES
@pytest.mark.parametrize('v', [12, 700, 5000])
def test_entries_that_do_not_count_and_that_come_again(v, dtype):
    z, t, i = make(8, v, 6, dtype, 9, holes=False)
    i[0] = -1
    i[1, 0], i[1, 1], i[1, 2] = v, -7, (1 << 32) + 3
    t[2] = -INF
    t[3, 1:] = -INF
    i[5] = i[5, 0]
    i[6, 3:5] = i[6, 2]
    check(z, t, i, 30.0)
    none = torch.full_like(i, -1)
    zs = z.clone().requires_grad_(True)
    for reduction in ('none', 'sum', 'mean'):
        loss = kadconv.distill_loss(zs, t, none, 30.0, reduction)
        assert not loss.any() and not torch.autograd.grad(loss.sum(), zs)[0].any()


@pytest.mark.parametrize('v', [5, 12, 700, 5000])
def test_not_finite_stays_in_its_row(v):
    z, t, i = make(8, v, 4, F32, 13, holes=False)
    z[1, v - 1] = NAN
    z[2] = -INF
    t[3, 1] = NAN
    z[4, 0] = INF
    i[5] = -1
    z[5] = NAN
    z[6, i[6, 2]] = -INF
    zs = z.requires_grad_(True)
    loss = kadconv.distill_loss(zs, t, i, 9.0, 'none')
    dz, = torch.autograd.grad(loss, zs, torch.ones_like(loss))
    assert torch.isfinite(loss[[0, 7]]).all() and torch.isfinite(dz[[0, 7]]).all()
    assert torch.isnan(loss[1:5]).all() and torch.isnan(dz[1:5]).any(1).all() and torch.isnan(dz[2:4]).all()
    assert loss[5] == 0 and not dz[5].any()
    assert loss[6] == INF and torch.isfinite(dz[6]).all() and dz[6, i[6, 2]] < 0


@pytest.mark.parametrize('shape', [(300, 60, 30), (50, 3000, 64), (3, 40000, 200)], ids=['short', 'wave', 'block'])
def test_captured_and_repeated(shape):
    """Forward and backward captured into one graph; every replay is checked, with eager work between."""
    g = torch.tensor(0.5, device=DEV)

    def both(z, t, i):
        loss, stats, share = ops.distill_loss_forward(z, t, i, 50.0, 'mean', -1)
        return loss, ops.distill_loss_backward(g, z, t, i, stats, share, 50.0, 'mean', -1)

    state = make(*shape, F16, 17)
    first = both(*state)
    assert all(torch.equal(a, b) for a, b in zip(first, both(*state)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(*state)
    for n in range(3):
        new = make(*shape, F16, 30 + n)
        for a, b in zip(state, new):
            a.copy_(b)
        graph.replay()
        want = both(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), n


def test_beside_the_other_form():
    """At the temperature where the form changes both are the same loss: 32-bit sums are off by some 1e-4 of it there."""
    z, t, i = make(50, 100, 20, F32, 2)
    a, b = (kadconv.distill_loss(z, t, i, temperature) for temperature in (8.0, 8.000001))
    torch.testing.assert_close(a, b, rtol=1e-4, atol=0)
