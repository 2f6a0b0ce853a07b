"""layer_norm on the GPU, forward and gradients, against the formulas in 64 bits: a row is the only group of an image of
one pixel, so group norm's reference and its bounds hold."""
import pytest
import torch

import kadconv
from kadconv import ops
from tests._norm_ref import assert_within, reference

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = pytest.mark.parametrize('dtype', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
DEV = 'cuda'


def rows_of(x, dim):
    return x.movedim(dim, -1).reshape(-1, x.shape[dim])


def make(rows, c, dtype, seed=0, loc=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, c, generator=g) + 0.3 * torch.randn(1, c, generator=g) + loc).to(dtype).to(DEV)


def make_map(n, c, h, w, dtype, seed=0, layout='cl'):
    v = make(n * h * w, c, dtype, seed).view(n, h, w, c)
    if layout == 'nchw':
        return v.permute(0, 3, 1, 2).contiguous()
    if layout == 'slice':  # channels 3 .. 3 + c of a wider map
        wide = torch.full((n, h, w, c + 8), 7.0, dtype=dtype, device=DEV)
        wide[..., 3:3 + c] = v
        return wide[..., 3:3 + c].permute(0, 3, 1, 2)
    return v.permute(0, 3, 1, 2)


def params(c, dtype=F32, seed=1):
    g = torch.Generator().manual_seed(seed)
    w = (1 + 0.3 * torch.randn(c, generator=g)).to(dtype).to(DEV)
    return w, (0.2 * torch.randn(c, generator=g)).to(dtype).to(DEV)


def expected(x, w, b, dy=None, dim=-1, eps=1e-5):
    r = rows_of(x.detach(), dim)[:, :, None, None]
    return reference(r, 1, w, b, eps, None, None if dy is None else rows_of(dy, dim)[:, :, None, None])


def close(got, ref, name, dim):
    assert_within(rows_of(got, dim)[:, :, None, None], ref[name], ref['tol_' + name], name)


def check(x, w, b, dy, dim=-1, eps=1e-5):
    ref = expected(x, w, b, dy, dim, eps)
    xs = x.detach().requires_grad_(True)
    ws = None if w is None else w.detach().requires_grad_(True)
    bs = None if b is None else b.detach().requires_grad_(True)
    with torch.no_grad():
        y0 = kadconv.layer_norm(xs, ws, bs, eps, dim)
    y = kadconv.layer_norm(xs, ws, bs, eps, dim)
    assert y.dtype == x.dtype and y.shape == x.shape and y.movedim(dim, -1).is_contiguous()
    assert torch.equal(y, y0)
    close(y, ref, 'y', dim)
    grads = iter(torch.autograd.grad(y, [t for t in (xs, ws, bs) if t is not None], dy))
    dx = next(grads)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    close(dx, ref, 'dx', dim)
    for name, p in (('dw', w), ('db', b)):
        if p is not None:
            got = next(grads)
            assert got.dtype == p.dtype and got.shape == p.shape
            assert_within(got, ref[name], ref['tol_' + name] + torch.finfo(p.dtype).eps / 2 * ref[name].abs() + 1e-30, name)


SHAPES = [  # rows, c: a thread's, a wave's and a block's rows, their borders, and rows shorter than a vector
    (1, 1), (5, 2), (3, 3), (9, 5), (4, 7), (1, 8), (300, 9), (7, 15), (1, 16), (33, 64), (1, 86), (129, 86), (65, 127), (2, 128),
    (50, 129), (400, 256), (31, 511), (17, 513), (9, 1000), (6, 1024), (5, 1025), (3, 2047), (4, 2051), (3, 4096), (2, 4099),
    (2, 8191), (3, 8192), (1, 8200), (2, 16383), (2, 16384), (2500, 40), (1100, 768), (2100, 2048), (530, 4104)]


@DTYPES
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(map(str, s)))
def test_forward_and_gradients(shape, dtype):
    rows, c = shape
    check(make(rows, c, dtype, seed=c), *params(c), make(rows, c, dtype, seed=c + 1))


@DTYPES
@pytest.mark.parametrize('layout', ['cl', 'nchw', 'slice'])
@pytest.mark.parametrize('shape', [(2, 48, 13, 17), (1, 86, 9, 5), (3, 5, 4, 1), (1, 64, 20, 20), (2, 1, 3, 3), (2, 130, 1, 1)],
                         ids=lambda s: 'x'.join(map(str, s)))
def test_maps(shape, layout, dtype):
    check(make_map(*shape, dtype, 3, layout), *params(shape[1]), make_map(*shape, dtype, 4, layout), dim=1)
    check(make_map(*shape, dtype, 3), *params(shape[1]), make_map(*shape, dtype, 4, layout), dim=-3)


@DTYPES
def test_rows_in_other_places(dtype):
    """Slices along the rows, odd beginnings, more and fewer axes, transposed and expanded tensors."""
    wt, bs = params(40)
    dy = make(6, 40, dtype, 5)
    for off in (0, 1, 3):
        wide = make(6, 51, dtype, 6)
        check(wide[:, off:off + 40], wt, bs, dy)
    check(make(12, 40, dtype, 6)[::2], wt, bs, dy)
    check(make(40, 6, dtype, 7).t(), wt, bs, dy)
    check(make(1, 40, dtype, 8).expand(6, 40), wt, bs, dy)
    check(make(24, 40, dtype, 9).view(2, 3, 4, 40)[:, :, ::2], wt, bs, make(12, 40, dtype, 10).view(2, 3, 2, 40))
    check(make(24, 40, dtype, 9).view(2, 3, 4, 40).transpose(0, 2), wt, bs, make(24, 40, dtype, 10).view(4, 3, 2, 40))
    check(make(1, 40, dtype, 11)[0], wt, bs, make(1, 40, dtype, 12)[0])
    flat = make(1, 6 * 40 + 1, dtype, 13)[0]
    check(flat[1:].view(6, 40), wt, bs, dy)
    check(make(6, 40, dtype, 6), wt, bs, make(1, 1, dtype, 14).expand(6, 40))
    odd = make(1, 41, F32, 15)[0]  # parameters that begin anywhere
    check(make(6, 40, dtype, 6), odd[1:], bs, dy)
    check(make(6, 40, dtype, 6), make(1, 80, F32, 16)[0][::2], bs, dy)


@DTYPES
def test_parameters(dtype):
    for rows, c in ((6, 24), (3, 1500)):
        x, dy = make(rows, c, dtype, 5), make(rows, c, dtype, 6)
        for pdt in {F32, dtype}:
            wt, bs = params(c, pdt)
            for pw, pb in ((wt, bs), (wt, None), (None, bs), (None, None)):
                check(x, pw, pb, dy)


def test_mean_far_from_zero():
    """Values whose spread is a thousandth of their mean, and an outlier."""
    for c in (64, 1000, 5000):
        x = make(5, c, F32, 7, loc=1000.0)
        check(x, *params(c), make(5, c, F32, 8))
        x = make(5, c, F32, 7)
        x[:, 0] = 3000.0
        check(x, *params(c), make(5, c, F32, 8))


def test_constant_row():
    """No spread at all: y is the bias, and the gradient finite; without eps it is not (0 / 0)."""
    x = torch.full((3, 48), 3.0, device=DEV)
    check(x, *params(48), make(3, 48, F32, 9))
    assert torch.isnan(kadconv.layer_norm(x, eps=0.0)).all()


@DTYPES
def test_large_and_small_values(dtype):
    """The largest 16-bit values, and spreads far under eps."""
    big = make(3, 256, dtype, 20) * (16000.0 if dtype != F32 else 1e15)
    check(big, *params(256), make(3, 256, dtype, 21))
    tiny = make(3, 256, F32, 22) * 1e-4
    check(tiny.to(dtype), *params(256), make(3, 256, dtype, 23), eps=1e-3)


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
@pytest.mark.parametrize('c', [5, 86, 700, 9000])
def test_not_finite_stays_in_its_row(bad, c):
    x = make(9, c, F16, 11)
    x[4, c - 1] = bad
    wt, bs = params(c)
    xs, ws = x.requires_grad_(True), wt.requires_grad_(True)
    y = kadconv.layer_norm(xs, ws, bs)
    dx, dw = torch.autograd.grad(y, (xs, ws), torch.ones_like(y))
    for t in (y, dx):
        assert torch.isnan(t[4]).all() and torch.isfinite(t[:4]).all() and torch.isfinite(t[5:]).all()
    assert torch.isnan(dw).all()


def test_a_row_does_not_depend_on_the_others():
    """The same row gives the same bits, whichever rows are around it."""
    x, (wt, bs) = make(700, 96, F32, 12), params(96)
    y = kadconv.layer_norm(x, wt, bs)
    for part in (slice(0, 1), slice(699, 700), slice(100, 333)):
        assert torch.equal(kadconv.layer_norm(x[part], wt, bs), y[part])


def test_empty():
    wt, bs = params(8)
    for shape, dim in (((0, 8), -1), ((3, 0, 8), -1), ((0, 8, 4, 4), 1), ((2, 8, 0, 4), 1)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        wr, br = wt.clone().requires_grad_(True), bs.clone().requires_grad_(True)
        y = kadconv.layer_norm(x, wr, br, dim=dim)
        assert y.shape == x.shape
        dx, dw, db = torch.autograd.grad(y, (x, wr, br), torch.empty_like(y))
        assert dx.shape == x.shape and not dw.any() and not db.any()


def test_gradient_of_some_inputs():
    x, (wt, bs) = make(20, 24, F32, 12), params(24)
    ref = expected(x, wt, bs, torch.ones_like(x))
    xs, ws, bb = x.clone().requires_grad_(True), wt.clone().requires_grad_(True), bs.clone().requires_grad_(True)
    kadconv.layer_norm(xs, wt, bs).sum().backward()
    close(xs.grad, ref, 'dx', -1)
    kadconv.layer_norm(x, ws, bs).sum().backward()
    assert_within(ws.grad, ref['dw'], ref['tol_dw'], 'dw')
    kadconv.layer_norm(x, wt, bb).sum().backward()
    assert_within(bb.grad, ref['db'], ref['tol_db'], 'db')


def test_gradient_against_differences():
    """(f(x + t d) - f(x - t d)) / 2t of the 64-bit forward equals <dx, d>, off by its third derivative times t^2."""
    x, (wt, bs), dy = make(7, 12, F32, 13), params(12), make(7, 12, F32, 14)
    leaves = [t.clone().requires_grad_(True) for t in (x, wt, bs)]
    grads = torch.autograd.grad(kadconv.layer_norm(*leaves), leaves, dy)
    g, t = torch.Generator().manual_seed(15), 1e-4
    for k, grad in enumerate(grads):
        d = torch.randn(leaves[k].shape, generator=g, dtype=torch.float64)
        f = []
        for s in (t, -t):
            q = [p.detach().double().cpu() for p in (x, wt, bs)]
            q[k] = q[k] + s * d
            f.append((torch.nn.functional.layer_norm(q[0], (12,), q[1], q[2], 1e-5) * dy.double().cpu()).sum())
        want, got = ((f[0] - f[1]) / (2 * t)).item(), (grad.double().cpu() * d).sum().item()
        assert abs(got - want) <= 1e-5 * (grad.double().cpu() * d).abs().sum().item()


def test_same_result_every_time():
    x, dy, (wt, bs) = make(7000, 96, BF16, 16), make(7000, 96, BF16, 17), params(96)
    leaves = [t.requires_grad_(True) for t in (x, wt, bs)]
    first = None
    for _ in range(3):
        y = kadconv.layer_norm(*leaves)
        got = (y, *torch.autograd.grad(y, leaves, dy))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_other_stream():
    x, (wt, bs) = make(3000, 64, F16, 18), params(64)
    want = kadconv.layer_norm(x, wt, bs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kadconv.layer_norm(x * 1, wt, bs)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize('shape', [(40, 32), (3000, 700), (600, 9000)], ids=['small', 'wave', 'block'])
def test_captured(shape):
    """Forward and backward captured into one graph; every replay is checked, with eager work between."""
    x, dy, (wt, bs) = make(*shape, F16, 19), make(*shape, F16, 20), params(shape[1])

    def both(x, dy):
        y, mean, rstd = ops.layer_norm_forward(x, wt, bs, 1e-5, -1)
        return (y, *ops.layer_norm_backward(dy, x, wt, bs, mean, rstd, 1e-5, -1))

    sx, sdy = x.clone(), dy.clone()
    both(sx, sdy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(sx, sdy)
    for k in range(4):
        nx, ndy = make(*shape, F16, 30 + k), make(*shape, F16, 40 + k)
        sx.copy_(nx)
        sdy.copy_(ndy)
        graph.replay()
        want = both(nx, ndy)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_more_than_2_31_values():
    """Offsets that pass 32 bits: the last rows' results equal those of these rows alone."""
    rows, c = 530_000, 4104
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip('needs 40 GiB of GPU memory')
    assert rows * c > 2 ** 31
    x = torch.empty(rows, c, dtype=F16, device=DEV).normal_()
    wt, bs = params(c)
    y, mean, rstd = ops.layer_norm_forward(x, wt, bs, 1e-5, -1)
    dx, _, _ = ops.layer_norm_backward(y, x, wt, bs, mean, rstd, 1e-5, -1)
    last = slice(rows - 500, rows)
    ya, ma, ra = ops.layer_norm_forward(x[last], wt, bs, 1e-5, -1)
    assert torch.equal(y[last], ya) and torch.equal(mean[last], ma)
    assert torch.equal(dx[last], ops.layer_norm_backward(ya, x[last], wt, bs, ma, ra, 1e-5, -1)[0])


def test_compiled():
    """torch.compile traces the operator and its gradient without a graph break."""
    for dim, x in ((-1, make(20, 24, F32, 21)), (1, make_map(2, 24, 5, 4, F32, 21))):
        m = kadconv.LayerNorm(24, dim=dim).to(DEV)
        xs, dy = x.clone().requires_grad_(True), torch.randn_like(x)
        want = torch.autograd.grad(m(xs), (xs, m.weight, m.bias), dy)
        got = torch.autograd.grad(torch.compile(m, fullgraph=True, backend='aot_eager')(xs), (xs, m.weight, m.bias), dy)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals():
    x, (wt, bs) = make(3, 8, F32), params(8)
    with pytest.raises(TypeError):
        kadconv.layer_norm(x.double())
    with pytest.raises(ValueError, match='one device'):
        kadconv.layer_norm(x, wt.cpu())
    with pytest.raises(TypeError):
        kadconv.layer_norm(x, wt.half(), bs)
    with pytest.raises(ValueError, match='16384'):
        kadconv.layer_norm(torch.empty(1, 16385, device=DEV))
    with pytest.raises(ValueError, match='mean and rstd'):
        ops.layer_norm_backward(x, x, wt, bs, wt, wt, 1e-5, -1)
    with pytest.raises(ValueError, match='dy must'):
        ops.layer_norm_backward(x[:2], x, wt, bs, x[:, 0].contiguous(), x[:, 0].contiguous(), 1e-5, -1)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        xs = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(kadconv.layer_norm(xs, wt, bs).square().sum(), xs, create_graph=True)
        g.sum().backward()
