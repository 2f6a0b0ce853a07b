"""group_norm_act on the GPU, forward and gradients, against the formulas in 64 bits."""
import pytest
import torch

import kadconv
from kadconv import ops
from tests._norm_ref import assert_within, reference

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEV = 'cuda'


def make(n, c, h, w, dtype, seed=0, layout='cl', loc=0.0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    v = (torch.randn(n, c, h, w, generator=g) * scale + loc + 0.3 * torch.randn(1, c, 1, 1, generator=g)).to(dtype).to(DEV)
    if layout == 'nchw':
        return v.contiguous()
    if layout == 'slice':  # channels 8 .. 8 + c of a wider channels-last map
        wide = torch.full((n, h, w, c + 24), 7.0, dtype=dtype, device=DEV)
        wide[..., 8:8 + c] = v.permute(0, 2, 3, 1)
        return wide[..., 8:8 + c].permute(0, 3, 1, 2)
    if layout == 'odd':  # dense, but its memory begins one value after a 16-byte border
        flat = torch.empty(v.numel() + 1, dtype=dtype, device=DEV)[1:]
        out = flat.view(n, h, w, c).permute(0, 3, 1, 2)
        return out.copy_(v)
    return v.contiguous(memory_format=torch.channels_last)


def params(c, dtype=F32, seed=1):
    g = torch.Generator().manual_seed(seed)
    w = (1 + 0.3 * torch.randn(c, generator=g)).to(dtype).to(DEV)
    return w, (0.2 * torch.randn(c, generator=g)).to(dtype).to(DEV)


def away_from_zero(x, groups, w, b, eps):
    """x with the values moved whose normalised value is so near 0 that 32 bits cannot tell its sign."""
    for _ in range(20):
        z = reference(x, groups, w, b, eps, None)['y']
        near = (z.abs() < 1e-3).to(x.device)
        if not near.any():
            break
        x = torch.where(near, x + 0.05, x).contiguous(memory_format=torch.channels_last)
    return x


def check(x, groups, w, b, act, dy, eps=1e-5):
    ref = reference(x, groups, w, b, eps, act, dy)
    xs = x.detach().requires_grad_(True)
    ws = None if w is None else w.detach().requires_grad_(True)
    bs = None if b is None else b.detach().requires_grad_(True)
    with torch.no_grad():
        y0 = kadconv.group_norm_act(xs, groups, ws, bs, eps, act)
    y = kadconv.group_norm_act(xs, groups, ws, bs, eps, act)
    assert y.dtype == x.dtype and y.permute(0, 2, 3, 1).is_contiguous()
    assert torch.equal(y, y0)
    assert_within(y, ref['y'], ref['tol_y'], 'y')
    wanted = [t for t in (xs, ws, bs) if t is not None]
    grads = iter(torch.autograd.grad(y, wanted, dy))
    dx = next(grads)
    assert dx.dtype == x.dtype
    assert_within(dx, ref['dx'], ref['tol_dx'], 'dx')
    for name, p in (('dw', w), ('db', b)):
        if p is None:
            continue
        got = next(grads)
        assert got.dtype == p.dtype and got.shape == p.shape
        assert_within(got, ref[name], ref['tol_' + name] + torch.finfo(p.dtype).eps / 2 * ref[name].abs() + 1e-30, name)


SHAPES = [  # n, c, groups, h, w
    (1, 1, 1, 1, 2), (2, 8, 8, 1, 2), (1, 8, 1, 1, 1), (3, 16, 4, 1, 1), (1, 64, 8, 20, 20), (2, 48, 6, 13, 17),
    (2, 86, 2, 23, 19), (3, 27, 3, 11, 7), (2, 12, 4, 9, 5), (1, 30, 10, 31, 3), (5, 7, 7, 6, 6), (2, 256, 32, 16, 15),
    (1, 1023, 11, 5, 4), (2, 512, 1, 7, 9), (1, 2560, 32, 4, 3), (1, 96, 32, 40, 41), (4, 40, 5, 1, 129),
    (1, 3, 1, 100, 101), (2, 34, 17, 33, 29), (1, 8192, 2, 2, 3), (1, 128, 16, 120, 110), (2, 20, 2, 150, 90)]


@pytest.mark.parametrize('dtype', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(map(str, s)))
def test_forward_and_gradients(shape, dtype):
    n, c, g, h, w = shape
    x = make(n, c, h, w, dtype, seed=c)
    wt, bs = params(c)
    dy = make(n, c, h, w, dtype, seed=c + 1)
    check(x, g, wt, bs, 'silu', dy)


@pytest.mark.parametrize('dtype', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('layout', ['nchw', 'slice', 'odd'])
@pytest.mark.parametrize('shape', [(2, 48, 6, 13, 17), (2, 27, 3, 9, 7), (1, 128, 4, 61, 53), (3, 16, 2, 1, 5)],
                         ids=lambda s: 'x'.join(map(str, s)))
def test_layouts(shape, layout, dtype):
    n, c, g, h, w = shape
    wt, bs = params(c)
    check(make(n, c, h, w, dtype, 3, layout), g, wt, bs, None, make(n, c, h, w, dtype, 4, layout))
    check(make(n, c, h, w, dtype, 3, 'cl'), g, wt, bs, 'silu', make(n, c, h, w, dtype, 4, layout))


@pytest.mark.parametrize('dtype', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('act', [None, 'relu', 'silu'])
def test_activations_and_parameters(act, dtype):
    for n, c, g, h, w in [(2, 24, 3, 10, 9), (1, 22, 2, 45, 40)]:
        x, dy = make(n, c, h, w, dtype, 5), make(n, c, h, w, dtype, 6)
        for pdt in {F32, dtype}:
            wt, bs = params(c, pdt)
            for pw, pb in ((wt, bs), (wt, None), (None, bs), (None, None)):
                xa = away_from_zero(x, g, pw, pb, 1e-5) if act == 'relu' else x
                check(xa, g, pw, pb, act, dy)


def test_mean_far_from_zero():
    """Values whose spread is a thousandth of their mean, and an outlier in the first place."""
    wt, bs = params(32)
    for h, w in ((12, 12), (90, 80)):
        x = make(2, 32, h, w, F32, 7, loc=1000.0)
        check(x, 4, wt, bs, 'silu', make(2, 32, h, w, F32, 8))
        x = make(2, 32, h, w, F32, 7)
        x[:, :, 0, 0] = 3000.0
        check(x, 4, wt, bs, None, make(2, 32, h, w, F32, 8))


def test_constant_group():
    """No spread at all: z is the bias, and the gradient is finite."""
    wt, bs = params(16)
    x = torch.full((2, 16, 9, 8), 3.0, device=DEV).contiguous(memory_format=torch.channels_last)
    check(x, 4, wt, bs, 'silu', make(2, 16, 9, 8, F32, 9))
    one = make(2, 4, 1, 1, F32, 9)  # groups of a single value
    check(one, 4, *params(4), 'silu', make(2, 4, 1, 1, F32, 10))


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
@pytest.mark.parametrize('hw', [(6, 5), (70, 65)])
def test_not_finite_stays_in_its_group(bad, hw):
    x = make(2, 32, *hw, F16, 11)
    x[1, 9, 3, 2] = bad   # group 2 of 8, image 1
    wt, bs = params(32)
    xs, ws = x.requires_grad_(True), wt.requires_grad_(True)
    y = kadconv.group_norm_act(xs, 8, ws, bs, act='silu')
    dx, dw = torch.autograd.grad(y, (xs, ws), torch.ones_like(y))
    hit = torch.zeros(2, 32, dtype=torch.bool, device=DEV)
    hit[1, 8:12] = True
    for t in (y, dx):
        assert torch.isnan(t[hit]).all() and torch.isfinite(t[~hit]).all()
    assert torch.isnan(dw[8:12]).all() and torch.isfinite(dw[12:]).all() and torch.isfinite(dw[:8]).all()


def test_empty():
    wt, bs = params(8)
    for n, h, w in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        x = torch.empty(n, 8, h, w, device=DEV, requires_grad=True)
        wr, br = wt.clone().requires_grad_(True), bs.clone().requires_grad_(True)
        y = kadconv.group_norm_act(x, 2, wr, br, act='silu')
        assert y.shape == x.shape
        dx, dw, db = torch.autograd.grad(y, (x, wr, br), torch.empty_like(y))
        assert dx.shape == x.shape and not dw.any() and not db.any()


def test_gradient_of_some_inputs():
    """Only what is asked for is computed, and an expanded gradient (a sum's) is read right."""
    x, (wt, bs) = make(2, 24, 8, 7, F32, 12), params(24)
    dy = torch.ones(2, 24, 8, 7, device=DEV)
    ref = reference(x, 3, wt, bs, 1e-5, 'silu', dy)
    xs = x.clone().requires_grad_(True)
    kadconv.group_norm_act(xs, 3, wt, bs, act='silu').sum().backward()
    assert_within(xs.grad, ref['dx'], ref['tol_dx'], 'dx')
    ws = wt.clone().requires_grad_(True)
    kadconv.group_norm_act(x, 3, ws, bs, act='silu').sum().backward()
    assert_within(ws.grad, ref['dw'], ref['tol_dw'], 'dw')
    bb = bs.clone().requires_grad_(True)
    kadconv.group_norm_act(x, 3, wt, bb, act='silu').sum().backward()
    assert_within(bb.grad, ref['db'], ref['tol_db'], 'db')


def test_gradient_against_differences():
    """Along random directions: (f(x + t d) - f(x - t d)) / 2t of the 64-bit forward equals <dx, d>.  The
    difference is off by its third derivative times t^2 (t = 1e-3: under 1e-4 of the sum of magnitudes)."""
    x, (wt, bs) = make(2, 12, 5, 6, F32, 13), params(12)
    dy = make(2, 12, 5, 6, F32, 14)
    xs, ws, bb = (t.clone().requires_grad_(True) for t in (x, wt, bs))
    y = kadconv.group_norm_act(xs, 3, ws, bb, act='silu')
    grads = torch.autograd.grad(y, (xs, ws, bb), dy)
    g = torch.Generator().manual_seed(15)
    t = 1e-3
    for k, (p, grad) in enumerate(zip((x, wt, bs), grads)):
        d = torch.randn(p.shape, generator=g, dtype=torch.float64)
        f = []
        for s in (t, -t):
            q = [x.double().cpu(), wt.double().cpu(), bs.double().cpu()]
            q[k] = q[k] + s * d
            f.append((reference(*q[:1], 3, q[1], q[2], 1e-5, 'silu')['y'] * dy.double().cpu()).sum())
        want = ((f[0] - f[1]) / (2 * t)).item()
        got = (grad.double().cpu() * d).sum().item()
        assert abs(got - want) <= 1e-4 * (grad.double().cpu() * d).abs().sum().item()


def test_same_result_every_time():
    x, dy = make(3, 96, 50, 47, BF16, 16), make(3, 96, 50, 47, BF16, 17)
    wt, bs = params(96)
    xs, ws, bb = x.requires_grad_(True), wt.requires_grad_(True), bs.requires_grad_(True)
    first = None
    for _ in range(3):
        y = kadconv.group_norm_act(xs, 6, ws, bb, act='silu')
        got = (y, *torch.autograd.grad(y, (xs, ws, bb), dy))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_other_stream():
    x, (wt, bs) = make(2, 64, 40, 40, F16, 18), params(64)
    want = kadconv.group_norm_act(x, 8, wt, bs, act='silu')
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x2 = x * 1
        got = kadconv.group_norm_act(x2, 8, wt, bs, act='silu')
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize('shape', [(1, 32, 4, 12, 12), (2, 64, 8, 90, 85)], ids=['small', 'split'])
def test_captured(shape):
    """Forward and backward captured into one graph; every replay is checked, with eager work between."""
    n, c, g, h, w = shape
    x, dy, (wt, bs) = make(n, c, h, w, F16, 19), make(n, c, h, w, F16, 20), params(c)

    def both(x, dy):
        y, mean, rstd = ops.group_norm_act_forward(x, g, wt, bs, 1e-5, 'silu')
        return (y, *ops.group_norm_act_backward(dy, x, g, wt, bs, mean, rstd, 1e-5, 'silu'))

    sx, sdy = x.clone(memory_format=torch.preserve_format), dy.clone(memory_format=torch.preserve_format)
    both(sx, sdy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(sx, sdy)
    for k in range(4):
        nx, ndy = make(n, c, h, w, F16, 30 + k), make(n, c, h, w, F16, 40 + k)
        sx.copy_(nx)
        sdy.copy_(ndy)
        graph.replay()
        want = both(nx, ndy)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_more_than_2_31_values():
    """Offsets that pass 32 bits: the last image's result equals that of the image alone."""
    n, c, h, w = 3, 64, 3400, 3400
    free, _ = torch.cuda.mem_get_info()
    if free < 60 << 30:
        pytest.skip('needs 60 GiB of GPU memory')
    assert n * c * h * w > 2 ** 31
    x = torch.empty(n, h, w, c, dtype=F16, device=DEV)
    for k in range(n):
        x[k].normal_(mean=0.1 * k)
    x = x.permute(0, 3, 1, 2)
    wt, bs = params(c)
    y, mean, rstd = ops.group_norm_act_forward(x, 8, wt, bs, 1e-5, 'silu')
    ya, ma, ra = ops.group_norm_act_forward(x[2:], 8, wt, bs, 1e-5, 'silu')
    # other splits of the sums: the statistics agree to 32-bit sums' rounding, the map to one step
    torch.testing.assert_close(mean[2:], ma, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(rstd[2:], ra, rtol=1e-5, atol=0)
    assert ((y[2:].float() - ya.float()).abs() <= 2 ** -10 * ya.float().abs() + 1e-5).all()
    dx, _, _ = ops.group_norm_act_backward(y, x, 8, wt, bs, mean, rstd, 1e-5, 'silu')
    da, _, _ = ops.group_norm_act_backward(ya, x[2:], 8, wt, bs, ma, ra, 1e-5, 'silu')
    assert ((dx[2:].float() - da.float()).abs() <= 2 ** -8 * da.float().abs() + 1e-3).all()


def test_compiled():
    """torch.compile traces the operator and its gradient without a graph break."""
    x, (wt, bs) = make(2, 24, 9, 8, F32, 21), params(24)
    dy = make(2, 24, 9, 8, F32, 22)
    m = kadconv.GroupNormAct(3, 24, act='silu').to(DEV)
    with torch.no_grad():
        m.weight.copy_(wt)
        m.bias.copy_(bs)
    xs = x.clone().requires_grad_(True)
    want = torch.autograd.grad(m(xs), (xs, m.weight, m.bias), dy)
    f = torch.compile(m, fullgraph=True, backend='aot_eager')
    got = torch.autograd.grad(f(xs), (xs, m.weight, m.bias), dy)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals():
    x = make(1, 8, 4, 4, F32)
    wt, bs = params(8)
    with pytest.raises(TypeError):
        kadconv.group_norm_act(x.double(), 2, None, None)
    with pytest.raises(ValueError, match='one device'):
        kadconv.group_norm_act(x, 2, wt.cpu(), None)
    with pytest.raises(TypeError):
        kadconv.group_norm_act(x, 2, wt.half(), bs)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        xs = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(kadconv.group_norm_act(xs, 2, wt, bs).square().sum(), xs, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize('dtype', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('at', [40.0, 400.0, 1020.0, 2.0 ** 25])
@pytest.mark.parametrize('shape', [(2, 16, 4, 6, 5), (2, 16, 4, 61, 60), (1, 9000, 30, 2, 3)], ids=['small', 'split', 'wide'])
def test_silu_far_from_zero(shape, at, dtype):
    """Where e^-z is under half a step of 1, SiLU's slope 1 + z e^-z (1 + ...) is 1 in 32 bits, however large z: the
    gradients are those without an activation, bit for bit.  Gradients dy that are small integers sum to db without
    a rounding."""
    n, c, g, h, w = shape
    x, (wt, _) = make(n, c, h, w, dtype, 23), params(c)
    wt = wt.clamp(0.2, 2.0)              # z within 10 of `at`: |xhat| of these sizes is under 5
    bias = torch.full((c,), at, device=DEV)
    gen = torch.Generator().manual_seed(24)
    dy = torch.randint(-3, 4, (n, h, w, c), generator=gen).to(dtype).to(DEV).permute(0, 3, 1, 2)
    grads = []
    for act in ('silu', None):
        leaves = [t.clone(memory_format=torch.preserve_format).requires_grad_(True) for t in (x, wt, bias)]
        grads.append(torch.autograd.grad(kadconv.group_norm_act(leaves[0], g, *leaves[1:], act=act), leaves, dy))
    assert torch.equal(grads[0][2].double(), dy.double().sum(dim=(0, 2, 3)))
    for got, want, name in zip(*grads, ('dx', 'dw', 'db')):
        assert torch.equal(got, want), name
