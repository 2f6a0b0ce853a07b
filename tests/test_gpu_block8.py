"""quantize8, matmul8 and linear8 on the GPU against their definitions in 64 bits."""
import copy

import pytest
import torch

import kadconv
from kadconv import Block8, _ext, block8
from tests._block8_ref import held, numbers, product, rounded
from tests._norm_ref import assert_within

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = pytest.mark.parametrize('dtype', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
DEV, INF, NAN = 'cuda', float('inf'), float('nan')


def make(rows, k, dtype, seed=0, spread=1.0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    v = torch.randn(rows, k, generator=g) * torch.exp(spread * torch.randn(k, generator=g)) * size
    return (v * (torch.rand(rows, k, generator=g) > 0.1)).to(dtype).to(DEV)


def check_held(codes, scales, v):
    """Codes and scales of rows v are those of the definition, and what is behind them is zeros and ones."""
    want, powers = held(v)
    k, blocks = v.shape[1], powers.shape[1]
    codes, scales = codes.reshape(v.shape[0], -1), scales.reshape(v.shape[0], -1)
    assert codes.shape[1] == blocks * 128 and scales.shape[1] == -(-blocks // 4) * 4
    got = codes[:, :k].float().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    assert not codes[:, k:].view(torch.uint8).any()
    bytes_ = scales.view(torch.uint8).int()
    assert torch.equal(bytes_[:, :blocks], powers.int() + 127) and (bytes_[:, blocks:] == 127).all()


@DTYPES
@pytest.mark.parametrize('shape', [(1, 1), (3, 7), (5, 127), (2, 128), (130, 129), (128, 256), (257, 300), (9, 520), (64, 1000), (300, 33)],
                         ids=lambda s: 'x'.join(map(str, s)))
def test_quantize(shape, dtype):
    v = make(*shape, dtype, seed=shape[1])
    q = kadconv.quantize8(v)
    assert tuple(q.shape) == shape and q.size == shape[1]
    check_held(q.codes, q.scales, v)
    assert torch.equal(q.dequantize(torch.float64), numbers(v))
    cpu = kadconv.quantize8(v.cpu())
    assert torch.equal(cpu.codes.view(torch.uint8), q.codes.cpu().view(torch.uint8))
    assert torch.equal(cpu.scales.view(torch.uint8), q.scales.cpu().view(torch.uint8))


@DTYPES
def test_quantize_rows_in_other_places(dtype):
    v = make(60, 200, dtype, 1)
    for t in (v[:, 3:150], v[::3], v[:, ::2], v.t(), v.view(3, 4, 5, 200)[:, 1:3], v[:1].expand(5, 200), v.view(3, 20, 200).transpose(0, 1)):
        q = kadconv.quantize8(t)
        assert q.codes.shape[:-1] == t.shape[:-1]
        check_held(q.codes, q.scales, t.reshape(-1, t.shape[-1]))
    m = v.view(3, 4, 5, 200).permute(0, 3, 1, 2)
    for t in (m, m.contiguous(), m[:, 7:90]):
        q = kadconv.quantize8(t, dim=1)
        check_held(q.codes, q.scales, t.permute(0, 2, 3, 1).reshape(60, -1))


def test_quantize_every_rounding():
    """Values on, between and next to the codes, ties to even; a block's largest at the border of its scale."""
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    middle = (codes[1:] + codes[:-1]) / 2
    line = torch.cat([codes, middle, torch.nextafter(middle, torch.tensor(INF)), torch.nextafter(middle, torch.tensor(-INF))])
    row = torch.cat([torch.tensor([448.0]), line.repeat_interleave(2)[:127 * 8]])
    rows = torch.stack([torch.cat([torch.tensor([448.0]), line[i * 100:i * 100 + 100], -line[i * 100:i * 100 + 27]])[:128] if
                        line[i * 100:].numel() >= 100 else torch.cat([torch.tensor([448.0]), line[-127:]]) for i in range(6)])
    for power in (-100, -20, 0, 7, 60):
        v = (rows * 2.0 ** power).to(DEV)
        q = kadconv.quantize8(v)
        check_held(q.codes, q.scales, v)
    del row
    for dtype in (F16, BF16):  # every 16-bit number, in blocks of neighbours and of all sizes
        every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
        for v in (every.view(512, 128), every.view(128, 512).t().contiguous(), every.view(128, 512)):
            q = kadconv.quantize8(v.to(DEV))
            check_held(q.codes, q.scales, v.to(DEV))
    edges = torch.tensor([448.0, 448.00003, 447.99997, 449.0, 256.0, 255.99998, 1.75, 1.7500001, 1e-38, 1.1754944e-38, 1e-40, 1.4e-45,
                          3.4028235e38, 3e38, 0.0]).to(DEV)
    v = edges[:, None] * torch.tensor([1.0, -0.37, 0.011]).to(DEV)
    q = kadconv.quantize8(v)
    check_held(q.codes, q.scales, v)


@DTYPES
def test_quantize_not_finite(dtype):
    v = make(6, 300, dtype, 2)
    v[0, 5], v[1, 5], v[2, 200] = NAN, INF, -INF
    v[3] = NAN
    v[4, :128] = 0
    q = kadconv.quantize8(v)
    check_held(q.codes, q.scales, v)


def exact_linear(x, w, bias=None, dtype=None):
    y, tol = product(numbers(x), numbers(w), dtype or x.dtype, bias)
    return y, rounded(y, tol, dtype or x.dtype)


SHAPES = [  # m, n, k: few rows and their borders, tiles and theirs, parts of k, short and long rows
    (1, 1, 1), (1, 16, 128), (1, 17, 129), (2, 5, 40), (7, 33, 1000), (16, 64, 300), (17, 48, 256), (33, 19, 520), (64, 100, 1300),
    (65, 1, 5), (66, 64, 128), (130, 40, 86), (100, 130, 700), (300, 43, 86), (257, 129, 513), (1000, 20, 64), (65, 65, 5000),
    (1, 300, 9000), (70, 3, 20000), (2100, 2050, 200)]


@DTYPES
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(map(str, s)))
def test_products(shape, dtype):
    m, n, k = shape
    x, w = make(m, k, dtype, 1), make(n, k, dtype, 2, spread=0.3)
    b = make(1, n, F32, 3)[0]
    y, tol = exact_linear(x, w, b)
    kept = kadconv.quantize8(w)
    with torch.no_grad():
        got = kadconv.linear8(x, kept, b)
        assert got.dtype == dtype and got.shape == (m, n)
        assert_within(got, y.cpu(), tol.cpu(), 'linear8')
        assert torch.equal(kadconv.linear8(x, w, b), got)
        assert torch.equal(block8.linear8_forward(x, w, b, None, -1), got)
        other = kadconv.matmul8(kadconv.quantize8(x), kept, b, dtype=dtype)
        assert_within(other, y.cpu(), tol.cpu(), 'matmul8')
        assert torch.equal(other, got)   # the same sums, whoever brought x to 8 bits
        for out in (F32, F16, BF16):
            z, t = product(numbers(x), numbers(w), out)
            assert_within(kadconv.matmul8(kadconv.quantize8(x), kept, dtype=out), z.cpu(), rounded(z, t, out).cpu(), 'matmul8')


@pytest.mark.parametrize('shape', [(2100, 4100, 300), (8200, 2048, 1024), (4096, 4096, 640), (2100, 4100, 1100), (4000, 4090, 1207),
                                   (3000, 5100, 1500), (4096, 4096, 1300), (8192, 4096, 1152), (4003, 4096, 2048)], ids=lambda s: 'x'.join(map(str, s)))
def test_large_tiles(shape):
    """Results in 16 bits next to those in 32, whose sums are exact: off by the cut of the products and two roundings.
    The cut is bounded by 7 * 2^-13 of the sum of magnitudes."""
    m, n, k = shape
    x, w = make(m, k, BF16, 1), make(n, k, BF16, 2, spread=0.3)
    qx, qw = kadconv.quantize8(x), kadconv.quantize8(w)
    want = kadconv.matmul8(qx, qw, dtype=F32).double()
    whole = torch.matmul(qx.dequantize().abs(), qw.dequantize().abs().t()).double()
    some = torch.matmul(qx.dequantize(torch.float64)[:300], qw.dequantize(torch.float64).t())
    assert ((want[:300] - some).abs() <= (k + 2) * 2.0 ** -24 * whole[:300] + 2.0 ** -24 * some.abs()).all()
    for dtype in (F16, BF16):
        got = kadconv.matmul8(qx, qw, dtype=dtype).double()
        tol = 7 * 2.0 ** -13 * whole + (k + 2) * 2.0 ** -23 * whole + torch.finfo(dtype).eps / 2 * want.abs() * 1.01 + 1e-7
        assert ((got - want).abs() <= tol).all()
        # and far nearer on the whole: 1e-4 of the norm beside the rounding
        assert (got - want).norm() <= (torch.finfo(dtype).eps / 2 + 1e-4) * want.norm()


@DTYPES
@pytest.mark.parametrize('act', [None, 'relu', 'silu'])
@pytest.mark.parametrize('m', [5, 50, 300])
def test_activations_and_bias(m, act, dtype):
    x, w = make(m, 140, dtype, 4), make(37, 140, dtype, 5, spread=0.1, size=0.1)
    kept = kadconv.quantize8(w)
    for b in (None, make(1, 37, F32, 6)[0], make(1, 37, dtype, 7)[0], make(37, 2, F32, 8)[:, 1]):
        y, tol = product(numbers(x), numbers(w), dtype, b)
        # slopes of at most 1.1; the sigmoid's own roundings
        if act == 'relu':
            y = y.clamp(min=0)
        elif act == 'silu':
            tol = 1.1 * tol + 16 * 2.0 ** -24 * y.abs()
            y = y * torch.sigmoid(y)
        assert_within(kadconv.linear8(x, kept, b, act), y.cpu(), rounded(y, tol, dtype).cpu(), 'y')
        assert torch.equal(kadconv.linear8(x, w, b, act), kadconv.linear8(x, kept, b, act))
        if b is None or b.is_contiguous():
            assert torch.equal(kadconv.matmul8(kadconv.quantize8(x), kept, b, act, dtype), kadconv.linear8(x, kept, b, act))


@DTYPES
@pytest.mark.parametrize('shape', [(33, 1, 1), (64, 64, 128), (65, 63, 127), (100, 65, 129), (129, 128, 512), (700, 300, 500), (2000, 129, 256),
                                   (20000, 200, 255), (16500, 256, 130), (40, 16300, 7), (8241, 43, 86), (16400, 100, 384), (5000, 1024, 500),
                                   (4100, 1000, 257), (3001, 5003, 256), (90, 30001, 65)], ids=str)
def test_short_rows_in_one_launch(shape, dtype):
    """Values of short rows that the product brings to 8 bits itself: as those that another launch brings there, to the bit
    (the sums of a result are taken in one order in both, but for 16-bit tiles of 256, which these sizes do not take)."""
    m, n, k = shape
    x, w, b = make(m, k, dtype, 1, spread=3.0), kadconv.quantize8(make(n, k, dtype, 2)), make(1, n, dtype, 3)[0]
    x[m // 2, k // 2] = float('nan')
    x[m // 3] = 0
    x[-1, 0] = float('inf')
    for act in (None, 'silu'):
        want = kadconv.matmul8(kadconv.quantize8(x), w, b, act, dtype)
        got = kadconv.linear8(x, w, b, act)
        assert torch.equal(got.nan_to_num(123.0), want.nan_to_num(123.0)) and torch.equal(got.isnan(), want.isnan())
        apart = torch.full((m, k + 3), float('nan'), device=DEV, dtype=dtype)[:, 2:-1]  # at odd places, other values around
        apart.copy_(x)
        assert torch.equal(kadconv.linear8(apart, w, b, act).nan_to_num(123.0), got.nan_to_num(123.0))


def check_gradients(x, w, b, dy, dim=-1):
    rows = x.detach().movedim(dim, -1).reshape(-1, x.shape[dim])
    drows = dy.movedim(dim, -1).reshape(-1, dy.shape[dim])
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = kadconv.linear8(leaves[0], leaves[1], leaves[2] if b is not None else None, dim=dim)
    want, tol = exact_linear(rows, w, b)
    assert_within(y.movedim(dim, -1).reshape(want.shape), want.cpu(), tol.cpu(), 'y')
    got = torch.autograd.grad(y, leaves, dy)
    assert [g.shape for g in got] == [t.shape for t in leaves] and [g.dtype for g in got] == [t.dtype for t in leaves]
    want, tol = exact_linear(drows, w.t(), None, x.dtype)
    assert got[0].movedim(dim, -1).is_contiguous()
    assert_within(got[0].movedim(dim, -1).reshape(want.shape), want.cpu(), tol.cpu(), 'dx')
    want, tol = exact_linear(drows.t(), rows.t(), None, w.dtype)
    assert_within(got[1], want.cpu(), tol.cpu(), 'dw')
    if b is not None:
        d = drows.double()
        tol = rounded(d.sum(0), (d.shape[0] + 2) * 2.0 ** -24 * d.abs().sum(0), b.dtype)
        assert_within(got[2], d.sum(0).cpu(), tol.cpu(), 'db')
    other = block8.linear8_backward(dy, x, w, b, dim)
    assert all(torch.equal(a, c) for a, c in zip(got, other))


@DTYPES
@pytest.mark.parametrize('shape', [(1, 3, 5), (2, 16, 128), (40, 33, 70), (64, 130, 129), (65, 7, 300), (130, 128, 128), (300, 43, 86),
                                   (513, 257, 140), (5000, 24, 33)], ids=lambda s: 'x'.join(map(str, s)))
def test_gradients(shape, dtype):
    m, n, k = shape
    x, w, dy = make(m, k, dtype, 1), make(n, k, dtype, 2, spread=0.3), make(m, n, dtype, 3, size=0.1)
    check_gradients(x, w, make(1, n, F32, 4)[0], dy)
    check_gradients(x, make(n, k, F32, 2, spread=0.3), None, dy)
    check_gradients(x, w, make(1, n, dtype, 4)[0], dy)


@DTYPES
@pytest.mark.parametrize('layout', ['cl', 'nchw', 'slice'])
def test_maps(layout, dtype):
    for n, c, h, w, co in ((2, 40, 6, 9, 24), (1, 86, 5, 5, 43), (1, 12, 1, 1, 5)):
        x, dy = (make(n * h * w, k, dtype, 6).view(n, h, w, k).permute(0, 3, 1, 2) for k in (c, co))
        if layout == 'nchw':
            x, dy = x.contiguous(), dy.contiguous()
        if layout == 'slice':
            x = torch.cat([x, x], 1).contiguous(memory_format=torch.channels_last)[:, 1:1 + c]
        check_gradients(x, make(co, c, dtype, 7), make(1, co, F32, 8)[0], dy, dim=1)


@DTYPES
def test_rows_in_other_places(dtype):
    w, b = make(20, 70, dtype, 9), make(1, 20, F32, 10)[0]
    for rows in (12, 150):
        wide = make(2 * rows, 90, dtype, 11)
        dy = make(rows, 20, dtype, 12)
        for x in (wide[:rows, 3:73], wide[::2, :70], wide[:rows].t()[:70].t(), wide[:1, :70].expand(rows, 70),
                  make(70, rows, dtype, 13).t()):
            check_gradients(x, w, b, dy)
        check_gradients(wide[:rows, :70], make(70, 20, dtype, 14).t(), b, dy[:, :1].expand(rows, 20))
        check_gradients(wide[:rows, :70].reshape(3, 2, -1, 70), w, b, dy.reshape(3, 2, -1, 20))
    check_gradients(wide[0, :70], w, b, dy[0])


def test_gradient_of_some_inputs():
    for m in (30, 200):
        x, w, b, dy = make(m, 50, F32, 1), make(20, 50, F32, 2), make(1, 20, F32, 3)[0], make(m, 20, F32, 4)
        full = block8.linear8_backward(dy, x, w, b, -1)
        for pick in ((0,), (1,), (2,), (0, 1), (1, 2), (0, 2)):
            leaves = [t.clone().requires_grad_(i in pick) for i, t in enumerate((x, w, b))]
            got = torch.autograd.grad(kadconv.linear8(*leaves), [leaves[i] for i in pick], dy)
            assert all(torch.equal(g, full[i]) for g, i in zip(got, pick))
            some = block8.linear8_backward(dy, x, w, b, -1, *(i in pick for i in range(3)))
            assert all((s is None) == (i not in pick) for i, s in enumerate(some))


def test_gradient_against_differences():
    """Of numbers that 8 bits hold exactly the product is bilinear: a difference is the gradient, where the upstream
    gradient is held exactly too."""
    g = torch.Generator().manual_seed(1)
    x, w, dy = (torch.randint(-8, 9, s, generator=g).float().to(DEV) for s in ((100, 40), (30, 40), (100, 30)))
    dx, dw, _ = block8.linear8_backward(dy, x, w, None, -1)
    f = lambda x, w: (kadconv.linear8(x, w).double() * dy.double()).sum()  # noqa: E731
    for i, j in ((0, 0), (99, 39), (50, 7)):
        e = torch.zeros_like(x)
        e[i, j] = 1 if x[i, j] < 8 else -1
        assert (f(x + e, w) - f(x, w)) * e[i, j] == dx[i, j].double()
    for i, j in ((0, 0), (29, 39), (12, 5)):
        e = torch.zeros_like(w)
        e[i, j] = 1 if w[i, j] < 8 else -1
        assert (f(x, w + e) - f(x, w)) * e[i, j] == dw[i, j].double()


@DTYPES
@pytest.mark.parametrize('m', [9, 200])
def test_not_finite_stays_in_its_row(m, dtype):
    x, w = make(m, 300, dtype, 1), make(40, 300, dtype, 2)
    x[3, 299], x[5, 0] = NAN, INF
    y = kadconv.linear8(x, kadconv.quantize8(w))
    assert torch.isnan(y[[3, 5]]).all() and torch.isfinite(y[[0, 1, 2, 4, 6, 8]]).all()
    x = make(m, 300, dtype, 1)
    w[7, 130] = -INF
    y = kadconv.linear8(x, kadconv.quantize8(w))
    assert torch.isnan(y[:, 7]).all() and torch.isfinite(y[:, :7]).all() and torch.isfinite(y[:, 8:]).all()


@DTYPES
def test_a_row_does_not_depend_on_the_others(dtype):
    """In one form the same row gives the same bits, whichever rows are around it; nothing behind the last is written."""
    x, w = make(700, 260, dtype, 1), kadconv.quantize8(make(130, 260, dtype, 2))
    y = kadconv.linear8(x, w)
    assert torch.equal(kadconv.linear8(x[100:400], w), y[100:400])
    few = kadconv.linear8(x[:32], w)
    assert torch.equal(kadconv.linear8(x[5:6], w), few[5:6])
    assert torch.equal(few, y[:32]) or dtype != F32  # the forms' sums may differ in order


def test_far_scales():
    """Blocks from 2^-100 to 2^100 in one row: their products cancel in the exponent."""
    g = torch.Generator().manual_seed(3)
    powers = torch.tensor([-100.0, 100.0, 0.0, 40.0, -40.0])
    x = torch.randn(80, 640, generator=g) * torch.exp2(powers).repeat_interleave(128)
    w = torch.randn(30, 640, generator=g) * torch.exp2(-powers).repeat_interleave(128)
    for m in (10, 80):
        y, tol = exact_linear(x[:m].to(DEV), w.to(DEV))
        assert_within(kadconv.linear8(x[:m].to(DEV), w.to(DEV)), y.cpu(), tol.cpu(), 'y')


def test_empty():
    w, b = make(6, 8, F32), make(1, 6, F32)[0]
    for shape, dim in (((0, 8), -1), ((3, 0, 8), -1), ((0, 8, 4, 4), 1), ((2, 8, 0, 4), 1)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        wr, br = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
        y = kadconv.linear8(x, wr, br, dim=dim)
        want = list(shape)
        want[dim] = 6
        assert list(y.shape) == want
        dx, dw, db = torch.autograd.grad(y, (x, wr, br), torch.empty_like(y))
        assert dx.shape == x.shape and not dw.any() and not db.any()
        assert list(kadconv.linear8(x.detach(), kadconv.quantize8(w), b, dim=dim).shape) == want
        q = kadconv.quantize8(x.detach(), dim)
        assert list(kadconv.matmul8(q, kadconv.quantize8(w)).shape) == [*q.shape[:-1], 6]


def test_changes_after_the_forward_pass_are_not_seen():
    x, w, dy = make(100, 50, F32, 1), make(20, 50, F32, 2), make(100, 20, F32, 3)
    want = block8.linear8_backward(dy, x, w, None, -1)
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = kadconv.linear8(xs, ws)
    with torch.no_grad():
        xs.zero_()
        ws.fill_(3)
    got = torch.autograd.grad(y, (xs, ws), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('shape', [(5000, 130, 200), (9, 300, 5000), (130, 70, 9000)], ids=['tiles', 'few', 'parts'])
def test_same_result_every_time(shape):
    m, n, k = shape
    x, w, b, dy = make(m, k, BF16, 1), make(n, k, BF16, 2), make(1, n, F32, 3)[0], make(m, n, BF16, 4)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    first = None
    for _ in range(3):
        y = kadconv.linear8(*leaves)
        got = (y, *torch.autograd.grad(y, leaves, dy))
        first = first or got
        assert all(torch.equal(a, c) for a, c in zip(first, got))


def test_other_stream():
    x, w = make(300, 200, F16, 1), make(50, 200, F16, 2)
    want = kadconv.linear8(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kadconv.linear8(x * 1, w * 1)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


@pytest.mark.parametrize('shape', [(3, 40, 300), (200, 40, 300), (100, 30, 9000), (2100, 2050, 140)], ids=['few', 'tiles', 'parts', 'large'])
def test_captured(shape):
    """Forward, backward and a served call captured into one graph; every replay is checked, with eager work between."""
    m, n, k = shape
    b = make(1, n, F32, 9)[0]

    def all_of(x, w, dy):
        kept = kadconv.quantize8(w)
        return (block8.linear8_forward(x, w, b, None, -1), block8.linear8_forward(x, kept, b, 'silu', -1),
                *block8.linear8_backward(dy, x, w, b, -1))

    def state(seed):
        return make(m, k, F16, seed), make(n, k, F16, seed + 1), make(m, n, F16, seed + 2)

    held_ = state(20)
    all_of(*held_)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = all_of(*held_)
    for r in range(4):
        new = state(30 + 3 * r)
        for a, c in zip(held_, new):
            a.copy_(c)
        graph.replay()
        want = all_of(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want)), r


def test_compiled():
    for dim, x in ((-1, make(90, 24, F32, 1)), (1, make(90, 24, F32, 1).view(2, 9, 5, 24).permute(0, 3, 1, 2))):
        m = kadconv.Linear8(24, 10, dim=dim).to(DEV)
        xs = x.clone().requires_grad_(True)
        y = m(xs)
        dy = torch.randn_like(y)
        want = torch.autograd.grad(y, (xs, m.weight, m.bias), dy)
        got = torch.autograd.grad(torch.compile(m, fullgraph=True, backend='aot_eager')(xs), (xs, m.weight, m.bias), dy)
        assert all(torch.equal(a, c) for a, c in zip(want, got))
        with torch.no_grad():
            kept = kadconv.quantize8(m.weight)

            def served(x):
                return kadconv.linear8(x, kept, m.bias, 'silu', dim)
            assert torch.equal(torch.compile(served, fullgraph=True, backend='aot_eager')(x), served(x))


def test_module():
    """Kept weights follow the parameter; calls that are differentiated go by the parameter itself."""
    x = make(100, 40, F16, 1)
    m = kadconv.Linear8(40, 12, act='silu').to(DEV, F16)
    trained = m(x)
    assert trained.requires_grad
    torch.testing.assert_close(trained, torch.nn.functional.silu(kadconv.linear8(x, m.weight, m.bias)), rtol=0, atol=0)
    trained.sum().backward()
    assert m.weight.grad is not None and m.bias.grad is not None
    m.eval()
    with torch.no_grad():
        y = m(x)
        assert torch.equal(y, kadconv.linear8(x, kadconv.quantize8(m.weight), m.bias, 'silu')) and torch.equal(m(x), y)
        m.weight.mul_(2)
        assert torch.equal(m(x), kadconv.linear8(x, kadconv.quantize8(m.weight), m.bias, 'silu'))
        m.weight = torch.nn.Parameter(torch.zeros_like(m.weight))
        assert torch.equal(m(x), torch.nn.functional.silu(m.bias).expand(100, 12))
        other = copy.deepcopy(m)
        other.weight.fill_(1)
        assert torch.equal(other(x), kadconv.linear8(x, other.weight, other.bias, 'silu'))
        m.load_state_dict(other.state_dict())
        assert torch.equal(m(x), other(x))
    assert m(x).requires_grad
    with torch.inference_mode():
        fresh = kadconv.Linear8(40, 12).to(DEV, F16).eval()
        assert torch.equal(fresh(x), kadconv.linear8(x, fresh.weight, fresh.bias))


def test_module_on_another_stream():
    """The weight is laid out on one stream, behind much other work, and used on another at once."""
    x, m = make(200, 300, F16, 1), kadconv.Linear8(300, 64).to(DEV, F16).eval()
    busy = torch.randn(4096, 4096, device=DEV)
    side = torch.cuda.Stream()
    with torch.no_grad():
        want = kadconv.linear8(x, kadconv.quantize8(m.weight), m.bias)
        torch.cuda.synchronize()
        for _ in range(20):
            busy = busy @ busy
            busy = busy / busy.norm()
        m(x)
        with torch.cuda.stream(side):
            got = m(x)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_module_in_a_graph_follows_its_weight():
    x, m = make(100, 300, F16, 1), kadconv.Linear8(300, 20, act='relu').to(DEV, F16).eval()
    with torch.no_grad():
        m(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x)
        for k in range(3):
            m.weight.normal_()
            graph.replay()
            want = kadconv.linear8(x, m.weight, m.bias, 'relu')
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(m(x), want), k


@pytest.mark.parametrize('rows', [(1 << 20) + 200, 1 << 22])
def test_gradient_over_many_rows(rows):
    """Sums over more than 2^20 rows, of numbers that 8 bits hold and whose sums 32 bits hold exactly."""
    x = torch.randint(-1, 2, (rows, 3), device=DEV).to(F16)
    dy = torch.randint(-1, 2, (rows, 2), device=DEV).to(F16)
    w = torch.ones(2, 3, device=DEV)
    _, dw, db = block8.linear8_backward(dy, x, w, torch.zeros(2, device=DEV), -1, need_x=False)
    assert torch.equal(dw.double(), dy.double().t() @ x.double()) and torch.equal(db.double(), dy.double().sum(0))


def test_refusals():
    x, w = make(3, 40, F32), make(5, 40, F32)
    many = torch.zeros((1 << 22) + 1, 1, device=DEV, dtype=F16)
    with pytest.raises(ValueError, match='rows'):
        kadconv.linear8(many, torch.ones(1, 1, device=DEV, requires_grad=True))
    with pytest.raises(ValueError, match='rows'):
        block8.linear8_backward(many, many, torch.ones(1, 1, device=DEV), None, -1)
    assert not kadconv.linear8(many, torch.ones(1, 1, device=DEV)).any()
    with pytest.raises(NotImplementedError, match='activation'):
        torch.ops.kadconv.linear8(x, w.clone().requires_grad_(True), None, 'silu', -1)
    q = kadconv.quantize8(w)
    with pytest.raises(TypeError):
        kadconv.linear8(x.double(), w)
    with pytest.raises(TypeError):
        kadconv.linear8(x, w.half())
    with pytest.raises(ValueError, match='one device'):
        kadconv.linear8(x, w.cpu())
    with pytest.raises(ValueError, match='on cuda'):
        kadconv.linear8(x, q.to('cpu'))
    with pytest.raises(ValueError, match='rows of 40'):
        kadconv.linear8(x[:, :39], w)
    with pytest.raises(ValueError, match='rows of 40'):
        kadconv.linear8(x[:, :39], q)
    with pytest.raises(ValueError, match='bias'):
        kadconv.linear8(x, w, torch.zeros(4, device=DEV))
    with pytest.raises(ValueError, match='act'):
        kadconv.linear8(x, w, act='gelu')
    with pytest.raises(NotImplementedError, match='activation'):
        kadconv.linear8(x, w.clone().requires_grad_(True), act='silu')
    with pytest.raises(NotImplementedError, match='8 bits'):
        kadconv.linear8(x.clone().requires_grad_(True), q)
    native = _ext.native()
    for codes, scales in ((q.codes[:, :127], q.scales), (q.codes, q.scales[:, :3]), (q.codes.t().contiguous().t(), q.scales)):
        with pytest.raises(ValueError):
            native.linear8_kept(x, codes, scales, 40, None, None, -1)
        with pytest.raises(ValueError):
            native.matmul8(q.codes, q.scales, codes, scales, 40, None, None, F32)
    with pytest.raises(TypeError):
        native.linear8_kept(x, q.codes.view(torch.uint8), q.scales, 40, None, None, -1)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        xs = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(kadconv.linear8(xs, w).square().sum(), xs, create_graph=True)
        g.sum().backward()
