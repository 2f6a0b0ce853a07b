"""distill_loss and its gradient at temperatures up to the largest, where entries cover all classes, against 50 digits.

T^2 times a difference of order 1 / T^2 is left of logarithms of order 1: what they are off by is multiplied by T^2.  In 64 bits
with exponentials taken as e^x - 1, a row's terms are of the size of its arguments (z - max) / T, which 1 / T divides, and
sums of n of them are off by (n + 16) 2^-53 of that size: T^2 size (V + K + 16) 2^-53 in all, and T (V + K + 16) 2^-53 for a
gradient's q and p, each at most 1.  Results are rounded once."""
import pytest
import torch

import kadconv
from tests._distill_exact import reference

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
TEMPERATURES = [8.0, 9.0, 100.0, 1e3, 1e4, 1e5, 1e6]


def make(rows, v, k, dtype, seed=0):
    """A student near its teacher, whose best k classes are known."""
    g = torch.Generator().manual_seed(seed)
    teacher = 2 * torch.randn(rows, v, generator=g)
    z = (teacher + 0.3 * torch.randn(rows, v, generator=g)).to(dtype)
    top = torch.topk(teacher, k, dim=1)
    return z, top.values.to(dtype), top.indices


def check(z, t, i, temperature, device):
    losses, grads, sizes = (torch.tensor(x, dtype=torch.float64) for x in reference(z, t, i, temperature))
    n = z.shape[1] + t.shape[1] + 16
    # up to 8 the sums are 32-bit on the GPU, as their documentation says
    eps = 2.0 ** -24 if device == 'cuda' and temperature <= 8 else 2.0 ** -53
    tol = temperature ** 2 * n * eps * (sizes if eps < 2.0 ** -50 else sizes + 4) + 2.0 ** -23 * losses.abs()
    zs = z.to(device).requires_grad_(True)
    loss = kadconv.distill_loss(zs, t.to(device), i.to(device), temperature, 'none')
    assert loss.dtype == torch.float32
    off = (loss.detach().double().cpu() - losses).abs()
    assert (off <= tol).all(), (off.max().item(), tol.min().item(), losses[off.argmax()].item())
    upstream = torch.linspace(0.5, 1.5, z.shape[0])
    dz, = torch.autograd.grad(loss, zs, upstream.to(device))
    want = upstream.double()[:, None] * grads
    info = torch.finfo(z.dtype)
    tol = upstream.double()[:, None] * temperature * n * eps * (1 if eps < 2.0 ** -50 else 4) + (info.eps / 2 + 2.0 ** -22) * want.abs() + info.tiny
    got, over = dz.double().cpu(), want.abs() > info.max  # T q and T p, rounded to infinity where the type ends before them
    assert torch.equal(got[over], want[over].sign() * float('inf'))
    off = (got - want)[~over].abs()
    assert (off <= tol[~over]).all(), off.max().item()
    for reduction in ('sum', 'mean'):
        some = kadconv.distill_loss(zs, t.to(device), i.to(device), temperature, reduction)
        rows = z.shape[0] if reduction == 'mean' else 1
        # the rows' own roundings and 64 additions: of their magnitudes, since losses may be negative (indexes that come again)
        assert abs(some.item() - loss.double().sum().item() / rows) <= 66 * 2.0 ** -24 * loss.double().abs().sum().item() / rows
        part, = torch.autograd.grad(some, zs)
        one, = torch.autograd.grad(kadconv.distill_loss(zs, t.to(device), i.to(device), temperature, 'none'), zs,
                                   torch.full((z.shape[0],), 1.0 / rows, device=device))
        torch.testing.assert_close(part, one, rtol=max(info.eps, 2.0 ** -21), atol=info.tiny)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('temperature', TEMPERATURES)
@pytest.mark.parametrize('shape', [(6, 16, 16), (3, 2, 2), (5, 7, 7), (40, 20, 4), (2, 300, 300), (2, 1000, 1000), (3, 1000, 30)],
                         ids=lambda s: 'x'.join(map(str, s)))
def test_every_temperature(shape, temperature, device):
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        check(*make(*shape, dtype, seed=shape[1]), temperature, device)


@pytest.mark.parametrize('device', DEVICES)
def test_an_equal_student(device):
    """Its loss is 0 and so is its gradient, at every temperature."""
    z, t, i = make(4, 30, 30, torch.float32, 3)
    z.scatter_(1, i, t + 1.0)
    t = z.gather(1, i)
    for temperature in TEMPERATURES[1:]:
        check(z, t, i, temperature, device)


@pytest.mark.parametrize('device', DEVICES)
def test_masked_classes(device):
    """Classes of -infinity have no weight: the entries cover all others."""
    z, t, i = make(4, 400, 12, torch.float32, 4)
    away = torch.ones(4, 400, dtype=torch.bool).scatter_(1, i, False)
    z[away] = -float('inf')
    for temperature in TEMPERATURES[1:]:
        check(z, t, i, temperature, device)


@pytest.mark.parametrize('device', DEVICES)
def test_indexes_that_come_again_or_do_not_count(device):
    z, t, i = make(5, 40, 40, torch.float32, 5)
    i[0, 1], i[1, 5:9] = i[0, 0], i[1, 4]
    i[2, 3:] = -1
    i[3, 0] = 1 << 40
    t[4, 20:] = -float('inf')
    for temperature in TEMPERATURES[1:]:
        check(z, t, i, temperature, device)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(1, 1500, 1024), (2, 5000, 900), (1, 40000, 256)], ids=lambda s: 'x'.join(map(str, s)))
def test_long_rows(shape):
    for masked in (False, True):
        z, t, i = make(*shape, torch.float32, 6)
        if masked:
            z[torch.ones(z.shape, dtype=torch.bool).scatter_(1, i, False)] = -float('inf')
        for temperature in (9.0, 1e3, 1e6):
            check(z, t, i, temperature, 'cuda')


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('temperature', [1.0, 20.0])
def test_not_finite_stays_in_its_row(temperature, device):
    nan, inf = float('nan'), float('inf')
    z, t, i = make(8, 12, 4, torch.float32, 7)
    z[1, 11], z[2], t[3, 1], z[4, 0] = nan, -inf, nan, inf
    i[5] = -1
    z[5] = nan
    z[6, i[6, 2]] = -inf
    zs = z.to(device).requires_grad_(True)
    loss = kadconv.distill_loss(zs, t.to(device), i.to(device), temperature, 'none')
    dz, = torch.autograd.grad(loss, zs, torch.ones_like(loss))
    loss, dz = loss.detach().cpu(), dz.cpu()
    assert torch.isfinite(loss[[0, 7]]).all() and torch.isfinite(dz[[0, 7]]).all()
    assert torch.isnan(loss[1:5]).all() and torch.isnan(dz[1:5]).any(1).all()
    assert loss[5] == 0 and not dz[5].any()
    assert loss[6] == inf and torch.isfinite(dz[6]).all() and dz[6, i[6, 2]] < 0
