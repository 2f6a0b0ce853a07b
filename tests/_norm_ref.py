"""group_norm_act and its gradients from their formulas in 64 bits, on the CPU, with the bounds that
32-bit sums and one rounding to the output's type may be off by."""
import torch

EPS32 = 2.0 ** -24
# Roundings of 32 bits that one value passes through in a row, at most: the serial part of a sum (a few
# hundred values of a thread at the sizes tested, whose errors add as their root), its tree, and the
# element-wise formula.  The sums' own bound is taken relative to the sum of magnitudes.
STEPS = 64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def act_and_slope(z, act):
    if act is None:
        return z, torch.ones_like(z)
    if act == 'relu':
        return z.clamp(min=0), (z > 0).to(z.dtype)
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s))


def reference(x, groups, weight, bias, eps, act, dy=None):
    """dict of y and, with dy, dx, dw, db, in 64 bits, and for each of them 'tol_...': the absolute bound
    for a result of x's dtype (dw, db: of 32 bits)."""
    N, C, H, W = x.shape
    D = C // groups
    x64 = x.detach().double().cpu()
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight.detach().double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if bias is None else bias.detach().double().cpu()
    v = x64.permute(0, 2, 3, 1).reshape(N, H * W, groups, D)
    mean = v.mean(dim=(1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = (v - mean) * rstd
    w, b = w.view(groups, D), b.view(groups, D)
    z = w * xhat + b
    y, slope = act_and_slope(z, act)

    def as_map(t):
        return t.reshape(N, H, W, C).permute(0, 3, 1, 2)

    # error of xhat: of the mean (relative to the values' size) times rstd, and of the formula
    dxhat = STEPS * EPS32 * (v.abs().amax(dim=(1, 3), keepdim=True) * rstd + xhat.abs() + 1)
    dz_err = w.abs() * dxhat + STEPS * EPS32 * (z.abs() + b.abs())
    out = dict(y=as_map(y), tol_y=as_map(half_step(x.dtype) * y.abs() + 1.2 * dz_err + torch.finfo(x.dtype).tiny),
               mean=mean.reshape(N, groups), rstd=rstd.reshape(N, groups))
    if dy is None:
        return out
    g = dy.detach().double().cpu().permute(0, 2, 3, 1).reshape(N, H * W, groups, D)
    dz = g * slope
    # |act''| <= 1.1 (silu); relu's jump is kept away from by the tests' values
    e_dz = STEPS * EPS32 * dz.abs() + g.abs() * dz_err * (1.1 if act == 'silu' else 0)
    out['dw'] = (dz * xhat).sum(dim=(0, 1)).reshape(C)
    out['db'] = dz.sum(dim=(0, 1)).reshape(C)
    out['tol_dw'] = (STEPS * EPS32 * (dz * xhat).abs() + e_dz * xhat.abs() + dz.abs() * dxhat).sum(dim=(0, 1)).reshape(C)
    out['tol_db'] = (STEPS * EPS32 * dz.abs() + e_dz).sum(dim=(0, 1)).reshape(C)
    wdz, e = w * dz, w.abs() * e_dz
    s1 = wdz.mean(dim=(1, 3), keepdim=True)
    s2 = (wdz * xhat).mean(dim=(1, 3), keepdim=True)
    e1 = (STEPS * EPS32 * wdz.abs() + e).mean(dim=(1, 3), keepdim=True)
    e2 = (STEPS * EPS32 * (wdz * xhat).abs() + e * xhat.abs() + wdz.abs() * dxhat).mean(dim=(1, 3), keepdim=True)
    dx = rstd * (wdz - s1 - xhat * s2)
    e_dx = rstd * (e + e1 + xhat.abs() * e2 + dxhat * s2.abs()) + \
        STEPS * EPS32 * rstd * (wdz.abs() + s1.abs() + (xhat * s2).abs())
    out['dx'] = as_map(dx)
    out['tol_dx'] = as_map(half_step(x.dtype) * dx.abs() + e_dx + torch.finfo(x.dtype).tiny)
    return out


def assert_within(got, ref, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), f'{what}: not finite'
    off = (got - ref).abs()
    bad = off > tol
    assert not bad.any(), f'{what}: {(off[bad] / tol[bad]).max().item():.3g} times its bound, {int(bad.sum())} values'
