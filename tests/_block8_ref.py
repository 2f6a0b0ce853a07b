"""Rows in 8 bits and their products, from the definitions in 64 bits, and the bounds that the GPU's sums may be off by."""
import torch

EPS32 = 2.0 ** -24


def _two_to(p):
    return ((p.long() + 1023) << 52).view(torch.float64)


def held(v):
    """(codes as values, scale exponents) of rows [rows, K] in 64 bits: [rows, K] and [rows, blocks]."""
    v = v.detach().double()
    rows, k = v.shape
    codes, powers = torch.zeros_like(v), []
    for at in range(0, k, 128):
        part = v[:, at:at + 128]
        most = torch.where(torch.isfinite(part), part.abs(), torch.zeros_like(part)).amax(1, keepdim=True)
        mantissa, exponent = torch.frexp(most)       # in [0.5, 1) times 2^exponent; 448 = 0.875 * 2^9
        power = (exponent - 9 + (mantissa > 0.875).int()).clamp(min=-127)
        power = torch.where(most == 0, torch.zeros_like(power), power)
        y = part / _two_to(power)
        step = _two_to(torch.frexp(torch.where(torch.isfinite(y), y, torch.ones_like(y)).abs().clamp(min=2.0 ** -6)).exponent - 4)
        codes[:, at:at + 128] = torch.where(torch.isfinite(y), torch.round(y / step) * step, torch.full_like(y, float('nan')))
        powers.append(power)
    return codes, torch.cat(powers, 1)


def numbers(v):
    """The numbers that rows are held as."""
    codes, powers = held(v)
    return codes * _two_to(powers).repeat_interleave(128, 1)[:, :codes.shape[1]]


def product(a, b, dtype, bias=None):
    """a [M, K] b [N, K]^T of held numbers in 64 bits, and the bound of a result in dtype.

    A 32-bit sum of K terms in any order is off by K 2^-24 of its terms' magnitudes; that of the scaled blocks likewise.
    16-bit results: of each eight consecutive products seven at most are cut, each by less than 2^-13 of the largest."""
    y = a @ b.t()
    whole = a.abs() @ b.abs().t()
    tol = (a.shape[1] + 2) * EPS32 * whole
    if dtype != torch.float32:
        largest = torch.zeros_like(y)
        for at in range(0, a.shape[1], 8):
            m = torch.zeros_like(y)
            for k in range(at, min(at + 8, a.shape[1])):
                m = torch.maximum(m, a[:, k:k + 1].abs() * b[None, :, k].abs())
            largest += m
        tol = tol + 7 * 2.0 ** -13 * largest
    if bias is not None:
        y = y + bias.double()
        tol = tol + 2 * EPS32 * y.abs()
    return y, tol


def rounded(y, tol, dtype):
    """The bound, with the rounding of the result to dtype."""
    info = torch.finfo(dtype)
    return tol * (1 + info.eps) + info.eps / 2 * y.abs() + info.tiny * info.eps
