"""AdamW from its formulas in 64 bits, 8-bit states as powers of two times integers, on the CPU."""
import math

import torch

SEG = 256


def mix32(x):
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(seed, step, first, count):
    """The 32 random bits of `count` values from place `first` of the state on."""
    key = mix32((mix32((seed + 0x9E3779B1) & 0xFFFFFFFF) + step) & 0xFFFFFFFF)
    i = torch.arange(first, first + count)
    return mix32(((i & 0xFFFFFFFF) * 0x9E3779B1 + (i >> 32) * 0x3C6EF373 + key) & 0xFFFFFFFF)


def hold(v, r16, positive):
    """(numbers held, scales) of v, 64-bit values a multiple of SEG long: |v| / scale = s q with q the step of
    e4m3 at that size (2^-9 below 2^-6) becomes floor(s + r16 / 65536) q."""
    most = v.reshape(-1, SEG).abs().amax(1)
    scale = most / 448
    y = v.abs() / torch.where(scale > 0, scale, torch.ones_like(scale)).repeat_interleave(SEG)
    q = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
    y = (torch.floor(y / q + r16.double() / 65536) * q).clamp(max=448.0)
    if positive:
        y = torch.where(v > 0, y.clamp(min=2.0 ** -9), y)
    return torch.where(v < 0, -y, y), scale


def step_of(y):
    """The step of e4m3 at numbers y."""
    return torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)


def update(p, g, m, v, t, lr, b1, b2, eps, wd):
    """(p, m, v) after step t, all in 64 bits."""
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    return p, m, v
