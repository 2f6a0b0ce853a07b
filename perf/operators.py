"""The training operators and the cases they are timed on: group norm with an activation on channels-last
maps, forward and with its gradients, and the AdamW step over a network's tensors with 32- and 8-bit states.

    own                 false: run() computes the operators' plain forms; true: it calls kadconv's kernels
    listed()            the fixed cases
    draw(rng)           one more case of the same ranges
    prepare(case, s)    inputs and state of a case on the GPU, made from the seed
    run(state)          one pass
    work(case)          bytes and flops that one pass cannot do without
    exact(case, s)      what run() returns, in 64 bits

The operators, for a map x [N, C, H, W] in G groups of D = C / G channels:

    z = w (x - mean) / sqrt(var + eps) + b     mean and var over the H W D values of an (image, group)
    y = act(z)                                 act: none, relu, silu

and for a parameter p with gradient g at step t:

    m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2
    p <- (1 - lr wd) p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

8-bit states hold m and u = sqrt(v) as e4m3 numbers times one fp32 scale (the largest magnitude / 448)
for each 256 elements, rounded stochastically: the 16 random bits of an element come from a hash of
(seed, t, element).  A u that is not zero is held as the smallest positive number at least.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
BYTES = {'f32': 4, 'f16': 2, 'bf16': 2}
GN_EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 1e-2
FIRST_STEP = 100
SEED = 7          # of the stochastic rounding
SEG = 256         # a tensor's state begins at a multiple of SEG elements; an 8-bit scale holds for SEG of them
MOST_MAP = 16 * 128 * 200 * 200
MOST_PARAMS = 64_000_000


def listed():
    return [
        # One image's coarse neck map at a served detector's smallest scale: launch latency is all.
        dict(name='gn_1x64x20x20_f16', op='gn', n=1, c=64, g=8, h=20, w=20, dtype='f16', act='silu', wide=0),
        # The neck map of the headline KAD-Conv layer, 32 groups, in fp16.
        dict(name='gn_8x256x100x100_f16', op='gn', n=8, c=256, g=32, h=100, w=100, dtype='f16', act='silu', wide=0),
        # A KAD-Conv branch's 86 channels in two groups of 43, ragged map, fp32.
        dict(name='gn_3x86x67x41_f32', op='gn', n=3, c=86, g=2, h=67, w=41, dtype='f32', act='relu', wide=0),
        # The finest map of a batch of 800 x 800 images: the largest.
        dict(name='gn_16x128x200x200_bf16', op='gn', n=16, c=128, g=16, h=200, w=200, dtype='bf16', act='silu', wide=0),
        # Forward and gradients of a small ragged head map, fp32.
        dict(name='gn_train_2x48x13x17_f32', op='gn_train', n=2, c=48, g=6, h=13, w=17, dtype='f32', act='silu', wide=0),
        # Forward and gradients at the middle neck scale, fp16.
        dict(name='gn_train_16x512x50x50_f16', op='gn_train', n=16, c=512, g=32, h=50, w=50, dtype='f16', act='silu', wide=0),
        # Forward and gradients of the headline map, bf16.
        dict(name='gn_train_8x256x100x100_bf16', op='gn_train', n=8, c=256, g=32, h=100, w=100, dtype='bf16', act='silu', wide=0),
        # A detector head's dozen tensors, fp32: latency.
        dict(name='adamw_head_f32', op='adamw', tensors=12, total=150_000, spread=6.0, dtype='f32', master=False),
        # All of a small detector's parameters (as many tensors and values as KAD-CNet-S has, most of them tiny), fp32.
        dict(name='adamw_net_f32', op='adamw', tensors=2944, total=6_968_486, spread=11.0, dtype='f32', master=False),
        # A large model's share of one GPU: bf16 parameters and gradients, fp32 masters and states.
        dict(name='adamw_64m_bf16', op='adamw', tensors=60, total=MOST_PARAMS, spread=6.0, dtype='bf16', master=True),
        # The small detector again, states in 8 bits.
        dict(name='adamw8_net_f32', op='adamw8', tensors=2944, total=6_968_486, spread=11.0, dtype='f32', master=False),
        # The large share again with 8-bit states and no masters.
        dict(name='adamw8_64m_bf16', op='adamw8', tensors=60, total=MOST_PARAMS, spread=6.0, dtype='bf16', master=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(('gn', 'gn', 'gn_train', 'gn_train', 'adamw', 'adamw8'))
    dtype = rng.choice(('f32', 'f16', 'bf16'))
    if op in ('adamw', 'adamw8'):
        total = _log_int(rng, 1000, MOST_PARAMS if dtype != 'f32' else MOST_PARAMS // 2)
        tensors = _log_int(rng, 1, min(3000, total // 10))
        return dict(op=op, tensors=tensors, total=total, spread=rng.uniform(0.0, 11.0), dtype=dtype,
                    master=dtype != 'f32' and rng.random() < 0.5)
    most = MOST_MAP // (2 if dtype == 'f32' else 1) // (3 if op == 'gn_train' else 1)
    while True:
        n, h, w = rng.randint(1, 16), _log_int(rng, 1, 200), _log_int(rng, 1, 200)
        g = rng.choice((1, 2, 3, 4, 8, 16, 32))
        c = g * _log_int(rng, 1, 1024 // g)
        if 64 <= n * c * h * w <= most and c * h * w // g >= 4:  # of 2 or 3 values a gradient is rounding alone
            break
    # wide: x is a slice of a map with that many channels more (a concat's buffer); its pieces stay 16-byte aligned
    wide = 32 if c % 8 == 0 and rng.random() < 0.25 else 0
    # a ReLU's gradient jumps at 0, where two correct 32-bit sums may be on either side: forward only
    act = rng.choice(('none', 'relu', 'silu') if op == 'gn' else ('none', 'silu'))
    return dict(op=op, n=n, c=c, g=g, h=h, w=w, dtype=dtype, act=act, wide=wide)


def _sizes(case):
    """The tensors' sizes: relative sizes spread evenly over exp(0 .. spread), in a fixed shuffled order."""
    t = case['tensors']
    rel = [math.exp(case['spread'] * (i + 0.5) / t) for i in range(t)]
    unit = case['total'] / sum(rel)
    sizes = [max(1, int(round(r * unit))) for r in rel]
    random.Random(t).shuffle(sizes)
    return sizes


def _map(n, c, h, w, dtype, gen, wide=0, loc=None, scale=None):
    """A channels-last map of normal values with each channel's own location and scale."""
    v = torch.randn(n, h, w, c + wide, generator=gen, device='cuda')
    if loc is not None:
        v = v * scale + loc
    return v.to(dtype)[..., :c].permute(0, 3, 1, 2)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dtype = DTYPES[case['dtype']]
    if case['op'] in ('gn', 'gn_train'):
        n, c, h, w = case['n'], case['c'], case['h'], case['w']
        ct = c + case['wide']
        loc = 0.5 * torch.randn(ct, generator=gen, device='cuda')
        scale = 0.5 + torch.rand(ct, generator=gen, device='cuda')
        s = dict(case=case, x=_map(n, c, h, w, dtype, gen, case['wide'], loc, scale),
                 weight=1.0 + 0.2 * torch.randn(c, generator=gen, device='cuda'),
                 bias=0.2 * torch.randn(c, generator=gen, device='cuda'))
        if case['op'] == 'gn_train':
            s['dy'] = _map(n, c, h, w, dtype, gen)
            for k in ('x', 'weight', 'bias'):
                s[k].requires_grad_(True)
        return s
    sizes = _sizes(case)
    segs = torch.tensor([-(-k // SEG) for k in sizes])
    total = int(segs.sum()) * SEG
    # gaps between a tensor's end and the next multiple of SEG hold zeros
    first = torch.cumsum(segs, 0) - segs
    left = torch.repeat_interleave(torch.tensor(sizes) + first * SEG, segs) - torch.arange(total // SEG) * SEG
    live = (torch.arange(SEG, device='cuda') < left.cuda()[:, None]).reshape(-1)

    def normal(size):
        return torch.randn(total, generator=gen, device='cuda') * size * live

    master = normal(0.05)
    p = master.to(dtype) if dtype != torch.float32 else master
    # gradients of sizes that differ from segment to segment, one in ten zero (a ReLU's dead inputs)
    size = torch.exp(torch.randn(total // SEG, 1, generator=gen, device='cuda')).expand(-1, SEG).reshape(-1)
    alive = torch.rand(total, generator=gen, device='cuda') > 0.1
    g = (normal(1e-3) * size * alive).to(dtype)
    m = normal(3e-4) * size
    u = (normal(1e-3).abs() + 1e-5 * live) * size
    s = dict(case=case, t=FIRST_STEP, p=p, g=g, sizes=sizes)
    if case['master']:
        s['master'] = master
    if case['op'] == 'adamw':
        s['state'] = dict(exp_avg=m, exp_avg_sq=u * u)
    else:
        s['state'] = {}
        for name, v in (('exp_avg', m), ('exp_avg_sq_root', u)):
            scale = v.reshape(-1, SEG).abs().amax(1) / 448.0
            unit = torch.where(scale > 0, scale, torch.ones_like(scale)).repeat_interleave(SEG)
            s['state'][name] = (v / unit).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
            s['state'][name + '_scale'] = scale
    if case['master']:
        s['state']['master'] = master
    begin = [SEG * int(f) for f in first]
    s['params'] = [p[b:b + k] for b, k in zip(begin, sizes)]
    s['grads'] = [g[b:b + k] for b, k in zip(begin, sizes)]
    if own:  # the plan of the tensors that the program keeps, over the same state
        s['plan'] = _kadconv().AdamWPlan(s['params'], s['grads'], state_bits=8 if case['op'] == 'adamw8' else 32,
                                         master_weights=case['master'], state=s['state'], seed=SEED)
    return s


def _kadconv():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'kad-conv_amd')
    if at not in sys.path:
        sys.path.insert(0, at)
    import kadconv
    return kadconv


def run(s):
    case = s['case']
    if own:
        if case['op'] == 'gn':
            return _kadconv().group_norm_act(s['x'], case['g'], s['weight'], s['bias'], GN_EPS, _act_name(case))
        if case['op'] == 'gn_train':
            y = _kadconv().group_norm_act(s['x'], case['g'], s['weight'], s['bias'], GN_EPS, _act_name(case))
            return (y.detach(), *torch.autograd.grad(y, (s['x'], s['weight'], s['bias']), s['dy']))
        s['t'] += 1
        s['plan'].step(s['t'], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY)
        return _returned(s)
    with torch.no_grad():
        if case['op'] == 'gn':
            return _plain_norm(s)[0]
        if case['op'] == 'gn_train':
            return _plain_norm_train(s)
        s['t'] += 1
        if case['op'] == 'adamw':
            _plain_adamw(s)
        else:
            _plain_adamw8(s)
        return _returned(s)


def _act_name(case):
    return None if case['act'] == 'none' else case['act']


def _returned(s):
    return dict(p=s['p'], **s['state'])


def _plain_norm(s):
    """The normalised map and what its gradient uses, each [N, P, G, D] in 32 bits."""
    case = s['case']
    n, c, g, h, w = (case[k] for k in ('n', 'c', 'g', 'h', 'w'))
    x = s['x'].permute(0, 2, 3, 1).reshape(n, h * w, g, c // g).float()
    mean = x.mean(dim=(1, 3), keepdim=True)
    x = x - mean
    rstd = 1.0 / torch.sqrt((x * x).mean(dim=(1, 3), keepdim=True) + GN_EPS)
    xhat = x * rstd
    z = xhat * s['weight'].reshape(g, c // g) + s['bias'].reshape(g, c // g)
    y = z
    if case['act'] == 'relu':
        y = torch.where(z > 0, z, torch.zeros_like(z))
    elif case['act'] == 'silu':
        y = z / (1.0 + torch.exp(-z))
    return _to_map(y, s), xhat, rstd, z


def _to_map(v, s):
    case = s['case']
    return v.reshape(case['n'], case['h'], case['w'], case['c']).to(s['x'].dtype).permute(0, 3, 1, 2)


def _plain_norm_train(s):
    case = s['case']
    n, c, g, h, w = (case[k] for k in ('n', 'c', 'g', 'h', 'w'))
    y, xhat, rstd, z = _plain_norm(s)
    dz = s['dy'].permute(0, 2, 3, 1).reshape(n, h * w, g, c // g).float()
    if case['act'] == 'relu':
        dz = torch.where(z > 0, dz, torch.zeros_like(dz))
    elif case['act'] == 'silu':
        sig = 1.0 / (1.0 + torch.exp(-z))
        dz = dz * sig * (1.0 + z * (1.0 - sig))
    dw = (dz * xhat).sum(dim=(0, 1)).reshape(c)
    db = dz.sum(dim=(0, 1)).reshape(c)
    dz = dz * s['weight'].reshape(g, c // g)
    s1 = dz.mean(dim=(1, 3), keepdim=True)
    s2 = (dz * xhat).mean(dim=(1, 3), keepdim=True)
    dx = rstd * (dz - s1 - xhat * s2)
    return y, _to_map(dx, s), dw, db


def _plain_update(s, m, u):
    """p from its moment m and the root u of its second one; the 32-bit p is the master's where there is one."""
    t = s['t']
    wide = s['state']['master'] if s['case']['master'] else s['p'].float()
    denom = u * (1.0 / math.sqrt(1.0 - BETA2 ** t)) + ADAM_EPS
    new = wide * (1.0 - LR * DECAY) - (LR / (1.0 - BETA1 ** t)) * m / denom
    if s['case']['master']:
        wide.copy_(new)
    s['p'].copy_(new)


def _plain_adamw(s):
    st, g = s['state'], s['g'].float()
    st['exp_avg'].mul_(BETA1).add_(g * (1.0 - BETA1))
    st['exp_avg_sq'].mul_(BETA2).add_(g * g * (1.0 - BETA2))
    _plain_update(s, st['exp_avg'], torch.sqrt(st['exp_avg_sq']))


M32 = 0xFFFFFFFF


def _mix(x):
    """32 bits in, 32 well mixed bits out (in 64-bit integers or Python's): the odd factors are fractions of
    the square roots of 2 and 3."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & M32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & M32
    return x ^ (x >> 16)


def _random_bits(count, t, device):
    key = _mix((_mix((SEED + 0x9E3779B1) & M32) + t) & M32)
    i = torch.arange(count, device=device)
    return _mix(((i & M32) * 0x9E3779B1 + (i >> 32) * 0x3C6EF373 + key) & M32)


def _held(v, r16, positive):
    """v [segments, SEG] as (e4m3 codes, scales): its magnitude over the scale, cut after r16 / 65536 of a step is added."""
    most = v.abs().amax(dim=1, keepdim=True)
    scale = most * (1.0 / 448.0)
    y = (v.abs() * torch.where(most > 0, 448.0 / most, torch.zeros_like(most))).clamp(max=448.0)
    fine = (y * 2.0 ** 29).to(torch.int64)                        # below 2^-6 steps are 2^-9 apart
    coarse = y.view(torch.int32).to(torch.int64) - (120 << 23)    # above, the exponent and three bits
    code = (torch.where(y < 2.0 ** -6, fine, coarse) + (r16 << 4)) >> 20
    if positive:
        code = torch.where(v > 0, code.clamp(min=1), code)
    else:
        code = torch.where(v < 0, code + 128, code)
    return code.to(torch.uint8).view(torch.float8_e4m3fn).reshape(-1), scale.reshape(-1)


def _plain_adamw8(s):
    st, g = s['state'], s['g'].float()
    m = (st['exp_avg'].float().reshape(-1, SEG) * st['exp_avg_scale'][:, None]).reshape(-1)
    u = (st['exp_avg_sq_root'].float().reshape(-1, SEG) * st['exp_avg_sq_root_scale'][:, None]).reshape(-1)
    m = m * BETA1 + g * (1.0 - BETA1)
    u = torch.sqrt(u * u * BETA2 + g * g * (1.0 - BETA2))
    _plain_update(s, m, u)
    r = _random_bits(g.numel(), s['t'], g.device).reshape(-1, SEG)
    for name, v, bits in (('exp_avg', m, r & 0xFFFF), ('exp_avg_sq_root', u, r >> 16)):
        codes, scales = _held(v.reshape(-1, SEG), bits, name != 'exp_avg')
        st[name].copy_(codes)
        st[name + '_scale'].copy_(scales)


def work(case):
    if case['op'] in ('gn', 'gn_train'):
        x = case['n'] * case['c'] * case['h'] * case['w']
        maps, ops = (2, 14) if case['op'] == 'gn' else (4, 40)
        return dict(bytes=maps * x * BYTES[case['dtype']] + 8 * case['c'] * (maps // 2), flops=ops * x)
    k, b = sum(_sizes(case)), BYTES[case['dtype']]
    per = 3 * b + (8 if case['master'] else 0)               # p (read only where there is no master), g, p written
    per -= b if case['master'] else 0
    per += 16 if case['op'] == 'adamw' else 4 + 16.0 / SEG   # both states, read and written
    return dict(bytes=per * k, flops=(16 if case['op'] == 'adamw' else 60) * k)


def exact(case, seed):
    """The definitions in 64 bits: the norm's gradients by differentiating its definition, the 8-bit
    numbers from powers of two."""
    s = prepare(case, seed)
    if case['op'] in ('gn', 'gn_train'):
        n, c, g = case['n'], case['c'], case['g']
        x = s['x'].detach().double().requires_grad_(case['op'] == 'gn_train')
        w = s['weight'].detach().double().requires_grad_(case['op'] == 'gn_train')
        b = s['bias'].detach().double().requires_grad_(case['op'] == 'gn_train')
        parts = x.reshape(n, g, -1)
        var, mean = torch.var_mean(parts, dim=2, correction=0, keepdim=True)
        z = ((parts - mean) / (var + GN_EPS) ** 0.5).reshape(x.shape) * w.reshape(1, c, 1, 1) + b.reshape(1, c, 1, 1)
        y = z if case['act'] == 'none' else z.clamp(min=0.0) if case['act'] == 'relu' else z * torch.sigmoid(z)
        if case['op'] == 'gn':
            return y
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), s['dy'].double()))
    t = FIRST_STEP + 1
    st, p, g = s['state'], s['p'].double(), s['g'].double()
    if case['op'] == 'adamw':
        m, v = st['exp_avg'].double(), st['exp_avg_sq'].double()
    else:
        m = st['exp_avg'].double() * st['exp_avg_scale'].double().repeat_interleave(SEG)
        v = (st['exp_avg_sq_root'].double() * st['exp_avg_sq_root_scale'].double().repeat_interleave(SEG)) ** 2
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g * g - v)
    p = st['master'].double() if case['master'] else p
    p = p - LR * (DECAY * p + (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS))
    out = dict(p=p)
    if case['master']:
        out['master'] = p
    if case['op'] == 'adamw':
        return dict(out, exp_avg=m, exp_avg_sq=v)
    r = _random_bits(g.numel(), t, g.device)
    for name, v, bits in (('exp_avg', m, r % 65536), ('exp_avg_sq_root', v.sqrt(), r // 65536)):
        most = v.reshape(-1, SEG).abs().max(dim=1).values
        unit = torch.where(most > 0, most / 448, torch.ones_like(most)).repeat_interleave(SEG)
        y = v.abs() / unit
        power = torch.floor(torch.log2(y.clamp(min=2.0 ** -6)))
        step = torch.exp2(power - 3)
        y = torch.floor(y / step + bits.double() / 65536) * step
        y = y.clamp(max=448.0)
        if name != 'exp_avg':
            y = torch.where(v > 0, y.clamp(min=2.0 ** -9), y)
        out[name] = torch.where(v < 0, -y, y)
        out[name + '_scale'] = most / 448
    return out
