"""The operators of a head that is trained from a teacher and served, and the cases they are timed on: layer norm,
matrix products in 8 bits with a scale for each block of 128, and distillation from a teacher's top logits.

    own                 false: run() computes the operators' plain forms; true: it calls kadconv's kernels
    listed()            the fixed cases
    draw(rng)           one more case of the same ranges
    prepare(case, s)    inputs and state of a case on the GPU, made from the seed
    run(state)          one pass
    work(case)          bytes and flops that one pass cannot do without
    exact(case, s)      what run() returns, in 64 bits

Rows are the last axis of [rows, C], or the channels of each pixel of a channels-last map [N, C, H, W].

Layer norm, over the C values of a row:

    y = w (x - mean) / sqrt(var + eps) + b

Products: x [M, K] and w [N, K] are cut into blocks of 128 along K, the last one short.  A block's scale s is the
smallest power of two with max |x| <= 448 s (1 for a block of zeros), and its values are held as e4m3 numbers
c = round(x / s), to nearest, ties to even.

    y[m, n] = act(sum over blocks b of sx[m, b] sw[n, b] sum over k in b of cx[m, k] cw[n, k] + bias[n])

The gradients are such products too, each along its own sums: dx of dy and w along N, dw of dy and x along M; that of
the bias is the sum of dy.

Distillation: a teacher's top logits t_k at the classes i_k and a student's z over all V classes, at temperature T.
Entries whose index is not in [0, V) do not count, rows without entries are 0:

    p = softmax(t / T) over the entries, q = softmax(z / T), loss = T^2 sum_k p_k (log p_k - log q[i_k])

and its mean over the rows that have entries, or the rows' own losses.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
BYTES = {'f32': 4, 'f16': 2, 'bf16': 2}
LN_EPS = 1e-5
BLOCK = 128
MOST_LN = 128 * 1024 * 1024    # values of a normalised tensor
MOST_PRODUCT = 8192 * 4096 * 4096
MOST_SIDE = 8192 * 8192        # values of x, w or y
MOST_LOGITS = 4096 * 32768


def listed():
    return [
        # One image's coarse neck map at a served detector's smallest scale: launch latency is all.
        dict(name='ln_1x64x20x20_f16', op='ln', n=1, c=64, h=20, w=20, dtype='f16', affine='f32', wide=0),
        # The neck maps of the headline KAD-Conv layer.
        dict(name='ln_8x256x100x100_bf16', op='ln', n=8, c=256, h=100, w=100, dtype='bf16', affine='f32', wide=0),
        # Rows of a wide hidden layer, forward and gradients, parameters in 16 bits.
        dict(name='ln_train_16384x4096_bf16', op='ln_train', n=16384, c=4096, h=0, w=0, dtype='bf16', affine='bf16', wide=0),
        # A KAD-Conv branch's 86 channels on a ragged map, forward and gradients in fp32.
        dict(name='ln_train_3x86x67x41_f32', op='ln_train', n=3, c=86, h=67, w=41, dtype='f32', affine='f32', wide=0),
        # One row through a large layer whose weights are kept in 8 bits: the weights are read, no more.
        dict(name='lin8_1x8192x4096_bf16', op='lin8', m=1, n=8192, k=4096, dtype='bf16', bias=False, act='none'),
        # A detector's 1 x 1 convolution with SiLU at its middle scale, 16 x 50 x 50 pixels, weights kept.
        dict(name='lin8_40000x512x512_f16', op='lin8', m=40000, n=512, k=512, dtype='f16', bias=True, act='silu'),
        # A branch's 86 channels to 43 over a ragged map's pixels, fp32.
        dict(name='lin8_8241x43x86_f32', op='lin8', m=8241, n=43, k=86, dtype='f32', bias=True, act='none'),
        # Forward and gradients of a head's 1 x 1 convolution, fp16.
        dict(name='lin8_train_20000x128x256_f16', op='lin8_train', m=20000, n=128, k=256, dtype='f16', bias=True, act='none'),
        # Forward and gradients of a large hidden layer: the largest.
        dict(name='lin8_train_8192x4096x4096_bf16', op='lin8_train', m=8192, n=4096, k=4096, dtype='bf16', bias=False, act='none'),
        # The cells of one image's coarse map, 20 classes, the teacher's 4 best: latency.
        dict(name='distill_1x20x20x20_f32', op='distill', n=1, v=20, h=20, w=20, k=4, dtype='f32', index='i64', temp=2.0, reduction='mean'),
        # The 16 bins of the four sides of 16 x 8400 anchor cells, all of the teacher's.
        dict(name='distill_537600x16_f16', op='distill', n=537600, v=16, h=0, w=0, k=16, dtype='f16', index='i32', temp=4.0, reduction='none'),
        # Rows over a large vocabulary, the teacher's 64 best, as a file of them holds them: in 32 bits.
        dict(name='distill_4096x32768_bf16', op='distill', n=4096, v=32768, h=0, w=0, k=64, dtype='bf16', index='i32', temp=1.0, reduction='mean'),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(('ln', 'ln_train', 'lin8', 'lin8', 'lin8_train', 'distill', 'distill'))
    dtype = rng.choice(('f32', 'f16', 'bf16'))
    wide = 2 if dtype == 'f32' else 1
    if op in ('ln', 'ln_train'):
        affine = rng.choice(('f32', dtype))
        # of 2 or 3 values a gradient is rounding alone
        least = 2 if op == 'ln' else 16
        while True:
            c = _log_int(rng, least, 8192)
            if rng.random() < 0.5:
                n, h, w = rng.randint(1, 16), _log_int(rng, 1, 200), _log_int(rng, 1, 200)
            else:
                n, h, w = _log_int(rng, 1, 200_000), 0, 0
            if n * max(1, h * w) * c <= MOST_LN // wide // (2 if op == 'ln_train' else 1):
                break
        # wide: x is a slice of a wider buffer's channels
        return dict(op=op, n=n, c=c, h=h, w=w, dtype=dtype, affine=affine, wide=rng.choice((0, 0, 0, 8, 13)))
    if op in ('lin8', 'lin8_train'):
        while True:
            m, n, k = _log_int(rng, 1, 60_000), _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)
            product = m * n * k * (3 if op == 'lin8_train' else 1)
            if product <= MOST_PRODUCT and max(m * n, m * k, n * k) <= MOST_SIDE // wide:
                break
        act = rng.choice(('none', 'relu', 'silu')) if op == 'lin8' else 'none'
        return dict(op=op, m=m, n=n, k=k, dtype=dtype, bias=rng.random() < 0.5, act=act)
    while True:
        v = _log_int(rng, 2, 150_000)
        if rng.random() < 0.5 and v <= 1024:
            n, h, w = rng.randint(1, 16), _log_int(rng, 1, 160), _log_int(rng, 1, 160)
        else:
            n, h, w = _log_int(rng, 1, 500_000), 0, 0
        k = _log_int(rng, 1, min(v, 256))
        rows = n * max(1, h * w)
        if rows * max(v, 4 * k) <= MOST_LOGITS // wide // 2:
            break
    return dict(op=op, n=n, v=v, h=h, w=w, k=k, dtype=dtype, index=rng.choice(('i32', 'i64')), temp=rng.choice((1.0, 2.0, 4.0)),
                reduction=rng.choice(('mean', 'none')))


def _as_map(v, case):
    """[rows, C] as [rows, C], or as a channels-last map [N, C, H, W]."""
    return v if not case['h'] else v.view(case['n'], case['h'], case['w'], -1).permute(0, 3, 1, 2)


def _as_rows(v, case):
    return v if not case['h'] else v.permute(0, 2, 3, 1).reshape(case['n'] * case['h'] * case['w'], -1)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dtype = DTYPES[case['dtype']]

    def normal(*size):
        return torch.randn(*size, generator=gen, device='cuda')

    s = dict(case=case)
    if case['op'] in ('ln', 'ln_train'):
        c, wide = case['c'], case['wide']
        rows = case['n'] * max(1, case['h'] * case['w'])
        # each channel with its own location and spread, each row with its own size
        x = (normal(rows, c + wide) * (0.5 + torch.rand(c + wide, generator=gen, device='cuda')) + 0.5 * normal(c + wide)) * torch.exp(0.5 * normal(rows, 1))
        s['x'] = _as_map(x.to(dtype), case)
        if wide:
            s['x'] = s['x'][:, :c]
        affine = DTYPES[case['affine']]
        s['weight'] = (1.0 + 0.2 * normal(c)).to(affine)
        s['bias'] = (0.2 * normal(c)).to(affine)
        if case['op'] == 'ln_train':
            s['dy'] = _as_map(normal(rows, c).to(dtype), case)
            s['x'] = s['x'].detach()
            for name in ('x', 'weight', 'bias'):
                s[name].requires_grad_(True)
        return s
    if case['op'] in ('lin8', 'lin8_train'):
        m, n, k = case['m'], case['n'], case['k']
        # activations: some channels are far larger than others, some values zero
        s['x'] = (normal(m, k) * torch.exp(normal(k)) * (torch.rand(m, k, generator=gen, device='cuda') > 0.1)).to(dtype)
        weight = (normal(n, k) / math.sqrt(k)).to(dtype)
        s['bias'] = 0.1 * normal(n) if case['bias'] else None
        if case['op'] == 'lin8':  # the weights that a served program keeps, in 8 bits
            s['codes'], s['scales'] = _held(weight.float())
            if own:
                s['kept'] = _kadconv().quantize8(weight)
            return s
        s['weight'] = weight
        s['dy'] = (0.1 * normal(m, n) * torch.exp(0.5 * normal(m, 1))).to(dtype)
        for name in ('x', 'weight', 'bias'):
            if s[name] is not None:
                s[name].requires_grad_(True)
        return s
    v, k = case['v'], case['k']
    rows = case['n'] * max(1, case['h'] * case['w'])
    teacher = 2.0 * normal(rows, v)
    z = (0.7 * teacher + normal(rows, v)).to(dtype)
    s['logits'] = _as_map(z, case).requires_grad_(True)
    top = torch.topk(teacher, k, dim=1)
    t, index = top.values.to(dtype), top.indices
    # one entry in 20 is left out (a shorter list), and one row in 16 has none at all (cells that teach nothing)
    out = torch.rand(rows, k, generator=gen, device='cuda') < 0.05
    out[:, 0] = False
    out |= torch.rand(rows, 1, generator=gen, device='cuda') < 1.0 / 16
    out[0] = False
    index = torch.where(out, torch.full_like(index, -1), index)
    index = index.to(torch.int32 if case['index'] == 'i32' else torch.int64)
    s['t'], s['index'] = (_as_map(a, case).contiguous() for a in (t, index))
    if case['reduction'] == 'none':  # each row's own weight
        s['dy'] = torch.rand(*((case['n'], case['h'], case['w']) if case['h'] else (rows,)), generator=gen, device='cuda')
    else:  # 1, or what a program that trains in fp16 scales its loss by
        s['dy'] = torch.tensor(2.0 ** int(math.log2(rows)) if case['dtype'] == 'f16' else 1.0, device='cuda')
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
        K = _kadconv()
        dim = 1 if case.get('h') else -1
        if case['op'] == 'ln':
            return K.layer_norm(s['x'], s['weight'], s['bias'], LN_EPS, dim=dim)
        if case['op'] == 'ln_train':
            y = K.layer_norm(s['x'], s['weight'], s['bias'], LN_EPS, dim=dim)
            return (y.detach(), *torch.autograd.grad(y, (s['x'], s['weight'], s['bias']), s['dy']))
        if case['op'] == 'lin8':
            return K.linear8(s['x'], s['kept'], s['bias'], act=None if case['act'] == 'none' else case['act'])
        if case['op'] == 'lin8_train':
            y = K.linear8(s['x'], s['weight'], s['bias'])
            return (y.detach(), *torch.autograd.grad(y, [t for t in (s['x'], s['weight'], s['bias']) if t is not None], s['dy']))
        loss = K.distill_loss(s['logits'], s['t'], s['index'], temperature=case['temp'], reduction=case['reduction'], dim=dim)
        return loss.detach(), torch.autograd.grad(loss, s['logits'], s['dy'])[0]
    with torch.no_grad():
        if case['op'] in ('ln', 'ln_train'):
            return _plain_norm(s)
        if case['op'] == 'lin8':
            return _plain_served(s)
        if case['op'] == 'lin8_train':
            return _plain_trained(s)
        return _plain_distill(s)


def _plain_norm(s):
    case = s['case']
    x = _as_rows(s['x'], case).float()
    w, b = s['weight'].float(), s['bias'].float()
    x = x - x.mean(dim=1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + LN_EPS)
    xhat = x * rstd
    y = _as_map((xhat * w + b).to(s['x'].dtype), case)
    if case['op'] == 'ln':
        return y
    dy = _as_rows(s['dy'], case).float()
    dw = (dy * xhat).sum(dim=0).to(s['weight'].dtype)
    db = dy.sum(dim=0).to(s['bias'].dtype)
    dy = dy * w
    dx = rstd * (dy - dy.mean(dim=1, keepdim=True) - xhat * (dy * xhat).mean(dim=1, keepdim=True))
    return y, _as_map(dx.to(s['x'].dtype), case), dw, db


def _held(v):
    """v [rows, K] in 32 bits as (e4m3 codes [rows, blocks, 128], scales [rows, blocks, 1])."""
    rows, k = v.shape
    blocks = -(-k // BLOCK)
    v = torch.nn.functional.pad(v, (0, blocks * BLOCK - k)).view(rows, blocks, BLOCK)
    bits = v.abs().amax(dim=2, keepdim=True).view(torch.int32)
    # 448 is 1.75 * 2^8: the exponent less 8, and one more where the mantissa is over 1.75
    power = (bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000).int()
    power = torch.where(bits == 0, torch.zeros_like(power), power.clamp(min=-127))
    # 2^-power, and 2^power from twice as much, which is never below the smallest normal number
    return (v * ((127 - power) << 23).view(torch.float32)).to(torch.float8_e4m3fn), 0.5 * ((128 + power) << 23).view(torch.float32)


def _number(held, k):
    codes, scales = held
    return (codes.float() * scales).reshape(codes.shape[0], -1)[:, :k]


def _product(a, b):
    """a [M, K] b [N, K]^T, both held in 8 bits along K, in 32 bits."""
    k = a.shape[1]
    return torch.matmul(_number(_held(a), k), _number(_held(b), k).t())


def _plain_served(s):
    case = s['case']
    k = case['k']
    z = torch.matmul(_number(_held(s['x'].float()), k), _number((s['codes'], s['scales']), k).t())
    if s['bias'] is not None:
        z = z + s['bias']
    if case['act'] == 'relu':
        z = torch.where(z > 0, z, torch.zeros_like(z))
    elif case['act'] == 'silu':
        z = z / (1.0 + torch.exp(-z))
    return z.to(s['x'].dtype)


def _plain_trained(s):
    x, w, dy, dtype = s['x'].float(), s['weight'].float(), s['dy'].float(), s['x'].dtype
    y = _product(x, w)
    if s['bias'] is not None:
        y = y + s['bias']
    dx = _product(dy, w.t().contiguous())
    dw = _product(dy.t().contiguous(), x.t().contiguous())
    out = (y.to(dtype), dx.to(dtype), dw.to(dtype))
    return out if s['bias'] is None else (*out, dy.sum(dim=0))


def _plain_distill(s):
    case, temp = s['case'], s['case']['temp']
    z = _as_rows(s['logits'], case).float() / temp
    t, index = _as_rows(s['t'], case).float() / temp, _as_rows(s['index'], case).long()
    counts = (index >= 0) & (index < case['v'])
    index = index.clamp(0, case['v'] - 1)
    live = counts.any(dim=1, keepdim=True)
    e = torch.where(counts, torch.exp(t - torch.where(counts, t, torch.full_like(t, -math.inf)).amax(dim=1, keepdim=True)), torch.zeros_like(t))
    total = torch.where(live, e.sum(dim=1, keepdim=True), torch.ones_like(t[:, :1]))
    p = e / total
    most = z.amax(dim=1, keepdim=True)
    ez = torch.exp(z - most)
    sum_z = ez.sum(dim=1, keepdim=True)
    log_q = torch.gather(z, 1, index) - most - torch.log(sum_z)
    loss = temp * temp * torch.where(p > 0, p * (torch.log(p) - log_q), torch.zeros_like(p)).sum(dim=1)
    grad = torch.where(live, ez / sum_z, torch.zeros_like(ez)).scatter_add_(1, index, -p)
    if case['reduction'] == 'none':
        grad = grad * (temp * s['dy'].reshape(-1, 1))
        loss = loss.view(s['dy'].shape)
    else:
        share = 1.0 / live.sum().float()
        loss, grad = loss.sum() * share, grad * (temp * share * s['dy'])
    return loss, _as_map(grad.to(s['logits'].dtype), case)


def work(case):
    b = BYTES[case['dtype']]
    if case['op'] in ('ln', 'ln_train'):
        x = case['n'] * max(1, case['h'] * case['w']) * case['c']
        maps, ops = (2, 8) if case['op'] == 'ln' else (4, 24)
        return dict(bytes=maps * x * b + maps * case['c'] * BYTES[case['affine']], flops=ops * x)
    if case['op'] in ('lin8', 'lin8_train'):
        m, n, k = case['m'], case['n'], case['k']
        if case['op'] == 'lin8':  # the weights in 8 bits, with a byte's scale for each 128
            return dict(bytes=b * m * (n + k) + n * k * (1 + 1 / BLOCK) + 4 * n * case['bias'], flops=2 * m * n * k)
        return dict(bytes=2 * b * (m * n + m * k + n * k) + 8 * n * case['bias'], flops=6 * m * n * k)
    rows = case['n'] * max(1, case['h'] * case['w'])
    per_row = 2 * b * case['v'] + case['k'] * (b + (4 if case['index'] == 'i32' else 8)) + (8 if case['reduction'] == 'none' else 0)
    return dict(bytes=rows * per_row, flops=rows * (8 * case['v'] + 12 * case['k']))


def _two_to(power):
    """2^power in 64 bits, from its own bits."""
    return ((power.long() + 1023) << 52).view(torch.float64)


def _exact_held(v):
    """The numbers that v [rows, K] is held as, in 64 bits."""
    k = v.shape[1]
    out = torch.zeros_like(v)
    for at in range(0, k, BLOCK):
        part = v[:, at:at + BLOCK]
        mantissa, exponent = torch.frexp(part.abs().max(dim=1, keepdim=True).values)
        # in [0.5, 1) times 2^exponent; 448 = 0.875 * 2^9
        power = (exponent - 9 + (mantissa > 0.875).int()).clamp(min=-127)
        scale = torch.where(mantissa == 0, torch.ones_like(mantissa), _two_to(power))
        part = part / scale
        step = _two_to(torch.frexp(part.abs().clamp(min=2.0 ** -6)).exponent - 4)  # three bits behind the first
        out[:, at:at + BLOCK] = torch.round(part / step) * step * scale
    return out


def exact(case, seed):
    """The definitions in 64 bits: the norm's and the loss's gradients by differentiating them."""
    s = prepare(case, seed)
    if case['op'] in ('ln', 'ln_train'):
        x = _as_rows(s['x'].detach(), case).double().requires_grad_(case['op'] == 'ln_train')
        w, b = (s[name].detach().double().requires_grad_(case['op'] == 'ln_train') for name in ('weight', 'bias'))
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        y = (x - mean) / (var + LN_EPS) ** 0.5 * w + b
        if case['op'] == 'ln':
            return _as_map(y, case)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), _as_rows(s['dy'], case).double())
        return _as_map(y.detach(), case), _as_map(dx, case), dw, db
    if case['op'] in ('lin8', 'lin8_train'):
        x = s['x'].detach().double()
        bias = 0.0 if s['bias'] is None else s['bias'].detach().double()
        if case['op'] == 'lin8':
            w = (s['codes'].double() * s['scales'].double()).reshape(case['n'], -1)[:, :case['k']]
            z = _exact_held(x) @ w.t() + bias
            return z if case['act'] == 'none' else z.clamp(min=0.0) if case['act'] == 'relu' else z * torch.sigmoid(z)
        w, dy = s['weight'].detach().double(), s['dy'].double()
        y = _exact_held(x) @ _exact_held(w).t() + bias
        dx = _exact_held(dy) @ _exact_held(w.t().contiguous()).t()
        dw = _exact_held(dy.t().contiguous()) @ _exact_held(x.t().contiguous()).t()
        return (y, dx, dw) if s['bias'] is None else (y, dx, dw, dy.sum(dim=0))
    z = _as_rows(s['logits'].detach(), case).double().requires_grad_(True)
    t, index = _as_rows(s['t'], case).double() / case['temp'], _as_rows(s['index'], case).long()
    counts = (index >= 0) & (index < case['v'])
    live = counts.any(dim=1)
    t = t.masked_fill(~counts, -math.inf)
    p = torch.softmax(t.masked_fill(~live[:, None], 0.0), dim=1) * counts
    log_q = torch.log_softmax(z / case['temp'], dim=1).gather(1, index.clamp(0, case['v'] - 1))
    rows = case['temp'] ** 2 * (torch.special.xlogy(p, p) - p * log_q).sum(dim=1)
    loss = rows.view(s['dy'].shape) if case['reduction'] == 'none' else rows.sum() / live.sum()
    grad, = torch.autograd.grad(loss, z, s['dy'].double())
    return loss.detach(), _as_map(grad, case)
