"""AdamWPlan and AdamW on the GPU against the formulas in 64 bits."""
import copy
import io

import pytest
import torch

import kadconv
from tests import _adamw_ref as R

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEV = 'cuda'
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [1, 3, 4, 255, 256, 257, 1000, 4095, 4096, 4097, 9001, 22]
# 32-bit roundings that a value passes through in one step: products and sums of m, v and p, the root, the
# quotient; half a step each, relative to the largest term
ROUNDINGS = 16
EPS32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tensors(sizes, dtype, seed, unaligned=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        v = torch.randn(n, generator=g) * 0.05
        if unaligned:  # a view one value into its storage
            out.append(torch.empty(n + 1, dtype=dtype, device=DEV)[1:].copy_(v.to(dtype)))
        else:
            out.append(v.to(dtype).to(DEV))
    return out


def gradients(params, seed):
    g = torch.Generator().manual_seed(seed)
    out = []
    for p in params:
        v = torch.randn(p.shape, generator=g) * 1e-2 * torch.exp(torch.randn((), generator=g))
        v[torch.rand(p.shape, generator=g) < 0.1] = 0
        out.append(torch.empty_like(p).copy_(v))
    return out


def check_step(p, p0, g, m0, v0, t, dtype, what):
    """One value's step from what was there before it, within the roundings."""
    lr, (b1, b2), eps, wd = HYPER['lr'], HYPER['betas'], HYPER['eps'], HYPER['weight_decay']
    want, m, v = R.update(p0, g, m0, v0, t, lr, b1, b2, eps, wd)
    moved = (want - p0 * (1 - lr * wd)).abs()
    # m is a difference of terms that may cancel: its error is relative to them, and p moves by lr / root of it
    terms = b1 * m0.abs() + (1 - b1) * g.abs()
    slack = torch.where(m.abs() > 0, terms / m.abs().clamp(min=1e-300), torch.zeros_like(m)) * moved
    tol = half_step(dtype) * want.abs() + ROUNDINGS * EPS32 * (p0.abs() + moved + slack)
    if dtype != F32:
        tol = tol + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (p.double().cpu() - want).abs()
    assert (off <= tol).all(), f'{what}: {(off / tol).max().item():.3g} times its bound'
    return m, v, terms


@pytest.mark.parametrize('unaligned', [False, True], ids=['aligned', 'unaligned'])
@pytest.mark.parametrize('dtype,master', [(F32, False), (F16, False), (BF16, False), (F16, True), (BF16, True)],
                         ids=['f32', 'f16', 'bf16', 'f16_master', 'bf16_master'])
@pytest.mark.parametrize('bits', [32, 8])
def test_steps(bits, dtype, master, unaligned):
    params = tensors(SIZES, dtype, 0, unaligned)
    grads = [torch.empty_like(p) if not unaligned else torch.empty(p.numel() + 1, dtype=dtype, device=DEV)[1:]
             for p in params]
    plan = kadconv.AdamWPlan(params, grads, state_bits=bits, master_weights=master, seed=5)
    scale = torch.tensor(0.5, device=DEV)
    for t in (1, 2, 3, 7):
        for g, new in zip(grads, gradients(params, 10 + t)):
            g.copy_(new)
        before = {k: v.clone() for k, v in plan.state.items()}
        p_before = [p.double().cpu() for p in params]
        plan.step(t, grad_scale=scale, **HYPER)
        torch.cuda.synchronize()
        for i, (p, g, n) in enumerate(zip(params, grads, SIZES)):
            a = plan.offsets[i]
            segs = -(-n // R.SEG)
            rows = slice(a // R.SEG, a // R.SEG + segs)

            def held(state, name):
                v = state[name][a:a + segs * R.SEG].double().cpu()
                return v * state[name + '_scale'][rows].double().cpu().repeat_interleave(R.SEG)

            if bits == 32:
                m0, v0 = (before[k][a:a + n].double().cpu() for k in ('exp_avg', 'exp_avg_sq'))
            else:
                m0, v0 = held(before, 'exp_avg')[:n], held(before, 'exp_avg_sq_root')[:n] ** 2
            p0 = before['master'][a:a + n].double().cpu() if master else p_before[i]
            gi = 0.5 * g.double().cpu()
            if master:
                w = plan.state['master'][a:a + n]
                m, v, terms = check_step(w, p0, gi, m0, v0, t, F32, f'step {t} master {i}')
                assert torch.equal(p, w.to(dtype))
            else:
                m, v, terms = check_step(p, p0, gi, m0, v0, t, dtype, f'step {t} tensor {i}')
            if bits == 32:
                got_m, got_v = (plan.state[k][a:a + n].double().cpu() for k in ('exp_avg', 'exp_avg_sq'))
                assert ((got_m - m).abs() <= 4 * EPS32 * terms + 1e-44).all()
                assert ((got_v - v).abs() <= 4 * EPS32 * v + 1e-44).all()
                continue
            r = R.random_bits(5, t, a, segs * R.SEG)
            for name, want, bits16 in (('exp_avg', m, r & 0xFFFF), ('exp_avg_sq_root', v.sqrt(), r >> 16)):
                full = torch.zeros(segs * R.SEG, dtype=torch.float64)
                full[:n] = want
                y, s = R.hold(full, bits16, name != 'exp_avg')
                got = plan.state[name][a:a + segs * R.SEG].double().cpu()
                got_s = plan.state[name + '_scale'][rows].double().cpu()
                # m is a sum of terms that may cancel: its roundings are relative to them, as above
                size = torch.zeros(segs * R.SEG, dtype=torch.float64)
                size[:n] = terms if name == 'exp_avg' else want
                assert ((got_s - s).abs() <= 8 * EPS32 * size.reshape(-1, R.SEG).amax(1) / 448).all()
                # 32 bits may fall on the other side of a border: then one step off, and hardly ever
                assert ((got - y).abs() <= R.step_of(y) * 1.001).all()
                assert int((got != y).sum()) <= 1, (name, int((got != y).sum()))
                assert not got[n:].any()
                if name != 'exp_avg':
                    assert (got[:n][want > 0] > 0).all()


def test_layouts_and_gaps():
    """Channels-last weights, an empty tensor, one without a gradient: stepped in their memory's order, or left."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn(16, 8, 3, 3, generator=g).to(DEV).contiguous(memory_format=torch.channels_last)
    t = torch.randn(5, 7, generator=g).to(DEV).t()
    empty, still = torch.empty(0, 4, device=DEV), torch.randn(300, generator=g).to(DEV)
    params = [w, empty, still, t]
    grads = [torch.randn(p.shape, generator=g).to(DEV) for p in params]
    grads = [torch.empty_like(p).copy_(d) for p, d in zip(params, grads)]
    grads[2] = None
    before = [p.clone() for p in params]
    plan = kadconv.AdamWPlan(params, grads)
    plan.step(1, **HYPER)
    assert torch.equal(still, before[2]) and not plan.part(plan.state['exp_avg'], 2).any()
    for i in (0, 3):
        m = plan.part(plan.state['exp_avg'], i)
        assert m.shape == params[i].shape and m.stride() == params[i].stride()
        d = grads[i].double().cpu()
        check_step(params[i], before[i].double().cpu(), d, 0 * d, 0 * d, 1, F32, f'tensor {i}')
        torch.testing.assert_close(m, grads[i] * 0.1, rtol=1e-6, atol=0)


def test_values_not_finite():
    for bits in (32, 8):
        for bad in (float('nan'), float('inf')):
            p = torch.zeros(1024, device=DEV)
            g = torch.full((1024,), 1e-2, device=DEV)
            plan = kadconv.AdamWPlan([p], [g], state_bits=bits)
            g[300] = bad
            plan.step(1, **HYPER)
            hit = torch.zeros(1024, dtype=torch.bool, device=DEV)
            hit[300] = True
            assert torch.isnan(p[hit]).all() and torch.isfinite(p[~hit]).all()
            g.fill_(1e-2)
            plan.step(2, **HYPER)
            if bits == 8:  # the segment is lost, and no other
                hit[256:512] = True
            assert torch.isnan(p[hit]).all() and torch.isfinite(p[~hit]).all()


def test_8_bit_states_of_any_size():
    """Gradients from 1e-30 (held as zeros: no scale could be a normal float) to 1e15, and all zeros."""
    p = torch.zeros(256 * 6, device=DEV)
    g = torch.zeros(6, 256, device=DEV)
    for k, size in enumerate((0.0, 1e-36, 1e-20, 1e-8, 1.0, 1e15)):
        g[k] = size * torch.linspace(0.5, 1, 256, device=DEV)
    g = g.reshape(-1)
    plan = kadconv.AdamWPlan([p], [g], state_bits=8)
    for t in (1, 2, 3):
        plan.step(t, **HYPER)
    assert torch.isfinite(p).all()
    scales = plan.state['exp_avg_sq_root_scale']
    assert not scales[:2].any() and (scales[2:] > 0).all()
    assert torch.equal(p[:256], torch.zeros_like(p[:256]))
    # a steady gradient moves by lr a step, whatever its size (eps aside)
    assert ((p[4 * 256:].abs() / (3 * HYPER['lr']) - 1).abs() < 0.2).all()


def test_8_bit_moments_follow_steady_gradients():
    """Rounded to nearest, m would stop two thirds of the way to a steady gradient that is small beside the
    segment's largest, and sqrt(v) would never leave its first value: rounded stochastically, their means over
    many values arrive.  After 60 steps of beta1 = 0.9, m = g (1 - 0.9^60) and beta2 = 0.99 leaves
    v = g^2 (1 - 0.99^60).  A held value is off its mean by less than a step (1/8 of it), each step's errors
    fading with beta: the mean over 4000 values by under 0.125 * sqrt(60 / 4000) = 1.6 %, and the root's
    curvature adds (1/8)^2 / 2 of it at most."""
    n = 4096
    p = torch.zeros(n, device=DEV)
    g = torch.full((n,), 0.37e-2, device=DEV)
    g[::256] = 1e-2
    plan = kadconv.AdamWPlan([p], [g], state_bits=8)
    for t in range(1, 61):
        plan.step(t, lr=1e-3, betas=(0.9, 0.99))
    rest = torch.ones(n, dtype=torch.bool, device=DEV)
    rest[::256] = False
    m = plan.state['exp_avg'].float() * plan.state['exp_avg_scale'].repeat_interleave(256)
    u = plan.state['exp_avg_sq_root'].float() * plan.state['exp_avg_sq_root_scale'].repeat_interleave(256)
    assert abs(m[rest].mean().item() / (0.37e-2 * (1 - 0.9 ** 60)) - 1) < 0.025
    assert abs(u[rest].mean().item() / (0.37e-2 * (1 - 0.99 ** 60) ** 0.5) - 1) < 0.025


def test_long_tensor():
    """A tensor of many chunks, the last one ragged."""
    n = 3_000_007
    p, g = torch.zeros(n, device=DEV), torch.empty(n, device=DEV).normal_()
    plan = kadconv.AdamWPlan([p], [g])
    plan.step(1, **HYPER)
    check_step(p, torch.zeros(n, dtype=torch.float64), g.double().cpu(), *(torch.zeros(n, dtype=torch.float64),) * 2, 1, F32,
               'long')


def test_refusals():
    p, g = torch.zeros(8, 4, device=DEV), torch.zeros(8, 4, device=DEV)
    plan = kadconv.AdamWPlan([p], [g])
    for bad, err in (([], ValueError), ([g.half()], TypeError), ([g.cpu()], TypeError), ([g[:4]], ValueError),
                     ([torch.zeros(4, 8, device=DEV).t()], ValueError)):
        with pytest.raises(err):
            plan.set_grads(bad)
    with pytest.raises(ValueError, match='share memory'):
        kadconv.AdamWPlan([p, p[:2]], [g, g[:2]])
    with pytest.raises(ValueError, match='dense'):
        kadconv.AdamWPlan([p[:, ::2]], [g[:, ::2]])
    with pytest.raises(TypeError):
        kadconv.AdamWPlan([p, p.half()], [g, g.half()])
    with pytest.raises(TypeError):
        kadconv.AdamWPlan([p.double()], [g.double()])
    with pytest.raises(ValueError, match='16-bit'):
        kadconv.AdamWPlan([p], [g], master_weights=True)
    with pytest.raises(ValueError, match='state'):
        kadconv.AdamWPlan([p], [g], state=dict(exp_avg=g))
    with pytest.raises(ValueError, match='exp_avg'):
        kadconv.AdamWPlan([p], [g], state=dict(exp_avg=torch.zeros(32, device=DEV), exp_avg_sq=torch.zeros(256, device=DEV)))
    with pytest.raises(ValueError, match='step'):
        plan.step(0)
    with pytest.raises(ValueError, match='grad_scale'):
        plan.step(1, grad_scale=torch.ones(2, device=DEV))
    with pytest.raises(TypeError):
        plan.step(1, lr=torch.tensor(1e-3, device=DEV))
    with pytest.raises(ValueError, match='step'):
        plan.step(torch.tensor(1, dtype=torch.int32, device=DEV))


def test_kept_weights_follow_a_step():
    """What the package keeps by a parameter's version (packed weights) is made anew after a step."""
    m = kadconv.Conv1x1SiLU(16, 16).to(DEV).half().eval()
    x = torch.randn(1, 16, 8, 8, device=DEV, dtype=F16)
    m(x)
    params = list(m.parameters())
    plan = kadconv.AdamWPlan(params, [torch.ones_like(p) for p in params])
    plan.step(1, lr=0.1)
    fresh = copy.deepcopy(m)
    fresh._packed = {}
    assert torch.equal(m(x), fresh(x))


def _net(seed, dtype=F32):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Conv2d(8, 16, 3, padding=1), kadconv.GroupNormAct(4, 16),
                               torch.nn.Conv2d(16, 4, 1)).to(DEV, dtype).to(memory_format=torch.channels_last)


def _losses(net, opt, steps, dtype=F32, seed=3):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(4, 8, 12, 12, generator=g).to(DEV, dtype).contiguous(memory_format=torch.channels_last)
    y = torch.randn(4, 4, 12, 12, generator=g).to(DEV, dtype)
    out = []
    for _ in range(steps):
        opt.zero_grad()
        loss = (net(x).float() - y.float()).square().mean()
        loss.backward()
        opt.step()
        out.append(loss.item())
    return out


def test_optimizer_follows_torch():
    """Twenty steps as torch's AdamW makes them (fp32; the losses differ by the gradients' roundings, which Adam
    does not enlarge while no gradient is tiny: 1e-3)."""
    a, b = _net(0), _net(0)
    la = _losses(a, kadconv.AdamW(a.parameters(), lr=1e-2, weight_decay=0.1), 20)
    lb = _losses(b, torch.optim.AdamW(b.parameters(), lr=1e-2, weight_decay=0.1), 20)
    assert la[-1] < 0.9 * la[0]
    torch.testing.assert_close(torch.tensor(la), torch.tensor(lb), rtol=1e-3, atol=0)


@pytest.mark.parametrize('dtype,master', [(F32, False), (BF16, True)], ids=['f32', 'bf16_master'])
def test_optimizer_8_bits_trains_alike(dtype, master):
    """States in 8 bits reach the loss that 32 bits reach, give or take a tenth of the way."""
    a, b = _net(1, dtype), _net(1, dtype)
    la = _losses(a, kadconv.AdamW(a.parameters(), lr=1e-2, state_bits=8, master_weights=master), 60, dtype)
    lb = _losses(b, kadconv.AdamW(b.parameters(), lr=1e-2, master_weights=master), 60, dtype)
    assert la[-1] < lb[-1] + 0.1 * (lb[0] - lb[-1])


@pytest.mark.parametrize('bits', [32, 8])
def test_optimizer_state_dict(bits):
    """A run saved and taken up again goes on as the run itself does, bit for bit."""
    net = _net(2, BF16)
    opt = kadconv.AdamW([dict(params=net[0].parameters(), lr=1e-2), dict(params=net[1:].parameters(), weight_decay=0.0)],
                        state_bits=bits, master_weights=True, seed=9)
    _losses(net, opt, 3, BF16)
    file = io.BytesIO()
    torch.save((net.state_dict(), opt.state_dict()), file)
    file.seek(0)
    saved_net, saved_opt = torch.load(file, weights_only=True)
    other = _net(7, BF16)
    other.load_state_dict(saved_net)
    opt2 = kadconv.AdamW([dict(params=other[0].parameters()), dict(params=other[1:].parameters())], state_bits=bits,
                         master_weights=True)
    opt2.load_state_dict(saved_opt)
    assert _losses(net, opt, 3, BF16) == _losses(other, opt2, 3, BF16)
    for p, q in zip(net.parameters(), other.parameters()):
        assert torch.equal(p, q)


def test_optimizer_state_dict_refusals():
    net = _net(3)
    opt = kadconv.AdamW(net.parameters(), state_bits=8)
    _losses(net, opt, 1)
    saved = opt.state_dict()
    plain = torch.nn.Sequential(*[copy.deepcopy(m) for m in net]).to(memory_format=torch.contiguous_format)
    with pytest.raises(ValueError, match='strides'):
        kadconv.AdamW(plain.parameters(), state_bits=8).load_state_dict(saved)
    del saved['state'][0]
    with pytest.raises(ValueError, match='some'):
        kadconv.AdamW(net.parameters(), state_bits=8).load_state_dict(saved)


def test_optimizer_scale_and_missing_gradients():
    net = _net(4)
    opt = kadconv.AdamW(net.parameters(), lr=1e-2)
    net(torch.randn(1, 8, 6, 6, device=DEV)).square().mean().backward()
    net[2].bias.grad = None
    before = [p.detach().clone() for p in net.parameters()]
    opt.step(grad_scale=torch.zeros((), device=DEV))   # no gradient left: only the decay moves
    for i, (p, q) in enumerate(zip(net.parameters(), before)):
        want = q if i == len(before) - 1 else q * (1 - 1e-2 * 1e-2)
        torch.testing.assert_close(p.detach(), want, rtol=3e-7, atol=0)


def test_optimizer_captured():
    """Steps captured once and replayed with other gradients and rates, against an optimizer that is not."""
    a, b = tensors(SIZES, F32, 20), tensors(SIZES, F32, 20)
    lr = torch.tensor(1e-2, device=DEV)
    oa = kadconv.AdamW(a, lr=lr, capturable=True, state_bits=8, seed=4)
    ob = kadconv.AdamW(b, lr=1e-2, state_bits=8, seed=4)
    for p, q, g in zip(a, b, gradients(a, 21)):
        p.grad, q.grad = g, g.clone()
    oa.step()
    ob.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step()
    for k in range(4):
        for p, q, g in zip(a, b, gradients(a, 30 + k)):
            p.grad.copy_(g)
            q.grad.copy_(g)
        lr.fill_(1e-2 / (k + 1))
        ob.param_groups[0]['lr'] = lr.item()
        graph.replay()
        ob.step()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            torch.testing.assert_close(p, q, rtol=1e-6, atol=1e-9)
    assert oa.param_groups[0]['step'].item() == ob.param_groups[0]['step'] == 5
