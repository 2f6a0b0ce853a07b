"""What the autograd node and the optimizer's table in C++ have to keep of a torch program's rules."""
import copy

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.checkpoint import checkpoint

import kadconv
from kadconv import ops
from tests import _adamw_ref as R

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def _case(seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, 24, 9, 7, generator=g).to(DEV).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    w = (1 + 0.1 * torch.randn(24, generator=g)).to(DEV).requires_grad_(True)
    b = (0.1 * torch.randn(24, generator=g)).to(DEV).requires_grad_(True)
    return x, w, b


def f(x, w, b):
    return kadconv.group_norm_act(x, 3, w, b, act='silu')


def test_checkpoint_gives_the_same_gradients():
    x, w, b = _case()
    want = torch.autograd.grad(f(x, w, b).square().sum(), (x, w, b))
    for reentrant in (False, True):
        y = checkpoint(f, x, w, b, use_reentrant=reentrant)
        x.grad = w.grad = b.grad = None
        y.square().sum().backward()
        assert all(torch.equal(p.grad, g) for p, g in zip((x, w, b), want))


def test_saved_tensor_hooks_see_the_inputs():
    x, w, b = _case()
    want = torch.autograd.grad(f(x, w, b).sum(), (x, w, b))
    with torch.autograd.graph.save_on_cpu():
        y = f(x, w, b)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y.sum(), (x, w, b)), want))


def test_changed_input_is_noticed():
    x, w, b = _case()
    y = f(x, w, b)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_second_backward_and_retained_graph():
    x, w, b = _case()
    y = f(x, w, b)
    dy = torch.ones_like(y)
    first = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    again = torch.autograd.grad(y, (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    with pytest.raises(RuntimeError, match='second time'):
        torch.autograd.grad(y, (x, w, b), dy)


def test_no_graph_where_none_is_wanted():
    x, w, b = _case()
    with torch.no_grad():
        assert not f(x, w, b).requires_grad
    with torch.inference_mode():
        assert f(x, w, b).is_inference()
    assert not f(x.detach(), w.detach(), b.detach()).requires_grad
    assert f(x.detach(), w.detach(), b).grad_fn.name() == 'GroupNormActBackward'


def test_first_order_gradient_with_create_graph():
    """The gradient's value is there under create_graph; only its own gradient is refused."""
    x, w, b = _case()
    want = torch.autograd.grad(f(x, w, b).sum(), x)[0]
    got = torch.autograd.grad(f(x, w, b).sum(), x, create_graph=True)[0]
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        got.sum().backward()


def test_forward_mode_is_refused():
    x, w, b = _case()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            f(dual, w, b)


def test_backward_arguments_are_checked():
    x, w, b = (t.detach() for t in _case())
    y, mean, rstd = kadconv.ops.group_norm_act_forward(x, 3, w, b, 1e-5, 'silu')
    args = lambda **k: kadconv.ops.group_norm_act_backward(*{**dict(
        dy=y, x=x, num_groups=3, weight=w, bias=b, mean=mean, rstd=rstd, eps=1e-5, act='silu'), **k}.values())
    args()
    for bad in (dict(mean=mean.double()), dict(rstd=rstd[:1]), dict(mean=mean.cpu()), dict(dy=y[:1]), dict(dy=y.cpu()),
                dict(num_groups=6)):
        with pytest.raises(ValueError):
            args(**bad)
    with pytest.raises(TypeError):
        args(dy=y.half())


def _train(net, opt, steps):
    g = torch.Generator().manual_seed(5)
    for _ in range(steps):
        x = torch.randn(2, 8, 6, 6, generator=g).to(DEV)
        opt.zero_grad()
        net(x).square().mean().backward()
        opt.step()


@pytest.mark.parametrize('bits', [32, 8])
def test_copied_optimizer_goes_on(bits):
    net = torch.nn.Sequential(torch.nn.Conv2d(8, 16, 3), kadconv.GroupNormAct(4, 16), torch.nn.Conv2d(16, 4, 1)).to(DEV)
    opt = kadconv.AdamW(net.parameters(), lr=1e-2, state_bits=bits)
    _train(net, opt, 3)
    net2, opt2 = copy.deepcopy((net, opt))
    _train(net, opt, 2)
    _train(net2, opt2, 2)
    assert all(torch.equal(p, q) for p, q in zip(net.parameters(), net2.parameters()))


def test_moved_and_added_parameters_are_noticed():
    net = torch.nn.Conv2d(8, 4, 1).to(DEV)
    opt = kadconv.AdamW(net.parameters())
    _train(net, opt, 1)
    opt.param_groups[0]['params'].append(torch.nn.Parameter(torch.zeros(3, device=DEV)))
    with pytest.raises(RuntimeError, match='gained'):
        opt.step()
    opt.param_groups[0]['params'].pop()
    net.weight.data = net.weight.data.clone()
    with pytest.raises(RuntimeError, match='moved'):
        opt.step()


def test_gradients_of_other_strides():
    """A gradient laid out otherwise than its parameter is brought to its order."""
    p = torch.nn.Parameter(torch.zeros(6, 4, 3, 3, device=DEV).contiguous(memory_format=torch.channels_last))
    q = torch.nn.Parameter(torch.zeros(6, 4, 3, 3, device=DEV))
    g = torch.randn(6, 4, 3, 3, device=DEV)
    p.grad, q.grad = g, g.clone()
    kadconv.AdamW([p]).step()
    kadconv.AdamW([q]).step()
    assert torch.equal(p, q) and p.any()


def _formula_32_bits(g, codes, scales, t, seed):
    """One 8-bit step in 32-bit torch operations, each product and sum rounded by itself."""
    b1, b2 = 0.9, 0.999
    seg = 256
    m = (codes[0].float().reshape(-1, seg) * scales[0][:, None]).reshape(-1) * b1 + g * (1 - b1)
    u = (codes[1].float().reshape(-1, seg) * scales[1][:, None]).reshape(-1)
    u = torch.sqrt(u * u * b2 + g * g * (1 - b2))
    r = R.random_bits(seed, t, 0, g.numel()).to(g.device)
    out = []
    for v, bits, positive in ((m, r & 0xFFFF, False), (u, r >> 16, True)):
        most = v.reshape(-1, seg).abs().amax(1, keepdim=True)
        y = (v.reshape(-1, seg).abs() * torch.where(most > 0, 448.0 / most, torch.zeros_like(most))).clamp(max=448.0).reshape(-1)
        near, far = (y * 2.0 ** 29).long(), y.view(torch.int32).long() - (120 << 23)
        c = (torch.where(y < 2.0 ** -6, near, far) + (bits << 4)) >> 20
        c = torch.where(v > 0, c.clamp(min=1), c) if positive else torch.where(v < 0, c + 128, c)
        out.append((c.to(torch.uint8), (most * (1.0 / 448.0)).reshape(-1)))
    return out


def test_8_bit_codes_are_those_of_the_formula_in_32_bits():
    """Held numbers equal, code by code, what 32-bit operations and integer arithmetic on their bits give: a
    reciprocal that is off by a step in 1 / top * 448 may move one in a million of them to the next code."""
    n = 256 * 4096
    gen = torch.Generator(device=DEV).manual_seed(1)
    p = torch.randn(n, generator=gen, device=DEV)
    g = torch.empty(n, device=DEV)
    plan = kadconv.AdamWPlan([p], [g], state_bits=8, seed=11)
    for t in (1, 2, 3):
        size = torch.exp(3 * torch.randn(n, generator=gen, device=DEV))
        g.copy_(torch.randn(n, generator=gen, device=DEV) * 1e-3 * size * (torch.rand(n, generator=gen, device=DEV) > 0.1))
        st = plan.state
        before = [st['exp_avg'].clone(), st['exp_avg_sq_root'].clone()], [st['exp_avg_scale'].clone(), st['exp_avg_sq_root_scale'].clone()]
        want = _formula_32_bits(g, *before, t, 11)
        plan.step(t)
        for (c, s), name in zip(want, ('exp_avg', 'exp_avg_sq_root')):
            got = st[name].view(torch.uint8)
            torch.testing.assert_close(st[name + '_scale'], s, rtol=2.0 ** -22, atol=0)
            same = (got == c) | ((got & 127) == 0) & ((c & 127) == 0)   # zeros of either sign
            assert int((~same).sum()) <= 2, (t, name, int((~same).sum()))


def test_steps_of_more_than_the_last_cache_holds():
    """Over 256 MB a step: loads go past the caches; the result is that of the same values in two plans."""
    n = 12_000_007
    gen = torch.Generator(device=DEV).manual_seed(2)
    p = torch.randn(n, generator=gen, device=DEV)
    g = torch.randn(n, generator=gen, device=DEV)
    half = 4096 * 1400
    q = [p[:half].clone(), p[half:].clone()]
    whole = kadconv.AdamWPlan([p], [g])
    parts = [kadconv.AdamWPlan([v], [w.clone()]) for v, w in zip(q, (g[:half], g[half:]))]
    for t in (1, 2):
        whole.step(t)
        for plan in parts:
            plan.step(t)
    assert torch.equal(p, torch.cat(q))
    for name in ('exp_avg', 'exp_avg_sq'):
        assert torch.equal(whole.state[name][:n], torch.cat([parts[0].state[name][:half], parts[1].state[name][:n - half]]))


def test_captured_step_outlives_its_table():
    """A step captured, an eager step by gradients elsewhere (which lays another table out), then replays."""
    n = 5000
    p, q = torch.nn.Parameter(torch.zeros(n, device=DEV)), torch.nn.Parameter(torch.zeros(n, device=DEV))
    g = torch.randn(n, device=DEV)
    opt, ref = kadconv.AdamW([p], lr=1e-2, capturable=True), kadconv.AdamW([q], lr=1e-2, capturable=True)
    p.grad, q.grad = g, g
    opt.step(), ref.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(3):
        other = torch.randn(n, device=DEV)
        p.grad, q.grad = other.clone(), other.clone()
        opt.step(), ref.step()
        junk = [torch.full((64,), -1, dtype=torch.int32, device=DEV) for _ in range(50)]   # of the size of a table
        g.normal_()
        q.grad = g
        graph.replay()
        ref.step()
        torch.cuda.synchronize()
        del junk
        assert torch.equal(p, q), k


def test_steps_on_another_stream():
    """A plan made on one stream and stepped on another, its gradients changed at once."""
    n = 3_000_000
    p, q = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    grads = [torch.randn(n, device=DEV) for _ in range(4)]
    plan, ref = kadconv.AdamWPlan([p], [grads[0]]), kadconv.AdamWPlan([q], [grads[0]])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for t, g in enumerate(grads, 1):
        plan.set_grads([g])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            plan.step(t, lr=1e-2)
    torch.cuda.current_stream().wait_stream(side)
    for t, g in enumerate(grads, 1):
        ref.set_grads([g])
        ref.step(t, lr=1e-2)
    assert torch.equal(p, q)


def test_group_norm_refusals_on_the_gpu():
    """The GPU path's checks are those of the CPU path: the same errors for the same arguments."""
    x = torch.randn(2, 12, 3, 3, device=DEV)
    w = torch.ones(12, device=DEV)
    cases = [((x[0], 3), ValueError, 'N, C, H, W'), ((x, 5), ValueError, 'divide'), ((x, 0), ValueError, 'divide'),
             ((x, 3, None, None, 1e-5, 'gelu'), ValueError, 'act'), ((x, 3, torch.ones(11, device=DEV)), ValueError, 'shape'),
             ((x, 3, torch.ones(1, 12, device=DEV)), ValueError, 'shape'), ((x, 3, w, None, -1.0), ValueError, 'eps'),
             ((x, 3, w, None, float('nan')), ValueError, 'eps'), ((x, 3, w.half()), TypeError, 'float32'),
             ((x.half(), 3, w.half(), w), TypeError, 'share'), ((x, 3, None, w.cpu()), ValueError, 'one device')]
    for args, error, words in cases:
        with pytest.raises(error, match=words):
            kadconv.group_norm_act(*args)
        if words != 'one device':
            with pytest.raises(error, match=words):
                kadconv.group_norm_act(*(a.cpu() if isinstance(a, torch.Tensor) else a for a in args))


def test_sizes_past_an_int_are_refused():
    """Before anything of such a size is allocated: the map is one value, expanded."""
    x = torch.zeros(1, 1, 1, 1, dtype=torch.float16, device=DEV)
    stat = torch.zeros(1, 1, device=DEV)
    for big in (x.expand((1 << 32) + 1, 1, 1, 1), x.expand(1, 1, (1 << 32) + 1, 1), x.expand(1, 1 << 32, 1, 1)):
        for call in (lambda: kadconv.group_norm_act(big, 1),
                     lambda: ops.group_norm_act_forward(big, 1, None, None, 1e-5, None),
                     lambda: ops.group_norm_act_backward(big, big, 1, None, None, stat, stat, 1e-5, None)):
            with pytest.raises(ValueError, match='sizes'):
                call()


def test_entries_check_weight_and_bias():
    """Refused on the host by the functions below the autograd one, with nothing launched."""
    x, w, b = (t.detach() for t in _case())
    y, mean, rstd = ops.group_norm_act_forward(x, 3, w, b, 1e-5, 'silu')
    for kw, error in ((dict(w=w[:23].contiguous()), ValueError), (dict(b=b.cpu()), ValueError), (dict(w=w.cpu()), ValueError),
                      (dict(b=b.half()), TypeError), (dict(w=w.half(), b=b.half()), TypeError)):
        p = {**dict(w=w, b=b), **kw}
        with pytest.raises(error):
            ops.group_norm_act_forward(x, 3, p['w'], p['b'], 1e-5, 'silu')
        with pytest.raises(error):
            ops.group_norm_act_backward(y, x, 3, p['w'], p['b'], mean, rstd, 1e-5, 'silu')
        with pytest.raises(error):
            torch.ops.kadconv.group_norm_act_backward(y, x, 3, p['w'], p['b'], mean, rstd, 1e-5, 'silu')


@pytest.mark.parametrize('bits', [32, 8])
def test_captured_step_goes_on_from_a_loaded_state(bits):
    """A step captured, a state loaded into the optimizer, replays: those of an optimizer that is not captured."""
    dtype, gen = torch.bfloat16, torch.Generator().manual_seed(3)
    sizes = (5000, 3, 256)
    first = [torch.randn(n, generator=gen).to(DEV, dtype) for n in sizes]
    a, b = ([torch.nn.Parameter(t.clone()) for t in first] for _ in range(2))
    for p, q in zip(a, b):
        p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)
    kw = dict(lr=1e-2, state_bits=bits, master_weights=True, seed=4)
    oa, ob = kadconv.AdamW(a, capturable=True, **kw), kadconv.AdamW(b, **kw)

    def grads():
        for p, q in zip(a, b):
            p.grad.copy_(torch.randn(p.shape, generator=gen))
            q.grad.copy_(p.grad)

    def same():
        torch.cuda.synchronize()
        assert oa.param_groups[0]['step'].item() == ob.param_groups[0]['step']
        for p, q in zip(a, b):
            # the graph computes its rates on the GPU: a bf16 parameter may be rounded the other way
            torch.testing.assert_close(p, q, rtol=2.0 ** -8, atol=1e-9)
            for name, t in oa.state[p].items():
                torch.testing.assert_close(t.float(), ob.state[q][name].float(), rtol=1e-6, atol=1e-9)

    grads()
    oa.step(), ob.step()
    saved = copy.deepcopy((oa.state_dict(), [p.detach().clone() for p in a]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step()
    for _ in range(2):
        grads()
        graph.replay()
        ob.step()
    same()
    where = {k: t.data_ptr() for k, t in oa.state[a[0]].items()}
    state_dict, values = saved
    with torch.no_grad():
        for p, q, v in zip(a, b, values):
            p.copy_(v), q.copy_(v)
    oa.load_state_dict(state_dict)
    state_dict['param_groups'][0].update(capturable=False, step=1)
    ob.load_state_dict(state_dict)
    assert where == {k: t.data_ptr() for k, t in oa.state[a[0]].items()}
    same()
    for _ in range(2):
        grads()
        graph.replay()
        ob.step()
    same()
    # a state dict without states: as an optimizer that has not stepped
    empty = dict(state={}, param_groups=copy.deepcopy(state_dict['param_groups']))
    empty['param_groups'][0].update(capturable=True, step=0)
    oa.load_state_dict(empty)
    empty['param_groups'][0].update(capturable=False)
    ob.load_state_dict(empty)
    assert not any(t.float().any() for p in a for name, t in oa.state[p].items() if name != 'master')
    for _ in range(2):
        grads()
        graph.replay()
        ob.step()
    same()


def test_captured_step_outlives_a_load_that_replaces_it():
    """Options loaded that ask for other states: the plan that a graph writes by stays, and eager steps go on."""
    p = torch.nn.Parameter(torch.zeros(5000, device=DEV))
    p.grad = torch.randn(5000, device=DEV)
    opt, other = kadconv.AdamW([p], capturable=True), kadconv.AdamW([torch.nn.Parameter(torch.zeros(5000, device=DEV))], state_bits=8)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    plan = opt._plans[0][0][0]
    opt.load_state_dict(other.state_dict())
    assert opt._retired == [plan] and opt.param_groups[0]['state_bits'] == 8
    opt.step()
    assert set(opt.state[p]) == {'exp_avg', 'exp_avg_scale', 'exp_avg_sq_root', 'exp_avg_sq_root_scale'}


def test_loaded_rates_are_on_the_gpu():
    """A rate that is a GPU scalar, from a state dict brought to host memory: into the optimizer's own scalar, which
    a graph may read, and where two groups of one scalar load two rates, each into its own."""
    p, q = (torch.nn.Parameter(torch.zeros(8, device=DEV)) for _ in range(2))
    p.grad, q.grad = torch.ones(8, device=DEV), torch.ones(8, device=DEV)
    lr = torch.tensor(1e-2, device=DEV)
    opt = kadconv.AdamW([dict(params=[p]), dict(params=[q])], lr=lr, weight_decay=0.0, capturable=True)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    for group in saved['param_groups']:
        group['lr'] = torch.tensor(0.25)
        group['step'] = group['step'].cpu()
    opt.load_state_dict(saved)
    assert all(group['lr'] is lr for group in opt.param_groups) and lr.item() == 0.25
    with torch.no_grad():
        p.zero_(), q.zero_()
    opt.step()
    # a steady gradient's step is lr, up to eps and a few roundings
    torch.testing.assert_close(p.detach(), torch.full_like(p, -0.25), rtol=1e-5, atol=0)
    assert torch.equal(p, q)
    saved['param_groups'][1]['lr'] = torch.tensor(0.5)
    opt.load_state_dict(saved)
    assert [group['lr'].item() for group in opt.param_groups] == [0.25, 0.5]
    assert all(group['lr'].is_cuda for group in opt.param_groups)
    opt.step()
    fresh = kadconv.AdamW([dict(params=[p]), dict(params=[q])])
    fresh.load_state_dict(saved)
    assert all(group['lr'].is_cuda and group['step'].is_cuda for group in fresh.param_groups)
    fresh.step()


def test_refused_load_leaves_the_optimizer():
    """A state dict whose second group does not fit: the error, and an optimizer that goes on as it was."""
    def make():
        gen = torch.Generator().manual_seed(6)
        params = [torch.nn.Parameter(torch.randn(300, generator=gen).to(DEV)) for _ in range(2)]
        for p in params:
            p.grad = torch.randn(300, generator=gen).to(DEV)
        opt = kadconv.AdamW([dict(params=params[:1]), dict(params=params[1:])], lr=1e-2)
        opt.step()
        return params, opt
    (a, oa), (b, ob) = make(), make()
    saved = copy.deepcopy(oa.state_dict())
    for group in saved['param_groups']:
        group.update(lr=0.5, step=40)
    saved['state'][0]['exp_avg'].fill_(7)
    saved['state'][1]['exp_avg'] = torch.zeros(299, device=DEV)
    with pytest.raises(ValueError, match='exp_avg'):
        oa.load_state_dict(saved)
    assert [group['step'] for group in oa.param_groups] == [1, 1] and oa.param_groups[0]['lr'] == 1e-2
    oa.step(), ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    for p, q in zip(a, b):
        assert torch.equal(oa.state[p]['exp_avg'], ob.state[q]['exp_avg'])


class _Ops(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize('grad', [False, True])
def test_traced_call_is_in_the_trace(grad):
    """A traced network computes on what it is given, not on the example."""
    net = torch.nn.Sequential(kadconv.GroupNormAct(3, 24), torch.nn.Sigmoid()).to(DEV)
    a, b = _case(0)[0].detach(), _case(1)[0].detach()
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(net, a)
        assert 'group_norm_act' in str(traced.inlined_graph)
        for x in (a, b):
            assert torch.equal(traced(x), net(x))
        if grad:
            b.requires_grad_(True)
            assert torch.equal(*(torch.autograd.grad(f(b).square().sum(), b)[0] for f in (traced, net)))


def test_dispatch_modes_see_the_call():
    x, w, b = _case()
    want = torch.autograd.grad(f(x, w, b).sum(), (x, w, b))
    with _Ops() as mode:
        got = torch.autograd.grad(f(x, w, b).sum(), (x, w, b))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert 'kadconv.group_norm_act.default' in mode.seen and 'kadconv.group_norm_act_backward.default' in mode.seen
    graph = make_fx(lambda t: f(t, w.detach(), b.detach()).relu())(x.detach())
    other = _case(1)[0].detach()
    assert torch.equal(graph(other), f(other, w.detach(), b.detach()).relu())


def test_fake_maps_have_gradients():
    with FakeTensorMode() as mode:
        x, w, b = (mode.from_tensor(t) for t in _case())
        grads = torch.autograd.grad(f(x, w, b).sum(), (x, w, b))
    assert [g.shape for g in grads] == [t.shape for t in (x, w, b)]


def test_replaced_parameters_are_noticed():
    """Another parameter in the same place, a group gone with another in its place, two that changed places: errors
    that leave the parameters and the count of steps as they are."""
    def param(dtype=torch.float32):
        p = torch.nn.Parameter(torch.zeros(8, dtype=dtype, device=DEV))
        p.grad = torch.ones_like(p)
        return p

    def refused(opt, params):
        steps = [group['step'] for group in opt.param_groups]
        before = [p.detach().clone() for p in params]
        with pytest.raises(RuntimeError, match='new optimizer'):
            opt.step()
        assert steps == [group['step'] for group in opt.param_groups]
        assert all(torch.equal(p, q) for p, q in zip(params, before))

    p, new = param(), param()
    opt = kadconv.AdamW([p])
    opt.step()
    opt.param_groups[0]['params'][0] = new
    refused(opt, [p, new])
    a, b, c = param(), param(), param()
    opt = kadconv.AdamW([dict(params=[a]), dict(params=[b])])
    opt.step()
    opt.param_groups.pop(0)
    refused(opt, [a, b])
    opt = kadconv.AdamW([a, b])
    opt.step()
    opt.param_groups[0]['params'].reverse()
    refused(opt, [a, b])
    # several dtypes in a group: a plan each
    h, i, new = param(torch.float16), param(torch.float16), param(torch.float16)
    opt = kadconv.AdamW([a, h, b, i])
    opt.step(), opt.step()
    assert h.any() and torch.equal(h, i)
    opt.param_groups[0]['params'][3] = new
    refused(opt, [a, h, b, i, new])
    opt = kadconv.AdamW([a, h, c])       # one of a dtype alone
    opt.step(), opt.step()
    opt.param_groups[0]['params'][1] = new
    refused(opt, [a, h, c, new])


@pytest.mark.parametrize('views', [False, True])
@pytest.mark.parametrize('captured', [False, True])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('bits', [32, 8])
def test_written_parameters_take_over_from_their_masters(bits, dtype, captured, views):
    """Some values of a parameter written between steps: the step is that of a plan whose masters hold these values
    there, and elsewhere (also where a value was written as it was) what they held."""
    gen = torch.Generator().manual_seed(8)
    sizes = (1000, 257, 5)
    flat = torch.randn(1280 if views else 0, generator=gen).to(DEV, dtype)
    at = (0, 1001, 1264)
    params = [flat[a:a + n] if views else torch.randn(n, generator=gen).to(DEV, dtype) for a, n in zip(at, sizes)]
    grads = [torch.randn(n, generator=gen).to(DEV, dtype) for n in sizes]
    kw = dict(state_bits=bits, master_weights=True, seed=3)
    plan = kadconv.AdamWPlan(params, grads, **kw)
    t = torch.tensor(1, device=DEV)
    plan.step(t, lr=1e-3)
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.step(t, lr=1e-3)
    for k in range(2, 5):
        t.fill_(k)
        params[0][100:300] = 0.5
        params[0][500:600].clamp_(-0.2, 0.2)
        params[1].mul_(1)
        params[2][3] = float('inf') if k == 4 else -7.0
        masters, values = plan.state['master'].clone(), [p.clone() for p in params]
        for i, p in enumerate(params):
            m = plan.part(masters, i)
            m.copy_(torch.where(m.to(dtype) == p, m, p.float()))
        assert (plan.state['master'] != masters).any() and (plan.state['master'] == masters).sum() > 1000
        other = kadconv.AdamWPlan(values, grads, state=dict({n: s.clone() for n, s in plan.state.items()}, master=masters), **kw)
        graph.replay() if captured else plan.step(t, lr=1e-3)
        other.step(t, lr=1e-3)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(params, values)), k
        for name, s in plan.state.items():
            assert all(torch.equal(plan.part(s, i), other.part(other.state[name], i)) for i in range(3) if 'scale' not in name)


def test_loaded_model_and_optimizer_in_either_order():
    """Masters are more than the parameters tell: a model's and its optimizer's state dicts, loaded in either order
    between steps, leave the masters' bits as they were saved."""
    def make():
        p = torch.nn.Parameter(torch.linspace(-1, 1, 300, device=DEV, dtype=torch.bfloat16))
        p.grad = torch.linspace(1, 2, 300, device=DEV, dtype=torch.bfloat16)
        opt = kadconv.AdamW([p], master_weights=True)
        opt.step()
        return p, opt
    p, opt = make()
    opt.step()
    saved = copy.deepcopy((p.detach(), opt.state_dict()))
    opt.step()
    for first in ('model', 'optimizer'):
        q, other = make()
        for what in sorted(('model', 'optimizer'), key=lambda w: w != first):
            if what == 'model':
                with torch.no_grad():
                    q.copy_(saved[0])
            else:
                other.load_state_dict(saved[1])
        other.step()
        assert torch.equal(q, p) and torch.equal(other.state[q]['master'], opt.state[p]['master']), first


@pytest.mark.parametrize('master', [False, True], ids=['f32', 'bf16_master'])
@pytest.mark.parametrize('bits', [32, 8])
def test_parameters_of_32_bits_are_those_of_the_formula_in_32_bits(bits, master):
    """Parameters and masters in fp32 after a step, bit for bit as the CPU's operations round the formula, each
    operation by itself: no fewer bits in the quotient, whatever holds the states."""
    n, lr, (b1, b2), eps, wd = 256 * 512, 3e-3, (0.9, 0.999), 1e-8, 0.1
    gen = torch.Generator().manual_seed(12)
    dtype = torch.bfloat16 if master else torch.float32
    start = torch.randn(n, generator=gen) * (torch.rand(n, generator=gen) < 0.5)   # half of them 0: the quotient alone
    p = start.to(DEV, dtype)
    g = torch.empty(n, dtype=dtype, device=DEV)
    plan = kadconv.AdamWPlan([p], [g], state_bits=bits, master_weights=master)
    for t in (1, 2, 3):
        g.copy_(torch.randn(n, generator=gen) * torch.exp(3 * torch.randn(n, generator=gen)) * 1e-3)
        st = {k: v.cpu() for k, v in plan.state.items()}
        x, gc = (st['master'] if master else p.cpu()), g.float().cpu()
        f32 = lambda v: torch.tensor(v, dtype=torch.float64).float()
        if bits == 8:
            m, u = (st[k].float() * st[k + '_scale'].repeat_interleave(256) for k in ('exp_avg', 'exp_avg_sq_root'))
            v = u * u
        else:
            m, v = st['exp_avg'], st['exp_avg_sq']
        m = m * f32(b1) + gc * f32(1 - b1)
        v = v * f32(b2) + (gc * gc) * f32(1 - b2)
        u = torch.from_numpy(np.sqrt(v.numpy()))   # rounded; torch's on the CPU is off by a step for one in six
        want = x * f32(1 - lr * wd) - (f32(lr / (1 - b1 ** t)) * m) / (u * f32(1 / (1 - b2 ** t) ** 0.5) + f32(eps))
        plan.step(t, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd)
        got = plan.state['master'] if master else p
        assert torch.equal(got.cpu(), want), (t, int((got.cpu() != want).sum()))


@pytest.mark.parametrize('change', [lambda t: t.half(), lambda t: t.cpu(), lambda t: t[:1]], ids=['dtype', 'device', 'shape'])
def test_saved_tensors_that_a_hook_replaced_are_checked(change):
    """What unpacking gives is compared with the gradient before a kernel reads it as the map."""
    x, w, b = _case()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        y = f(x, w, b)
    with pytest.raises((TypeError, ValueError)):
        torch.autograd.grad(y, (x, w, b), torch.ones_like(y))


def test_statistics_are_saved_as_the_map_is():
    """Hooks see them, and they are freed with the rest of what a graph has saved."""
    x, w, b = _case()
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.shape) or t, lambda t: t):
        f(x, w, b)
    assert sorted(map(tuple, seen)) == sorted([tuple(x.shape), (24,), (24,), (2, 2, 3)])

    class Kept:
        alive = 0

        def __init__(self, t):
            self.t = t
            Kept.alive += 1

        def __del__(self):
            Kept.alive -= 1

    with torch.autograd.graph.saved_tensors_hooks(Kept, lambda k: k.t):
        y = f(x, w, b)
    assert Kept.alive == 4
    torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert Kept.alive == 0 and y.grad_fn is not None
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:1] if t.dim() == 3 else t):
        y = f(x, w, b)
    with pytest.raises(ValueError, match='statistics'):
        torch.autograd.grad(y, (x, w, b), torch.ones_like(y))


def test_buffers_of_a_plan_outlive_their_kernels_on_another_stream():
    """A plan stepped on a stream that is still busy, and dropped: its table, scalars and states (which were made on
    the first stream) are not free yet, as the allocator counts them, and are once the stream is through."""
    def held_back():  # blocks that are freed, but wait for a stream
        stats = torch.cuda.memory_stats()
        return stats['active.all.current'] - stats['allocation.all.current']

    p, g = torch.zeros(5000, device=DEV), torch.ones(5000, device=DEV)
    t = torch.tensor(1, device=DEV)
    side = torch.cuda.Stream()
    plan = kadconv.AdamWPlan([p], [g], state_bits=8)
    plan.step(t)
    torch.cuda.synchronize()
    before = held_back()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        plan.step(t)
    del plan
    assert held_back() - before == 2 + 4
    torch.cuda.synchronize()
    torch.empty(1, device=DEV)  # the allocator looks at its events
    assert held_back() == before


def test_captured_scalars_outlive_a_load_that_replaces_them():
    """Options loaded that count in Python, and rates that groups shared and share no more: what a graph reads and
    writes stays allocated."""
    p, q = (torch.nn.Parameter(torch.zeros(8, device=DEV)) for _ in range(2))
    p.grad, q.grad = torch.ones(8, device=DEV), torch.ones(8, device=DEV)
    lr = torch.tensor(1e-2, device=DEV)
    opt = kadconv.AdamW([dict(params=[p]), dict(params=[q])], lr=lr, capturable=True)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    counts = [group['step'] for group in opt.param_groups]
    saved = copy.deepcopy(opt.state_dict())
    for group, rate in zip(saved['param_groups'], (0.25, 0.5)):
        group['lr'] = torch.tensor(rate)
    opt.load_state_dict(saved)
    assert [group['step'] for group in opt.param_groups] == counts
    assert [t is lr for t in opt._retired_scalars] == [True, True]
    for group in saved['param_groups']:
        group.update(capturable=False, lr=1e-2, step=7)
    opt.load_state_dict(saved)
    assert all(any(t is c for t in opt._retired_scalars) for c in counts)
    opt.step()
    assert [group['step'] for group in opt.param_groups] == [8, 8]


def test_masters_of_more_than_the_last_cache_holds():
    """The same in one plan, whose loads go past the caches, and in two whose do not: masters, and written parameters."""
    n, half = 12_000_007, 4096 * 1400
    gen = torch.Generator(device=DEV).manual_seed(21)
    p = torch.randn(n, generator=gen, device=DEV).bfloat16()
    g = torch.randn(n, generator=gen, device=DEV).bfloat16()
    q = [p[:half].clone(), p[half:].clone()]
    whole = kadconv.AdamWPlan([p], [g], master_weights=True)
    parts = [kadconv.AdamWPlan([v], [w.clone()], master_weights=True) for v, w in zip(q, (g[:half], g[half:]))]
    for t in (1, 2, 3):
        whole.step(t)
        for plan in parts:
            plan.step(t)
        if t == 2:   # so that the third step compares
            for v in (p, *q):
                v.clamp_(-0.5, 0.5)
    assert torch.equal(p, torch.cat(q)) and p.abs().max() < 0.51
    for name in ('exp_avg', 'exp_avg_sq', 'master'):
        assert torch.equal(whole.state[name][:n], torch.cat([parts[0].state[name][:half], parts[1].state[name][:n - half]])), name
