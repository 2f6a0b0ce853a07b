"""What the autograd node and the optimizer's table in C++ have to keep of a torch program's rules."""
import copy

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import kadconv

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
