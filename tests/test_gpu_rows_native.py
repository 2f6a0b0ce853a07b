"""What the autograd nodes of layer norm, linear8 and distill_loss have to keep of a torch program's rules."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.checkpoint import checkpoint

import kadconv

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def _layer_norm(x, w, b):
    return kadconv.layer_norm(x, w, b)


def _linear8(x, w, b):
    return kadconv.linear8(x, w, b)


def _distill(x):
    t, i = torch.topk(x.new_tensor(range(30)).cos().expand(x.shape[0], 30), 5)
    return kadconv.distill_loss(x, t.contiguous(), i.contiguous(), 2.0, 'none')


OPERATORS = {  # the call, the shapes of its differentiable inputs, its node's name
    'layer_norm': (_layer_norm, ((70, 30), (30,), (30,)), 'LayerNormBackward'),
    'linear8': (_linear8, ((70, 30), (12, 30), (12,)), 'Linear8Backward'),
    'distill_loss': (_distill, ((70, 30),), 'DistillBackward'),
}
EACH = pytest.mark.parametrize('name', list(OPERATORS))


def case(name, seed=0):
    f, shapes, _ = OPERATORS[name]
    return f, [randn(*s, seed=seed + k).requires_grad_(True) for k, s in enumerate(shapes)]


def gradients(f, leaves):
    y = f(*leaves)
    return torch.autograd.grad(y, leaves, randn(*y.shape, seed=9))


@EACH
def test_checkpoint_gives_the_same_gradients(name):
    f, leaves = case(name)
    want = gradients(f, leaves)
    for reentrant in (False, True):
        for t in leaves:
            t.grad = None
        y = checkpoint(f, *leaves, use_reentrant=reentrant)
        y.backward(randn(*y.shape, seed=9))
        assert all(torch.equal(t.grad, g) for t, g in zip(leaves, want))


@EACH
def test_second_backward_and_retained_graph(name):
    f, leaves = case(name)
    y = f(*leaves)
    dy = torch.ones_like(y)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(y, leaves, dy)))
    with pytest.raises(RuntimeError, match='second time'):
        torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize('name', ['layer_norm', 'distill_loss'])
def test_changed_input_is_noticed(name):
    f, leaves = case(name)
    y = f(*leaves)
    with torch.no_grad():
        leaves[0].mul_(2)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


@EACH
def test_no_graph_where_none_is_wanted(name):
    f, leaves = case(name)
    with torch.no_grad():
        assert not f(*leaves).requires_grad
    with torch.inference_mode():
        assert f(*leaves).is_inference()
    assert not f(*(t.detach() for t in leaves)).requires_grad
    assert f(*leaves[:1], *(t.detach() for t in leaves[1:])).grad_fn.name() == OPERATORS[name][2]


@EACH
def test_first_order_gradient_with_create_graph(name):
    f, leaves = case(name)
    want = torch.autograd.grad(f(*leaves).sum(), leaves[0])[0]
    got = torch.autograd.grad(f(*leaves).sum(), leaves[0], create_graph=True)[0]
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        got.sum().backward()


@EACH
def test_forward_mode_is_refused(name):
    f, leaves = case(name)
    for k in range(len(leaves)):
        with torch.autograd.forward_ad.dual_level():
            args = [t.detach() for t in leaves]
            args[k] = torch.autograd.forward_ad.make_dual(args[k], torch.ones_like(args[k]))
            with pytest.raises(NotImplementedError, match='forward-mode'):
                f(*args)


def test_forward_mode_of_a_kept_weight_is_refused():
    x, b = randn(40, 30), randn(12, seed=2)
    q, kept = kadconv.quantize8(x), kadconv.quantize8(randn(12, 30, seed=1))
    with torch.autograd.forward_ad.dual_level():
        dual_x, dual_b = (torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, b))
        for call in (lambda: kadconv.linear8(dual_x, kept, b), lambda: kadconv.linear8(x, kept, dual_b),
                     lambda: kadconv.matmul8(q, kept, dual_b)):
            with pytest.raises(NotImplementedError, match='forward-mode'):
                call()


@EACH
def test_mapped_calls_are_right_or_refused(name):
    """torch.vmap and torch.func.grad: the rows' own results, or an error."""
    f, leaves = case(name)
    rest = [t.detach() for t in leaves[1:]]
    x = randn(3, 70, 30, seed=4)
    one = x[0].clone().requires_grad_(True)
    for call, want in ((lambda: torch.vmap(lambda v: f(v, *rest))(x), torch.stack([f(v, *rest) for v in x])),
                       (lambda: torch.func.grad(lambda v: f(v, *rest).sum())(x[0]), torch.autograd.grad(f(one, *rest).sum(), one)[0])):
        try:
            got = call()
        except (RuntimeError, NotImplementedError, ValueError, TypeError):
            continue
        assert torch.equal(got, want)


@EACH
@pytest.mark.parametrize('change', [lambda t: t.half(), lambda t: t.cpu(), lambda t: t[:1]], ids=['dtype', 'device', 'shape'])
def test_saved_tensors_that_a_hook_replaced_are_checked(name, change):
    f, leaves = case(name)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        y = f(*leaves)
    with pytest.raises((TypeError, ValueError)):
        torch.autograd.grad(y, leaves, torch.ones_like(y))


@EACH
def test_saved_tensors_are_freed(name):
    class Kept:
        alive = 0

        def __init__(self, t):
            self.t = t
            Kept.alive += 1

        def __del__(self):
            Kept.alive -= 1

    f, leaves = case(name)
    with torch.autograd.graph.saved_tensors_hooks(Kept, lambda k: k.t):
        y = f(*leaves)
    assert Kept.alive >= 2
    torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert Kept.alive == 0 and y.grad_fn is not None


class _Ops(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


@EACH
def test_dispatch_modes_see_the_call(name):
    f, leaves = case(name)
    want = gradients(f, leaves)
    with _Ops() as mode:
        got = gradients(f, leaves)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert f'kadconv.{name}.default' in mode.seen and f'kadconv.{name}_backward.default' in mode.seen
    rest = [t.detach() for t in leaves[1:]]
    graph = make_fx(lambda t: f(t, *rest).relu())(leaves[0].detach())
    other = randn(70, 30, seed=7)
    assert torch.equal(graph(other), f(other, *rest).relu())


@EACH
@pytest.mark.parametrize('grad', [False, True])
def test_traced_call_is_in_the_trace(name, grad):
    """What torch.jit.trace makes of a call computes on what it is given, and its gradients."""
    f, leaves = case(name)
    _, others = case(name, seed=20)
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(f, tuple(t.detach() for t in leaves))
        assert f'kadconv::{name}' in str(traced.inlined_graph if hasattr(traced, 'inlined_graph') else traced.graph)
        for args in (leaves, others):
            assert torch.equal(traced(*args), f(*args))
            if grad:
                assert all(torch.equal(p, q) for p, q in zip(gradients(traced, args), gradients(f, args)))


@EACH
def test_fake_tensors_have_gradients(name):
    f, leaves = case(name)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        fakes = [mode.from_tensor(t) for t in leaves]
        y = f(*fakes)
        grads = torch.autograd.grad(y.sum(), fakes)
    assert [g.shape for g in grads] == [t.shape for t in leaves] and [g.dtype for g in grads] == [t.dtype for t in leaves]


def test_served_products_in_traces():
    """quantize8, matmul8 and linear8 with a kept weight under both tracers, on other inputs than they were traced with."""
    w, b = randn(12, 30, seed=1), randn(12, seed=2)
    kept = kadconv.quantize8(w)

    def served(x):
        return kadconv.linear8(x, kept, b, 'silu')

    def product(x):
        return kadconv.matmul8(kadconv.quantize8(x), kept, b, dtype=torch.float32)

    a, c = randn(70, 30, seed=3), randn(70, 30, seed=4)
    with torch.no_grad():
        for f in (served, product):
            for traced in (torch.jit.trace(f, a), make_fx(f)(a)):
                assert torch.equal(traced(a), f(a)) and torch.equal(traced(c), f(c))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
def test_short_rows_of_the_most_values_in_a_graph(dtype):
    """Rows of 500 values take more LDS than a launch has by default: what it asks for is asked for in captures too."""
    x, kept = randn(2100, 500).to(dtype), kadconv.quantize8(randn(600, 500, seed=1))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = kadconv.linear8(x, kept, act='silu')
    for k in range(3):
        x.copy_(randn(2100, 500, seed=5 + k))
        graph.replay()
        want = kadconv.linear8(x, kept, act='silu')
        torch.cuda.synchronize()
        assert torch.equal(y, want) and y.any(), k
