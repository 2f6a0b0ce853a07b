"""Layer norm, products in 8 bits and distillation in traces and under dispatch modes: what is traced computes on what it is
given, by the parameters as they are."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import kadconv

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def trace_jit(m, x):
    return torch.jit.trace(m, x)


def trace_fx(m, x):
    return make_fx(lambda t: m(t))(x)


@pytest.mark.parametrize('trace', [trace_jit, trace_fx])
@pytest.mark.parametrize('warm', [False, True], ids=['cold', 'warm'])
@pytest.mark.parametrize('act', [None, 'silu'])
def test_traced_linear8_follows_its_weight(trace, warm, act):
    """In eval mode, called before it is traced or not: after its weight has changed, the results are the new weight's."""
    m = kadconv.Linear8(40, 12, act=act).to(DEV).eval()
    a, b = randn(70, 40), randn(70, 40, seed=1)
    with torch.no_grad():
        if warm:
            m(a)
        traced = trace(m, a)
        for change in (lambda: None, lambda: m.weight.mul_(-2), lambda: m.weight.copy_(randn(12, 40, seed=2))):
            change()
            for x in (a, b):
                want = kadconv.linear8(x, m.weight, m.bias, act)
                assert torch.equal(traced(x), want) and torch.equal(m(x), want)


def test_compiled_gradients_are_those_that_are_needed(monkeypatch):
    """The gradients of frozen tensors are not computed, and their limits do not hold."""
    from kadconv import block8, ops
    asked = []
    for module, name in ((block8, 'linear8_backward'), (ops, 'layer_norm_backward')):
        def spy(*args, was=getattr(module, name), **kw):
            asked.append(was.__name__)
            out = was(*args, **kw)
            asked.append([g is not None for g in out])
            return out
        monkeypatch.setattr(module, name, spy)
    x, w, b = randn(70, 40), randn(12, 40, seed=1), randn(12, seed=2)
    scale, shift = randn(40, seed=3), randn(40, seed=4)

    def both(x, w, b, scale, shift):
        return kadconv.linear8(kadconv.layer_norm(x, scale, shift), w, b)

    values = x, w, b, scale, shift
    for pick in ((0,), (1,), (2,), (3,), (4,), (0, 1, 2, 3, 4), (0, 2, 4)):
        leaves = [v.clone().requires_grad_(k in pick) for k, v in enumerate(values)]
        of = [leaves[k] for k in pick]
        dy = randn(70, 12, seed=5)
        want = torch.autograd.grad(both(*leaves), of, dy)
        asked.clear()
        got = torch.autograd.grad(torch.compile(both, fullgraph=True, backend='aot_eager')(*leaves), of, dy)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        of_h = bool({0, 3, 4} & set(pick))
        assert asked[:2] == ['linear8_backward', [of_h, 1 in pick, 2 in pick]], (pick, asked)
        assert asked[2:] == (['layer_norm_backward', [k in pick for k in (0, 3, 4)]] if of_h else []), (pick, asked)
        torch._dynamo.reset()


def test_compiled_over_more_rows_than_a_weight_has_gradients_of():
    x, w = torch.ones((1 << 22) + 1, 1, device=DEV, dtype=torch.float16, requires_grad=True), torch.ones(1, 1, device=DEV)

    def f(x):
        return kadconv.linear8(x, w)

    dx, = torch.autograd.grad(torch.compile(f, fullgraph=True, backend='aot_eager')(x), x, torch.ones_like(x))
    assert torch.equal(dx, torch.ones_like(x))


@pytest.mark.parametrize('need', [(True, True, True), (True, False, False), (False, True, False), (False, False, True)], ids=str)
def test_registered_gradients(need):
    """They agree with their descriptions on fake tensors, whichever are needed."""
    x, w, b, dy, h = randn(70, 40), randn(12, 40, seed=1), randn(12, seed=2), randn(70, 12, seed=3), randn(70, 40, seed=4)
    rows = randn(70, seed=5).abs()
    for op, args in ((torch.ops.kadconv.linear8_backward, (dy, x, w, b, -1)), (torch.ops.kadconv.linear8_backward, (dy, x, w, None, -1)),
                     (torch.ops.kadconv.layer_norm_backward, (h, x, w[0], w[1], rows, rows, 1e-5, -1)),
                     (torch.ops.kadconv.layer_norm_backward, (h, x, None, None, rows, rows, 1e-5, -1))):
        torch.library.opcheck(op, (*args, *need), test_utils=['test_schema', 'test_faketensor'])
        full, some = op(*args), op(*args, *need)
        for f, s, n in zip(full, some, need):
            assert torch.equal(f, s) if n else s.numel() == 0
