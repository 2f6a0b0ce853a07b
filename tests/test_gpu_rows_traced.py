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
