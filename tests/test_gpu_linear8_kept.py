"""Linear8 in eval mode gives the results of its weight as it is, however that was changed."""
import pytest
import torch

import kadconv

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def check(m, x):
    with torch.no_grad():
        want = kadconv.linear8(x, m.weight, m.bias, m.act)
        got = m(x)
    assert got.shape == want.shape and torch.equal(got, want)


def served(m):
    """The module with a copy of its weight, with which it gives what it gives without."""
    x = randn(30, m.in_features, seed=9)
    with torch.no_grad():
        want = m.eval()(x)
        assert m._kept is None and m.keep() is m and m._kept is not None
        assert torch.equal(m(x), want) and m._kept is not None
    return m


def test_replayed_changes_are_seen():
    """A graph that writes the weight bumps its version where it is captured, not where it is replayed."""
    m, x = kadconv.Linear8(40, 12).to(DEV).eval(), randn(70, 40)
    check(m, x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        m.weight.mul_(-1.5)
    for _ in range(3):
        check(m, x)
        graph.replay()
        check(m, x)


def test_replayed_steps_are_seen():
    m, x = kadconv.Linear8(40, 12).to(DEV), randn(70, 40)
    opt = kadconv.AdamW(m.parameters(), lr=0.1, capturable=True)
    for p in m.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        check(m.eval(), x)
        graph.replay()
        check(m, x)
        m.train()
        graph.replay()
        check(m.eval(), x)


@pytest.mark.parametrize('change', ['fewer rows', 'transposed', 'other parameter', 'through data'])
def test_other_views_of_the_same_numbers_are_seen(change):
    m, x = kadconv.Linear8(24, 24, bias=False).to(DEV).eval(), randn(50, 24)
    check(m, x)
    w = m.weight
    if change == 'fewer rows':
        w.data = w.data[:4]
    elif change == 'transposed':
        w.data = w.data.t()
    elif change == 'other parameter':
        m.weight = torch.nn.Parameter(w.detach()[:4])
    else:
        w.data.mul_(-2)
    check(m, x)


def test_a_kept_weight_is_read():
    """Without its copy the module would give other results: of a write that no version tells."""
    m, x = served(kadconv.Linear8(40, 12, act='silu').to(DEV)), randn(70, 40)
    with torch.no_grad():
        before = m(x)
        m.weight.data.zero_()
        assert torch.equal(m(x), before)
        assert m.keep() is m
        check(m, x)
        assert not torch.equal(m(x), before)
        assert m.keep(False)._kept is None
        check(m, x)


@pytest.mark.parametrize('change', ['in place', 'loaded', 'fewer rows', 'transposed', 'other parameter', 'other type', 'trained', 'stepped'])
def test_a_kept_weight_is_dropped_where_it_changed(change):
    m, x = served(kadconv.Linear8(24, 24, bias=False).to(DEV)), randn(50, 24)
    w = m.weight
    with torch.no_grad():
        if change == 'in place':
            w.mul_(-2)
        elif change == 'loaded':
            m.load_state_dict(dict(weight=randn(24, 24, seed=3)))
        elif change == 'fewer rows':
            w.data = w.data[:4]
        elif change == 'transposed':
            w.data = w.data.t()
        elif change == 'other parameter':
            m.weight = torch.nn.Parameter(w.detach()[:4])
        elif change == 'other type':
            m.half()
            x = x.half()
        elif change == 'trained':
            m.train()
            w.data.zero_()
            m.eval()
        else:
            w.grad = torch.ones_like(w)
            kadconv.AdamW([w], lr=0.1).step()
    check(m, x)
    assert m._kept is None


def test_calls_that_do_not_go_by_the_copy():
    """Differentiated, captured and traced ones: a write that no version tells is in their results."""
    m, x = served(kadconv.Linear8(40, 12, bias=False).to(DEV)), randn(70, 40)
    with torch.no_grad():
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x)
        traced = torch.jit.trace(m, x)
        m.weight.data.zero_()
        graph.replay()
        assert not y.any() and not traced(x).any() and m(x).any()
    assert not m(x).any() and m(x).requires_grad


def test_refusals():
    m = kadconv.Linear8(8, 4)
    with pytest.raises(RuntimeError, match='GPU'):
        m.eval().keep()
    m.to(DEV).train()
    with pytest.raises(RuntimeError, match='eval'):
        m.keep()
    m.eval()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.weight.detach() + 1
        with pytest.raises(RuntimeError, match='captured'):
            m.keep()
    assert m._kept is None


def test_another_stream():
    """The copy is made on one stream, behind much other work, and used on another at once."""
    m, x = kadconv.Linear8(300, 64).to(DEV).eval(), randn(200, 300)
    busy, side = randn(4096, 4096, seed=1), torch.cuda.Stream()
    with torch.no_grad():
        want = m(x)
        torch.cuda.synchronize()
        for _ in range(20):
            busy = busy @ busy
            busy = busy / busy.norm()
        m.keep()
        with torch.cuda.stream(side):
            got = m(x)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_a_served_head():
    from kadcnet import finetune
    torch.manual_seed(0)
    head = finetune.StudentHead([32, 64], 9, width=48).to(DEV)
    maps = [randn(2, 9, 7, 32, seed=1).permute(0, 3, 1, 2), randn(2, 5, 4, 64, seed=2).permute(0, 3, 1, 2)]
    trained = head(maps)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(head.serve()(maps), trained))
    linears = [m for m in head.modules() if isinstance(m, kadconv.Linear8)]
    assert len(linears) == 6 and all(m._kept is not None for m in linears)
    assert all(m._kept is None for m in head.train().modules() if isinstance(m, kadconv.Linear8))
