"""Layer norm, products in 8 bits and distillation, called in the less usual ways that they allow."""
import threading

import pytest
import torch

import kadconv
from kadconv import block8

pytestmark = pytest.mark.gpu

DEV = 'cuda'
F16 = torch.float16


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def inputs(rows=70, c=200, n=60, entries=9):
    x, w, b = randn(rows, c), randn(n, c, seed=1), randn(n, seed=2)
    t, i = torch.topk(randn(rows, c, seed=3), entries)
    return x, w, b, t, i


def every_call(x, w, b, t, i):
    """Results and gradients of the three operators, of these values."""
    x, w, b = (v.detach().requires_grad_(True) for v in (x, w, b))
    scale, shift = w[0].detach().clone().requires_grad_(True), w[1].detach().clone().requires_grad_(True)
    out = []
    for y, of in ((kadconv.layer_norm(x, scale, shift), (x, scale, shift)), (kadconv.linear8(x, w, b), (x, w, b)),
                  (kadconv.distill_loss(x, t, i, 2.0), (x,))):
        out += [y.detach(), *torch.autograd.grad((y * y).sum(), of)]
    q = kadconv.quantize8(w.detach())
    out += [q.codes.float(), q.scales.float(), kadconv.matmul8(kadconv.quantize8(x.detach()), q, b.detach(), dtype=torch.float32)]
    return out


def negative_view(v):
    """A view of -(-v): its storage holds -v."""
    z = torch.complex(torch.zeros_like(v), -v).conj().imag
    assert z.is_neg() and torch.equal(z, v)
    return z


def test_views_that_negate():
    x, w, b, t, i = inputs()
    for got, want in zip(every_call(negative_view(x), negative_view(w), negative_view(b), negative_view(t), i), every_call(x, w, b, t, i)):
        assert torch.equal(got, want)
    dy = randn(70, 200, seed=4)
    mean, rstd = randn(70, seed=5), randn(70, seed=6).abs()
    for got, want in zip(kadconv.ops.layer_norm_backward(negative_view(dy), x, w[0], w[1], mean, rstd, 1e-5, -1),
                         kadconv.ops.layer_norm_backward(dy, x, w[0], w[1], mean, rstd, 1e-5, -1)):
        assert torch.equal(got, want)
    y = kadconv.linear8(x, w)
    for got, want in zip(block8.linear8_backward(negative_view(y), x, w, b, -1), block8.linear8_backward(y, x, w, b, -1)):
        assert torch.equal(got, want)


@pytest.mark.parametrize('rows', [3, 70, 700])
def test_saved_tensors_elsewhere(rows):
    """Saved tensors that wait in host memory until they are used."""
    args = inputs(rows)
    want = every_call(*args)
    with torch.autograd.graph.save_on_cpu():
        got = every_call(*args)
    for g, w in zip(got, want):
        assert torch.equal(g, w)


@pytest.mark.parametrize('rows', [3, 700])
def test_two_threads(rows):
    """Two threads at once, a stream each, with other values."""
    args = [inputs(rows), [v.flip(0) for v in inputs(rows)]]
    want = [every_call(*a) for a in args]
    torch.cuda.synchronize()
    got = [[], []]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[k].append(every_call(*args[k]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert len(got[k]) == 10
        for run in got[k]:
            for g, w in zip(run, want[k]):
                assert torch.equal(g, w)


def test_two_graphs():
    """Two captured calls of each operator with workspaces, replayed on two streams at once, and eager calls between."""
    x, w, b, t, i = inputs(100, 9000, 40)
    big, big_t, big_i = randn(2, 40000, seed=7), *torch.topk(randn(2, 40000, seed=8), 20)
    dy = randn(100, 9000, seed=9)

    def run(x, w, z):
        y, mean, rstd = kadconv.ops.layer_norm_forward(x, w[0], w[1], 1e-5, -1)
        loss, stats, share = kadconv.ops.distill_loss_forward(z, big_t, big_i, 2.0, 'mean', -1)
        return [block8.linear8_forward(x, w, b, None, -1), y, loss, *kadconv.ops.layer_norm_backward(dy, x, w[0], w[1], mean, rstd, 1e-5, -1),
                kadconv.ops.distill_loss_backward(loss, z, big_t, big_i, stats, share, 2.0, 'mean', -1),
                *block8.linear8_backward(y[:, :40].contiguous(), x, w, b, -1)]

    sets = [(x, w, big), (x.flip(1).contiguous(), w.flip(0).contiguous(), big.flip(1).contiguous())]
    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(*s))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for o in outs:
            for v in o:
                v.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = run(*sets[turn % 2])
        torch.cuda.synchronize()
        for k in range(2):
            for got, exp in zip(outs[k], want[k]):
                assert torch.equal(got, exp), turn
        for got, exp in zip(eager, want[turn % 2]):
            assert torch.equal(got, exp), turn


def test_registered_operators():
    """The registered operators agree with their own descriptions: results on fake tensors, gradients, and no input changed."""
    x, w, b, t, i = inputs(40, 140, 12)
    leaf = [v.detach().clone().requires_grad_(True) for v in (x, w[0], w[1], w, b)]
    q, p = kadconv.quantize8(x), kadconv.quantize8(w)
    tests = ['test_schema', 'test_autograd_registration', 'test_faketensor']
    ops = torch.ops.kadconv
    for op, args in ((ops.layer_norm, (leaf[0], leaf[1], leaf[2], 1e-5, -1)), (ops.layer_norm, (x, None, None, 1e-5, -1)),
                     (ops.distill_loss, (leaf[0], t, i, 2.0, 'mean', -1)), (ops.distill_loss, (leaf[0], t, i, 2.0, 'none', -1)),
                     (ops.linear8, (leaf[0], leaf[3], leaf[4], None, -1)), (ops.linear8, (x, w, None, 'silu', -1)),
                     (ops.linear8_kept, (x, p.codes, p.scales, 140, b, 'relu', -1)), (ops.quantize8, (x, -1)),
                     (ops.matmul8, (q.codes, q.scales, p.codes, p.scales, 140, b, 'silu', F16))):
        held = op in (ops.linear8_kept, ops.quantize8, ops.matmul8)  # test_schema multiplies results, which torch does not in e4m3
        torch.library.opcheck(op, args, test_utils=tests[1:] if held else tests)


def test_quantize_more_than_2_31_values():
    rows, k = (1 << 20) + 300, 2100
    x = torch.zeros(rows, k, device=DEV, dtype=F16)
    x[-1] = randn(k, dtype=F16)
    x[-200:, -1] = randn(200, seed=1, dtype=F16)
    q = kadconv.quantize8(x)
    tail = kadconv.quantize8(x[-256:].contiguous())
    assert torch.equal(q.codes[-256:].view(torch.uint8), tail.codes.view(torch.uint8))
    assert torch.equal(q.scales[-256:].view(torch.uint8), tail.scales.view(torch.uint8))
    assert not q.codes[:-256].view(torch.uint8).any()


@pytest.mark.parametrize('rows, n', [((1 << 20) + 300, 2100), (32, 60000000)], ids=str)
def test_results_far_from_the_first(rows, n):
    """Results of tiles beyond 2^31 values; of few rows by codes beyond 2^31 bytes."""
    k = 4
    x = torch.randint(-8, 9, (rows, k), device=DEV).to(F16)
    w = torch.zeros(n, k, device=DEV, dtype=F16)
    w[-900:] = torch.randint(-8, 9, (900, k), device=DEV).to(F16)  # all held exactly
    y = kadconv.linear8(x, w)
    want = (x.float() @ w[-900:].float().t()).half()
    assert torch.equal(y[:, -900:], want) and not y[:, :-900].any()


def test_gradients_beyond_2_31_values():
    """The gradients of a weight whose rows' codes lie beyond 2^31 bytes, along its columns too."""
    rows, n, k = 40, 300000, 8000
    w = torch.zeros(n, k, device=DEV, dtype=F16)
    w[-500:] = torch.randint(-1, 2, (500, k), device=DEV).to(F16)
    w[:, -3:] = torch.randint(-1, 2, (n, 3), device=DEV).to(F16)
    x = torch.randint(-1, 2, (rows, k), device=DEV).to(F16)
    dy = torch.zeros(rows, n, device=DEV, dtype=F16)
    dy[:, -700:] = torch.randint(-1, 2, (rows, 700), device=DEV).to(F16)
    dx, dw, db = block8.linear8_backward(dy, x, w, torch.zeros(n, device=DEV), -1)
    # sums of small whole numbers, which fp32 holds; results of up to 2048 fp16 does
    assert torch.equal(dx, (dy[:, -700:].float() @ w[-700:].float()).half())
    assert torch.equal(dw[-700:], (dy[:, -700:].float().t() @ x.float()).half()) and not dw[:-700].any()
    assert torch.equal(db, dy.float().sum(0))
    y = kadconv.linear8(x, w)
    assert torch.equal(y[:, -500:], (x.float() @ w[-500:].float().t()).half())
