"""Layer norm, products in 8 bits and distillation run together, as a head that is trained by a teacher and served."""
import copy

import pytest
import torch

import kadconv
from kadcnet import finetune

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
def test_program_runs(dtype, capsys):
    losses, student = finetune.main(['--steps', '3', '--batch', '2', '--size', '256', '--dtype', dtype, '--distill', '3'])
    assert len(losses) == len(student) == 3 and all(x == x and x >= 0 for x in student)
    assert 'student: 3 steps by 3 entries' in capsys.readouterr().out


def setup(sizes=((2, 32, 12, 9), (2, 64, 5, 7)), classes=9, entries=4, seed=0):
    g = torch.Generator().manual_seed(seed)
    maps = [torch.randn(n, h, w, c, generator=g).permute(0, 3, 1, 2) for n, c, h, w in sizes]
    top = []
    for n, _, h, w in sizes:
        t, i = torch.topk(2 * torch.randn(n, classes, h, w, generator=g), entries, dim=1)
        i[0, :, 0, 0] = -1       # a cell without a teacher
        top.append((t, i))
    torch.manual_seed(seed)
    return finetune.StudentHead([s[1] for s in sizes], classes, width=48), maps, top


def loss_of(head, maps, top):
    return sum(kadconv.distill_loss(z, t, i, 2.0, dim=1) for z, (t, i) in zip(head(maps), top))


def to_gpu(head, maps, top):
    return copy.deepcopy(head).cuda(), [m.cuda() for m in maps], [(t.cuda(), i.cuda()) for t, i in top]


def test_gradients_of_the_head():
    """Against the plain compositions on the CPU.  Both bring numbers to 8 bits that differ by some 1e-7 of themselves: one in
    3e5 of them (2e-7 of 2^-4) is rounded the other way, which changes it by 2^-3 at most, one of the 32 to 240 terms of
    each of its sums: 1e-3 of the norm covers a hundred of them, and a wrong formula is off by far more."""
    head, maps, top = setup()
    there, gmaps, gtop = to_gpu(head, maps, top)
    want = loss_of(head, maps, top)
    got = loss_of(there, gmaps, gtop)
    assert abs(got.item() - want.item()) <= 1e-3 * want.item()
    want.backward()
    got.backward()
    for (name, p), q in zip(head.named_parameters(), there.parameters()):
        off = (q.grad.cpu() - p.grad).norm()
        assert off <= 1e-3 * p.grad.norm(), (name, off.item(), p.grad.norm().item())


def test_served_in_8_bits_as_it_was_trained():
    """Kept weights give what the training forward gives, bit for bit."""
    head, maps, _ = setup()
    head, maps, _ = to_gpu(head, maps, [])
    trained = head(maps)
    head.eval()
    with torch.no_grad():
        for _ in range(2):
            assert all(torch.equal(a, b.detach()) for a, b in zip(head(maps), trained))
    assert 0.0 <= finetune.agreement(head, head.train(), maps) == 1.0


def test_steps_change_the_student_alone():
    head, maps, top = to_gpu(*setup())
    before = [p.clone() for p in head.parameters()]
    kept = [m.clone() for m in maps]
    losses = finetune.distill_head(head, [(maps, top)] * 3, state_bits=32)
    assert losses.shape == (3,) and torch.isfinite(losses).all()
    assert not any(torch.equal(p, q) for p, q in zip(head.parameters(), before))
    assert all(torch.equal(a, b) for a, b in zip(maps, kept))


def test_a_step_in_a_graph():
    """Forward and gradients of the three, by their functions, captured into one graph; replays with eager work between."""
    from kadconv import block8, ops
    g = torch.Generator().manual_seed(1)
    w = (torch.randn(10, 40, generator=g) / 6).cuda()
    b, nw, nb = (torch.randn(n, generator=g).cuda() for n in (10, 40, 40))

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        t, i = torch.topk(torch.randn(300, 10, generator=g), 3, dim=1)
        return torch.randn(300, 40, generator=g).cuda(), t.cuda(), i.cuda()

    one = torch.ones((), device='cuda')

    def step(x, t, i):
        h, mean, rstd = ops.layer_norm_forward(x, nw, nb, 1e-5, -1)
        z = block8.linear8_forward(h, w, b, None, -1)
        loss, stats, share = ops.distill_loss_forward(z, t, i, 1.0, 'mean', -1)
        dz = ops.distill_loss_backward(one, z, t, i, stats, share, 1.0, 'mean', -1)
        dh, dw, db = block8.linear8_backward(dz, h, w, b, -1)
        return (loss, dw, db, *ops.layer_norm_backward(dh, x, nw, nb, mean, rstd, 1e-5, -1))

    held = inputs(2)
    step(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for r in range(4):
        new = inputs(3 + r)
        for a, c in zip(held, new):
            a.copy_(c)
        graph.replay()
        want = step(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want)), r
    x, t, i = new
    leaves = [v.clone().requires_grad_(True) for v in (x, nw, nb, w, b)]
    loss = kadconv.distill_loss(kadconv.linear8(kadconv.layer_norm(leaves[0], leaves[1], leaves[2]), leaves[3], leaves[4]), t, i)
    dx, dnw, dnb, dw, db = torch.autograd.grad(loss, leaves)
    assert all(torch.equal(a, c) for a, c in zip((loss, dw, db, dx, dnw, dnb), want))
