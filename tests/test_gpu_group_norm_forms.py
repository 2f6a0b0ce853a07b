"""The group norm's forms at their borders: groups that just fit a block and just do not, more groups than a
block has threads, widths that need several pixels a row or no rows at all, tiles that end in short rows."""
import pytest
import torch

from kadconv import ops
from tests._norm_ref import EPS32, assert_within, reference
from tests.test_gpu_group_norm import BF16, DEV, F16, F32, check, make, params

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [F32, F16, BF16], ids=['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('shape', [
    (1, 1024, 1024, 12, 13), (1, 1024, 512, 20, 21), (2, 768, 384, 9, 40),   # more groups than threads
    (1, 64, 8, 64, 32), (1, 64, 8, 64, 33), (1, 64, 8, 32, 32), (1, 64, 8, 33, 32),  # 32 KB and a row more
    (2, 1501, 19, 5, 4), (1, 2049, 3, 9, 7), (1, 8200, 8, 3, 3),             # wider than a block
    (1, 1023, 1, 13, 11), (2, 515, 5, 11, 9), (1, 333, 333, 17, 9),          # odd widths: rows of several pixels
    (3, 3, 3, 50, 51), (1, 1, 1, 300, 301), (2, 5, 1, 97, 89),               # and narrow ones
    (1, 2, 2, 1, 3), (1, 3, 1, 1, 2), (2, 9, 3, 1, 1), (1, 24, 8, 1, 7),     # fewer pixels than a row has
    (300, 8, 2, 2, 2), (33, 16, 4, 31, 31), (260, 40, 5, 12, 11),            # many images
    (1, 160, 5, 55, 60), (1, 36, 4, 120, 110), (2, 72, 8, 64, 80)],
    ids=lambda s: 'x'.join(map(str, s)))
def test_forms(shape, dtype):
    n, c, g, h, w = shape
    wt, bs = params(c)
    check(make(n, c, h, w, dtype, seed=h), g, wt, bs, 'silu', make(n, c, h, w, dtype, seed=w + 1))


@pytest.mark.parametrize('layout', ['slice', 'odd'])
def test_wide_and_many_groups_in_other_layouts(layout):
    for n, c, g, h, w in ((1, 1024, 1024, 9, 8), (1, 1504, 4, 7, 6), (1, 8200, 4, 3, 2)):
        wt, bs = params(c, F16)
        check(make(n, c, h, w, F16, 3, layout), g, wt, bs, None, make(n, c, h, w, F16, 4, layout))


def test_parts_of_the_gradient_in_every_form():
    """dx alone, dw alone and db alone equal those of a call that asks for all, bit for bit."""
    for n, c, g, h, w in ((2, 64, 8, 10, 10), (2, 64, 8, 60, 60), (1, 86, 2, 40, 41), (2, 1501, 19, 5, 4)):
        x, dy, (wt, bs) = make(n, c, h, w, F16, 5), make(n, c, h, w, F16, 6), params(c)
        y, mean, rstd = ops.group_norm_act_forward(x, g, wt, bs, 1e-5, 'silu')

        def grads(*need):
            return ops.group_norm_act_backward(dy, x, g, wt, bs, mean, rstd, 1e-5, 'silu', *need)

        whole = grads()
        for k in range(3):
            need = [i == k for i in range(3)]
            part = grads(*need)
            assert torch.equal(part[k], whole[k]) and all(p is None for i, p in enumerate(part) if i != k)


def test_images_do_not_depend_on_their_batch():
    """Small groups stay in a block, whatever else is in the batch."""
    wt, bs = params(64)
    x = make(9, 64, 20, 20, BF16, 7)
    y, _, _ = ops.group_norm_act_forward(x, 8, wt, bs, 1e-5, 'silu')
    for k in (0, 8):
        assert torch.equal(ops.group_norm_act_forward(x[k:k + 1], 8, wt, bs, 1e-5, 'silu')[0], y[k:k + 1])


def test_backward_captured_many_times():
    """Forward and backward of a split map in one graph, replayed with eager work and host syncs between."""
    n, c, g, h, w = 2, 86, 2, 70, 61
    wt, bs = params(c)
    sx, sdy = make(n, c, h, w, F32, 8), make(n, c, h, w, F32, 9)

    def both(x, dy):
        y, mean, rstd = ops.group_norm_act_forward(x, g, wt, bs, 1e-5, 'silu')
        return (y, *ops.group_norm_act_backward(dy, x, g, wt, bs, mean, rstd, 1e-5, 'silu'))

    both(sx, sdy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(sx, sdy)
    for k in range(6):
        nx, ndy = make(n, c, h, w, F32, 20 + k), make(n, c, h, w, F32, 40 + k)
        sx.copy_(nx)
        sdy.copy_(ndy)
        graph.replay()
        want = both(nx, ndy)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_values_past_a_slice_stay_out():
    """A slice's neighbours in the wider map are neither read into the result nor written."""
    wide = torch.full((1, 40, 40, 96), float('nan'), dtype=F16, device=DEV)
    wide[..., 32:64] = torch.randn(1, 40, 40, 32, device=DEV)
    x = wide[..., 32:64].permute(0, 3, 1, 2)
    keep = wide.clone()
    wt, bs = params(32)
    y, mean, rstd = ops.group_norm_act_forward(x, 4, wt, bs, 1e-5, 'silu')
    grads = ops.group_norm_act_backward(x, x, 4, wt, bs, mean, rstd, 1e-5, 'silu')
    assert all(torch.isfinite(t).all() for t in (y, mean, rstd, *grads))
    assert torch.equal(wide.view(torch.int16), keep.view(torch.int16))


def test_more_images_and_groups_than_a_grid_has_layers():
    """65535 images of 128 groups: the first and the last images' results, their gradients the only ones."""
    n, c, g, h, w = 65535, 1024, 128, 1, 2
    wt, bs = params(c)
    x, dy = make(6, c, h, w, F16, 11), make(6, c, h, w, F16, 12)
    ends = torch.tensor([0, 1, 2, n - 3, n - 2, n - 1], device=DEV)

    def among_many(t):
        many = torch.zeros(n, h, w, c, dtype=F16, device=DEV).permute(0, 3, 1, 2)
        many[ends] = t
        return many

    xs, dys = among_many(x), among_many(dy)
    y, mean, rstd = ops.group_norm_act_forward(xs, g, wt, bs, 1e-5, 'silu')
    dx, dw, db = ops.group_norm_act_backward(dys, xs, g, wt, bs, mean, rstd, 1e-5, 'silu')
    want = reference(x, g, wt, bs, 1e-5, 'silu', dy)
    for name, got in (('y', y[ends]), ('dx', dx[ends]), ('dw', dw), ('db', db)):
        assert_within(got, want[name], want['tol_' + name] + EPS32 * want[name].abs(), name)
