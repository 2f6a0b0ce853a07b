"""linear8 with more outputs than a gradient can be brought to 8 bits along: refused before any work, and where nothing needs
that, not at all."""
import pytest
import torch

import kadconv

pytestmark = pytest.mark.gpu
DEV = 'cuda'
MOST = 1 << 20


def test_refused_in_the_forward_pass():
    w = torch.ones(MOST + 1, 2, device=DEV)
    x = torch.ones(40, 2, device=DEV)
    for call in (lambda x, w, b: kadconv.linear8(x, w, b), lambda x, w, b: torch.ops.kadconv.linear8(x, w, b, None, -1)):
        for x_grad, w_grad, b_grad in ((True, False, False), (False, True, False), (False, False, True)):
            args = x.clone().requires_grad_(x_grad), w.clone().requires_grad_(w_grad), w[:, 0].clone().requires_grad_(b_grad)
            with pytest.raises(ValueError, match='1048576'):
                call(*args)
            with torch.no_grad():
                assert (call(*args) == 3).all()


def test_few_rows_have_a_gradient_of_their_own():
    """Up to 32 rows the product brings dy to 8 bits itself, in parts as long as codes may be."""
    w = torch.ones(MOST + 129, 2, device=DEV)
    x = torch.ones(3, 2, device=DEV, requires_grad=True)
    for y in (kadconv.linear8(x, w), torch.ops.kadconv.linear8(x, w, None, None, -1)):
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert (dx == MOST + 129).all()


def test_as_many_as_there_may_be():
    w = torch.ones(MOST, 2, device=DEV, requires_grad=True)
    x = torch.ones(40, 2, device=DEV, requires_grad=True)
    b = torch.zeros(MOST, device=DEV, requires_grad=True)
    y = kadconv.linear8(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert (dx == MOST).all() and (dw == 40).all() and (db == 40).all()


def test_no_rows():
    w = torch.ones(MOST + 1, 2, device=DEV, requires_grad=True)
    x = torch.ones(0, 2, device=DEV)
    for y in (kadconv.linear8(x, w), torch.ops.kadconv.linear8(x, w, None, None, -1)):
        assert not torch.autograd.grad(y, w, torch.ones_like(y))[0].any()
