"""What the autograd nodes of layer norm, linear8 and distill_loss have to keep of a torch program's rules."""
import pytest
import torch

import kadconv

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def test_forward_mode_of_a_kept_weight_is_refused():
    x, b = randn(40, 30), randn(12, seed=2)
    q, kept = kadconv.quantize8(x), kadconv.quantize8(randn(12, 30, seed=1))
    with torch.autograd.forward_ad.dual_level():
        dual_x, dual_b = (torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, b))
        for call in (lambda: kadconv.linear8(dual_x, kept, b), lambda: kadconv.linear8(x, kept, dual_b),
                     lambda: kadconv.matmul8(q, kept, dual_b)):
            with pytest.raises(NotImplementedError, match='forward-mode'):
                call()
