"""Orthogonalised updates (optim.py, csrc/qz_ortho.hip): what is refused, and the ends of the number range."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_derivatives_of_an_orthogonalised_update_are_refused(gpu_device):
    """The result is a constant to autograd, in reverse and in forward mode: an input that asks for a derivative is refused."""
    import torch.autograd.forward_ad as fwd
    from alphazero_quoridor_amd import optim

    u = torch.randn((20, 30), generator=torch.Generator().manual_seed(1)).to(gpu_device)
    want = optim.orthogonalize(u)
    p = u.clone().requires_grad_(True)
    for x in (p, p * 1, [u, p]):
        with pytest.raises(ValueError, match="detach"):
            optim.orthogonalize(x)
    with torch.no_grad():
        assert torch.equal(optim.orthogonalize(p), want)
    assert torch.equal(optim.orthogonalize(p.detach()), want) and not want.requires_grad
    with fwd.dual_level():
        dual = fwd.make_dual(u, torch.ones_like(u))
        for x in (dual, dual.t(), [u, dual]):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                optim.orthogonalize(x)
        assert torch.equal(optim.orthogonalize(fwd.unpack_dual(dual).primal), want)
