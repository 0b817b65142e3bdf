"""Orthogonalised updates (optim.py, csrc/qz_ortho.hip): what is refused, and the ends of the number range."""
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


@pytest.mark.parametrize("shape", ((4, 30), (64, 80), (100, 128), (140, 150), (520, 600)), ids=lambda s: "%dx%d" % s)
def test_norms_near_the_end_of_float32(gpu_device, shape):
    """Entries of up to 3e38, whose norm lies beyond float32: the result is, bit for bit, that of the same update times 2^-120.  Squares, their
    sum, its root and its reciprocal, all in float64, scale by powers of two exactly, and so X_0 = U / |U| comes out the same."""
    from alphazero_quoridor_amd import optim

    g = torch.Generator().manual_seed(shape[0])
    u = (torch.rand(shape, generator=g) * 2 - 1).to(gpu_device)
    big = u * (2.0 ** 127 * 1.7)
    assert float(big.double().norm()) > 2.0 ** 126 and bool(torch.isfinite(big).all())
    assert torch.equal(optim.orthogonalize(big), optim.orthogonalize(big * 2.0 ** -120))


def test_negated_views(gpu_device):
    """The imaginary part of a conjugate is a view whose memory holds the other sign; nothing of it need be copied where it has one column."""
    from alphazero_quoridor_amd import optim

    c = torch.randn((30, 40), dtype=torch.complex64, generator=torch.Generator().manual_seed(2)).to(gpu_device).conj()
    for u in (c.imag, c[:, :1].imag, c[:1].imag.t(), torch._neg_view(c.real.contiguous())):
        assert u.is_neg()
        assert torch.equal(optim.orthogonalize(u), optim.orthogonalize(u.resolve_neg().contiguous()))
    p, q = (torch.nn.Parameter(torch.zeros((30, 1), device=gpu_device)) for _ in range(2))
    p.grad, q.grad = c[:, :1].imag, c[:, :1].imag.resolve_neg().contiguous()
    for x in (p, q):
        optim.Muon([x], lr=0.1).step()
    assert torch.equal(p, q)
