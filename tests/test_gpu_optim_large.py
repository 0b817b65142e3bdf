"""GPU parity of orthogonalised updates at the sizes that run in many tiles (optim.py, csrc/qz_ortho.hip), against the iteration in
float64, on updates of several kinds of spectrum.

Tolerance, in the 2-norm over all entries (F), with v = 2^-22 the relative size of what a split operand (hi + lo, two fp16 numbers)
loses.  A product P Q is off by at most 4 v |P|_F |Q|_2: two operands, the dropped lo lo, the float32 accumulation below that.  So
A = X X^T is off by dA = 4 v |X|_F |X|_2, B = b A + c A A by dB = |b| dA + 2 |c| |A|_2 dA + 4 v |c| |A|_F |A|_2 + v |B|_F, and X' by
a v |X|_F + dB |X|_2 + 4 v |B|_F |X|_2; the steps behind carry an error by at most sup |p'| = a = 3.4445, with p the step's polynomial.
p maps [0, 1] into [0, 1.2024], and that interval into itself, so |X|_2 <= 1.2024 throughout: no spectrum has to be computed.
A result x stored in 16 bits is the nearest to x, and |x - want| <= e, so |got - want| <= |got - x| + e <= |type(want) - x| + e
<= |type(want) - want| + 2 e."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
V, TOP = 2.0 ** -22, 1.2024


def update(kind, m, n, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    e = torch.randn((m, n), generator=g, device=device)
    if kind == "white":
        return e
    if kind == "sparse":  # one entry in a hundred
        return torch.where(torch.rand((m, n), generator=g, device=device) < 0.01, e, torch.zeros_like(e))
    if kind == "repeated":  # every row eight times, but for a little noise: most singular values small, the others large
        return e[: (m + 7) // 8].repeat_interleave(8, 0)[:m] + 0.01 * torch.randn((m, n), generator=g, device=device)
    r = min(m, n) // 8  # decaying directions under noise
    s = (torch.randn((m, r), generator=g, device=device) * torch.exp(-3.0 * torch.arange(r, device=device) / r)) @ torch.randn((r, n), generator=g, device=device)
    return 1e-3 * (s / s.norm() + 0.3 * e / e.norm())


def iterate(u, steps=5):
    """-> (float64 result, bound of the error over all entries)"""
    x = u.double()
    x = x if x.shape[0] <= x.shape[1] else x.t()
    x = (x / max(float(x.norm()), 1e-7)).contiguous()
    bound, x2 = V * float(x.norm()), 1.0
    for _ in range(steps):
        a = x @ x.t()
        b = B * a + C * (a @ a)
        xf, af, bf = float(x.norm()), float(a.norm()), float(b.norm())
        da = 4 * V * xf * x2
        db = abs(B) * da + 2 * C * x2 * x2 * da + 4 * V * C * af * x2 * x2 + V * bf
        bound = bound * A + A * V * xf + db * x2 + 4 * V * bf * x2
        x, x2 = A * x + b @ x, TOP
    return (x if u.shape[0] <= u.shape[1] else x.t()), bound


def check(got, u, steps=5):
    want, e = iterate(u, steps)
    bound = e if u.dtype == torch.float32 else float((want.to(u.dtype).double() - want).norm()) + 2 * e
    off = float((got.double() - want).norm())
    assert math.isfinite(off) and off <= bound, "%s %s: off by %.4g of %.4g, bound %.4g" % (tuple(u.shape), u.dtype, off, float(want.norm()), bound)


@pytest.mark.parametrize("kind", ("white", "sparse", "repeated", "decaying"))
@pytest.mark.parametrize("shape", ((1024, 1024), (1024, 4096), (4096, 1024), (1100, 1500), (2048, 2050)), ids=lambda s: "%dx%d" % s)
def test_bfloat16_results_lose_no_more_than_their_rounding_whatever_the_spectrum(gpu_device, shape, kind):
    from alphazero_quoridor_amd import optim

    u = update(kind, *shape, 3, gpu_device).bfloat16()
    check(optim.orthogonalize(u), u)
