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


# (s x l in tiles of 128: sum over tiles of the lower triangle, and all tiles of X'.)  2,048 x 5,000: B in tiles of 128, its sum split;
# X' in 640 tiles, of which 128 are left over a round and run in quarters.  4,100 x 4,100: 561 lower tiles, 49 left over in quarters, in all
# three products.  3,500 x 3,600: 406 lower tiles, not split.  5,000 x 2,048: the same as a tall matrix.
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16), ids=("f32", "bf16", "f16"))
@pytest.mark.parametrize("shape", ((2048, 5000), (5000, 2048), (3500, 3600), (4100, 4100)), ids=lambda s: "%dx%d" % s)
def test_products_of_many_tiles(gpu_device, shape, dtype):
    from alphazero_quoridor_amd import optim

    u = update("decaying", *shape, 4, gpu_device).to(dtype)
    check(optim.orthogonalize(u), u)


def test_a_list_with_many_symmetric_tiles(gpu_device):
    """252 lower tiles of 128 in one launch (B in tiles of 128, whole sums), with narrow matrices in the same call."""
    from alphazero_quoridor_amd import optim

    us = [update("decaying", m, n, i, gpu_device) for i, (m, n) in enumerate([(1024, 1024)] * 6 + [(1024, 4096), (64, 576), (16, 40), (300, 700)])]
    got = optim.orthogonalize(us)
    for u, o, again in zip(us, got, optim.orthogonalize(us)):
        check(o, u)
        assert torch.equal(o, again)


def test_muon_step_of_large_matrices(gpu_device):
    """U = (1 - mu) G + mu M is rounded to float32, and M before it: 4 x 2^-24 relative to X_0, carried by at most a^5; the weight's own update
    is rounded twice."""
    from alphazero_quoridor_amd import optim

    shapes, lr, mu, wd = ((1024, 1024), (4096, 1024), (2048, 5000), (1024, 4096)), 0.02, 0.95, 0.1
    ps = [torch.nn.Parameter(0.1 * update("white", *s, 20 + i, gpu_device)) for i, s in enumerate(shapes)]
    opt = optim.Muon(ps, lr=lr, momentum=mu, weight_decay=wd)
    for step in range(2):
        for i, p in enumerate(ps):
            p.grad = update("decaying", *p.shape, 40 + 10 * step + i, gpu_device)
        before = [(p.detach().double(), p.grad.double(), opt.state[p]["momentum_buffer"].double() if step else torch.zeros_like(p, dtype=torch.float64)) for p in ps]
        opt.step()
        for p, (w, g, m) in zip(ps, before):
            m = mu * m + (1 - mu) * g
            o, e = iterate((1 - mu) * g + mu * m)
            scale = lr * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
            want = w * (1 - lr * wd) - scale * o
            off = float((p.detach().double() - want).norm())
            assert off <= scale * (e + A ** 5 * 4 * 2.0 ** -24) + 4 * 2.0 ** -24 * float(want.norm()), (tuple(p.shape), off)
            assert float((opt.state[p]["momentum_buffer"].double() - m).norm()) <= 4 * 2.0 ** -24 * 2 * float(g.norm())
