"""GPU parity of the orthogonalised update and the Muon step (optim.py, csrc/qz_ortho.hip) against the iteration in float64.

Tolerance, in the 2-norm over all entries (F).  One step is X' = a X + B X, B = b A + c A A, A = X X^T.  With v = 2^-22 the
relative size of what a split operand loses (hi + lo of two fp16 numbers) and float32 accumulation below that, a product P Q is off by
at most 4 v |P|_F |Q|_2 (two operands, the dropped lo lo, the accumulation); so A is off by 4 v |X|_F |X|_2, B by
|b| dA + 2 |c| |A|_2 dA + 4 v |c| |A|_F |A|_2 + v |B|_F, and X' by a v |X|_F + dB |X|_2 + 4 v |B|_F |X|_2.  What a step adds is carried on
by the steps behind it, each a map whose derivative is at most L = a + |b| s^2 + |c| s^4 with s = |X|_2 (as a product of norms it
grows past what any matrix shows: the first-order bound a sup |f'| <= a = 3.4445 on [0, 1.3] is used, sup |a + 3 b s^2 + 5 c s^4| there).
bfloat16 results with a shorter side >= 256 use operands of 11 bits: v = 2^-11 in the products, 2^-22 in a X.  The result's own
rounding adds half a step of its type."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315


def gradient(m, n, seed, noise=0.3):
    g = torch.Generator().manual_seed(seed)
    r = max(1, min(m, n) // 8)
    s = (torch.randn((m, r), generator=g) * torch.exp(-3.0 * torch.arange(r) / r)) @ torch.randn((r, n), generator=g)
    e = torch.randn((m, n), generator=g)
    return 1e-3 * (s / s.norm() + noise * e / e.norm())


def spectral(m):
    return float(torch.linalg.eigvalsh(m @ m.t() if m.shape[0] <= m.shape[1] else m.t() @ m).clamp(min=0).max().sqrt())


def iterate(u, steps, v):
    """-> (float64 result, bound of the error in the 2-norm over all entries)"""
    x = u.double()
    x = x if x.shape[0] <= x.shape[1] else x.t()
    x = x / max(float(x.norm()), 1e-7)
    bound, v0 = 2.0 ** -22 * float(x.norm()), 2.0 ** -22
    for _ in range(steps):
        a = x @ x.t()
        b = B * a + C * (a @ a)
        xf, x2, af, a2, bf = float(x.norm()), spectral(x), float(a.norm()), spectral(a), float(b.norm())
        da = 4 * v * xf * x2
        db = abs(B) * da + 2 * C * a2 * da + 4 * v * C * af * a2 + v * bf
        bound = bound * A + A * v0 * xf + db * x2 + 4 * v * bf * x2
        x = A * x + b @ x
    return (x if u.shape[0] <= u.shape[1] else x.t()), bound


def check(got, u, steps=5):
    one = u.dtype == torch.bfloat16 and min(u.shape) >= 256
    want, bound = iterate(u.cpu(), steps, 2.0 ** -11 if one else 2.0 ** -22)
    bound += (0 if u.dtype == torch.float32 else torch.finfo(u.dtype).eps / 2) * float(want.norm()) + (2.0 ** -25 * math.sqrt(want.numel()) if u.dtype == torch.float16 else 0)
    off = float((got.double().cpu() - want).norm())
    assert off <= bound, "%s %s: off by %.3g, bound %.3g" % (tuple(u.shape), u.dtype, off, bound)
    return off, bound


SHAPES = ((1, 1), (1, 2), (2, 1), (1, 128), (3, 5), (4, 576), (2, 576), (15, 17), (16, 16), (17, 300), (31, 33), (63, 64), (64, 64), (64, 234), (64, 576), (65, 64),
          (65, 500), (128, 324), (129, 127), (140, 162), (300, 100), (700, 33), (255, 257), (256, 256), (384, 260), (511, 513), (513, 520), (700, 640), (1030, 520))


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16), ids=("f32", "bf16", "f16"))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_orthogonalize(gpu_device, shape, dtype):
    from alphazero_quoridor_amd import optim

    u = gradient(*shape, seed=shape[0] * 7 + shape[1]).to(dtype)
    check(optim.orthogonalize(u.to(gpu_device)), u)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16), ids=("f32", "bf16"))
@pytest.mark.parametrize("shape", ((10, 9000), (16, 8192), (16, 8193), (20, 9000), (40, 2048), (40, 2049), (64, 2100), (100, 512), (100, 513), (128, 600), (130, 9000), (9000, 130),
                                   (600, 5000), (5000, 520), (1, 70001), (1024, 4100)), ids=lambda s: "%dx%d" % s)
def test_long_sides(gpu_device, shape, dtype):
    """Both sides of every border between the ways a matrix is worked on, and sums split over workgroups."""
    from alphazero_quoridor_amd import optim

    u = gradient(*shape, seed=shape[0] * 7 + shape[1]).to(dtype)
    check(optim.orthogonalize(u.to(gpu_device)), u)


@pytest.mark.parametrize("shape", ((256, 1024), (320, 2500), (1536, 384), (700, 640), (512, 4096), (1023, 1100), (1024, 8192), (4097, 1024)), ids=lambda s: "%dx%d" % s)
def test_bfloat16_results_lose_no_more_than_their_rounding(gpu_device, shape):
    """Where the shorter side is short, or the longer long beside it, a 16-bit result is as near as the three products of float32
    results bring it.  Tolerance: with x the kernel's value before rounding, |x - want| = e, the stored value is the nearest to x, so
    |got - want| <= |got - x| + e <= |bf16(want) - x| + e <= |bf16(want) - want| + 2 e, and e is the split operands' bound."""
    from alphazero_quoridor_amd import optim

    u = gradient(*shape, seed=shape[0] * 7 + shape[1]).bfloat16()
    want, bound = iterate(u, 5, 2.0 ** -22)
    bound = float((want.bfloat16().double() - want).norm()) + 2 * bound
    off = float((optim.orthogonalize(u.to(gpu_device)).double().cpu() - want).norm())
    assert off <= bound, "%s: off by %.3g, bound %.3g" % (shape, off, bound)


def test_orthogonalize_a_list_equals_its_members(gpu_device):
    """More matrices than one launch takes, of all sizes and types, tall and wide, in one call."""
    from alphazero_quoridor_amd import optim

    us = [gradient(m, n, seed=i) for i, (m, n) in enumerate(list(SHAPES[:26]) + [(64, 64)] * 30)]
    us = [u.to((torch.float32, torch.bfloat16)[i % 2]).to(gpu_device) for i, u in enumerate(us)]
    us[5] = us[4]  # the same tensor twice
    got = optim.orthogonalize(us)
    for u, o in zip(us, got):
        assert torch.equal(o, optim.orthogonalize(u)) and o.dtype == u.dtype and o.shape == u.shape
    assert optim.orthogonalize([]) == []


@pytest.mark.parametrize("steps", (1, 2, 3, 7, 16))
def test_number_of_steps(gpu_device, steps):
    from alphazero_quoridor_amd import optim

    for shape in ((4, 30), (64, 100), (140, 162), (520, 513)):
        u = gradient(*shape, seed=steps)
        if steps <= 7:
            check(optim.orthogonalize(u.to(gpu_device), steps=steps), u, steps)
        else:  # (the first-order bound has grown past use: the result must still be near orthogonal)
            o = optim.orthogonalize(u.to(gpu_device), steps=steps).double().cpu()
            s = torch.linalg.svdvals(o)
            assert float(s.max()) < 1.3 and float(s.min()) > 0.5


def test_special_values(gpu_device):
    from alphazero_quoridor_amd import optim

    for shape in ((3, 7), (64, 80), (80, 64), (140, 150), (520, 600)):
        zero = torch.zeros(shape, device=gpu_device)
        assert (optim.orthogonalize(zero) == 0).all()
        assert (optim.orthogonalize(zero.bfloat16()) == 0).all()
        u = gradient(*shape, seed=1).to(gpu_device)
        # the scale of the update does not matter: powers of two from the smallest to the largest float32 magnitudes
        for k in (-100, -20, 20, 120):
            v = u * 2.0 ** k
            if float(v.norm().double()) > 1e-7 and bool((v.abs()[u != 0] > 2.0 ** -126).all()):
                assert torch.equal(optim.orthogonalize(v), optim.orthogonalize(u)), k
        big = torch.full(shape, 3e38, device=gpu_device)  # |U|_F and U U^T leave float32's range; rank one
        check(optim.orthogonalize(big), big)
        tiny = u * 1e-10  # below the floor of the norm: U / 1e-7
        want = tiny.double().cpu() / 1e-7 if float(tiny.double().norm()) < 1e-7 else None
        if want is not None:
            x = want if shape[0] <= shape[1] else want.t()
            for _ in range(5):
                a = x @ x.t()
                x = A * x + (B * a + C * (a @ a)) @ x
            x = x if shape[0] <= shape[1] else x.t()
            off = float((optim.orthogonalize(tiny).double().cpu() - x).norm())
            # entries near 2^-37 of the scaled planes' unit are kept to 2^-37 absolute each, carried by a^5
            assert off <= A ** 5 * 2.0 ** -37 * math.sqrt(x.numel()) + iterate(u.cpu(), 5, 2.0 ** -22)[1], off
        for bad in (math.nan, math.inf):
            v = u.clone()
            v[-1, -1] = bad
            assert torch.isnan(optim.orthogonalize(v)).all()


def test_rank_deficient_and_repeated_rows(gpu_device):
    from alphazero_quoridor_amd import optim

    for shape in ((64, 576), (576, 64), (140, 162), (530, 600)):
        g = torch.Generator().manual_seed(2)
        low = (torch.randn((shape[0], 3), generator=g) @ torch.randn((3, shape[1]), generator=g))
        check(optim.orthogonalize(low.to(gpu_device)), low)
        rep = torch.randn((1, shape[1]), generator=g).repeat(shape[0], 1)
        check(optim.orthogonalize(rep.to(gpu_device)), rep)
        gap = gradient(*shape, seed=3)
        gap[shape[0] // 2:] = 0
        check(optim.orthogonalize(gap.to(gpu_device)), gap)


def test_strided_and_convolution_shapes(gpu_device):
    from alphazero_quoridor_amd import optim

    for dtype in (torch.float32, torch.bfloat16):
        base = gradient(200, 700, seed=9).to(dtype).to(gpu_device)
        for v in (base[3:67, 5:500], base[::2, 1:600], base[:100, :300].t(), base[:64].view(64, 7, 10, 10), base[:, 0:699]):
            want = optim.orthogonalize(v.reshape(v.shape[0], -1).contiguous())
            got = optim.orthogonalize(v)
            assert got.shape == v.shape and torch.equal(got.reshape(v.shape[0], -1), want)
        rows = base[:1, :90].expand(70, 90)  # one row for all
        assert torch.equal(optim.orthogonalize(rows), optim.orthogonalize(rows.contiguous()))
    assert optim.orthogonalize(torch.zeros((0, 5), device=gpu_device)).shape == (0, 5)
    assert optim.orthogonalize([torch.zeros((5, 0, 3), device=gpu_device), base])[0].shape == (5, 0, 3)


def muon64(p, g, m, lr, mu, nesterov, wd, adjust):
    m = mu * m.double() + (1 - mu) * g.double()
    u = (1 - mu) * g.double() + mu * m if nesterov else m
    o, bound = iterate(u.reshape(u.shape[0], -1), 5, 2.0 ** -22)
    rows, cols = o.shape
    scale = math.sqrt(max(1.0, rows / cols)) if adjust == "original" else 0.2 * math.sqrt(max(rows, cols))
    # u is rounded to float32 (and m before it): 3 u24 relative, which the steps carry like an error of X_0
    bound += A ** 5 * 4 * 2.0 ** -24
    return p.double() * (1 - lr * wd) - lr * scale * o.reshape(p.shape), m, lr * scale * bound


@pytest.mark.parametrize("nesterov", (True, False))
@pytest.mark.parametrize("adjust", ("original", "match_rms_adamw"))
@pytest.mark.parametrize("gtype", (torch.float32, torch.bfloat16, torch.float16), ids=("f32", "bf16", "f16"))
def test_muon_steps(gpu_device, nesterov, adjust, gtype):
    """Three steps, each against the formulas from the state that the step before it left."""
    from alphazero_quoridor_amd import optim

    shapes = ((64, 26, 3, 3), (64, 576), (4, 64, 3, 3), (128, 324), (140, 162), (324, 128), (520, 600), (1, 9))
    ps = [torch.nn.Parameter((torch.randn(s, generator=torch.Generator().manual_seed(i)) * 0.1).to(gpu_device)) for i, s in enumerate(shapes)]
    for p in ps:
        p.grad_dtype = gtype  # gradients in another type than their weight's
    idle = torch.nn.Parameter(torch.ones((5, 5), device=gpu_device))  # no gradient: left alone
    opt = optim.Muon(ps + [idle], lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, adjust_lr=adjust)
    for step in range(3):
        for i, p in enumerate(ps):
            p.grad = (gradient(p.shape[0], p.numel() // p.shape[0], seed=10 * step + i) * 100).reshape(p.shape).to(gtype).to(gpu_device)
        before = [(p.detach().cpu().clone(), p.grad.cpu(), opt.state[p]["momentum_buffer"].cpu().clone() if step else torch.zeros(p.shape)) for p in ps]
        version = ps[0]._version
        opt.step()
        assert ps[0]._version > version
        for p, (w, g, m) in zip(ps, before):
            want, mom, tol = muon64(w, g, m, 0.02, 0.9, nesterov, 0.1, adjust)
            got = p.detach().double().cpu()
            off = float((got - want).norm())
            assert off <= tol + 4 * 2.0 ** -24 * float(want.norm()), (tuple(p.shape), off, tol)
            assert float((opt.state[p]["momentum_buffer"].double().cpu() - mom).norm()) <= 4 * 2.0 ** -24 * (float(mom.norm()) + float(m.norm()) + float(g.double().norm()))
    assert (idle == 1).all() and idle not in opt.state


def test_muon_state_round_trip_and_learning_rate_on_the_device(gpu_device):
    from alphazero_quoridor_amd import optim

    def make(lr):
        p = torch.nn.Parameter(gradient(64, 100, 5).to(gpu_device) * 100)
        return p, optim.Muon([p], lr=lr, weight_decay=0.01)

    grads = [gradient(64, 100, 20 + i).to(gpu_device) for i in range(4)]
    a, oa = make(0.02)
    b, ob = make(torch.tensor(0.02, device=gpu_device))
    for g in grads[:2]:
        a.grad, b.grad = g, g
        oa.step()
        ob.step()
    assert torch.equal(a, b)
    c, oc = make(0.5)
    with torch.no_grad():
        c.copy_(a)
    oc.load_state_dict(copy.deepcopy(oa.state_dict()))  # (a state dict holds the live buffers themselves)
    for g in grads[2:]:
        a.grad = c.grad = g
        oa.step()
        oc.step()
    assert torch.equal(a, c)


def test_captured_step_follows_the_learning_rate(gpu_device):
    from alphazero_quoridor_amd import optim

    shapes = ((64, 576), (4, 576), (140, 162), (520, 530))
    def fresh():
        return [torch.nn.Parameter((torch.randn(s, generator=torch.Generator().manual_seed(i))).to(gpu_device)) for i, s in enumerate(shapes)]

    eager, static = fresh(), fresh()
    lr = torch.tensor(0.01, device=gpu_device)
    oe, og = optim.Muon(eager, lr=0.01), optim.Muon(static, lr=lr)
    grads = [[gradient(*s, seed=100 * k + i).to(gpu_device) for i, s in enumerate(shapes)] for k in range(4)]
    for p, s, g in zip(eager, static, grads[0]):
        p.grad, s.grad = g.clone(), g.clone()
        og.state[s]["momentum_buffer"] = torch.zeros_like(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        og.step()
    for k in range(4):
        rate = 0.01 * (k + 1)
        oe.param_groups[0]["lr"] = rate
        lr.fill_(rate)
        for p, s, g in zip(eager, static, grads[k]):
            p.grad.copy_(g)
            s.grad.copy_(g)
        oe.step()
        graph.replay()
        torch.cuda.synchronize()
        for p, s in zip(eager, static):
            # lr arrives as a float64 rounded to float32 on both ways
            assert torch.equal(p, s), k


def test_first_step_in_a_capture_and_shared_memory_are_refused(gpu_device):
    from alphazero_quoridor_amd import optim

    p = torch.nn.Parameter(gradient(64, 64, 1).to(gpu_device))
    p.grad = gradient(64, 64, 2).to(gpu_device)
    opt = optim.Muon([p])
    before = p.detach().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before the capture"):
            opt.step()
    assert torch.equal(p, before)
    q = torch.nn.Parameter(p.detach())
    q.grad = p.grad
    with pytest.raises(ValueError, match="share their memory"):
        optim.Muon([p, q]).step()
    assert torch.equal(p, before)


def test_overlapping_parameters_are_refused(gpu_device):
    """Two weights that share some of their memory, neither starting where the other does."""
    from alphazero_quoridor_amd import optim

    whole = gradient(96, 64, 1).to(gpu_device)
    before = whole.clone()
    for cuts in (((0, 64), (32, 96)), ((32, 96), (0, 64)), ((0, 96), (40, 50))):
        ps = [torch.nn.Parameter(whole[a:b]) for a, b in cuts]
        for p in ps:
            p.grad = torch.ones_like(p)
        with pytest.raises(ValueError, match="share their memory"):
            optim.Muon(ps).step()
    assert torch.equal(whole, before)
    ps = [torch.nn.Parameter(whole[a:b]) for a, b in ((48, 96), (0, 48))]  # side by side is fine
    for p in ps:
        p.grad = torch.ones_like(p)
    optim.Muon(ps).step()
    assert not torch.equal(whole[:48], before[:48]) and not torch.equal(whole[48:], before[48:])


def test_two_lists_on_two_streams(gpu_device):
    from alphazero_quoridor_amd import optim

    lists = [[gradient(m, n, seed=k * 50 + i).to(gpu_device) for i, (m, n) in enumerate(((64, 576), (140, 162), (520, 600)))] for k in range(2)]
    want = [optim.orthogonalize(x) for x in lists]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        got = []
        for s, x in zip(streams, lists):
            with torch.cuda.stream(s):
                got.append(optim.orthogonalize(x))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for g, w in zip(got, want) for p, q in zip(g, w))


def test_refusals_on_the_device(gpu_device):
    from alphazero_quoridor_amd import _cabi, optim

    x = torch.zeros((4, 5), device=gpu_device)
    for bad, error in ((x[0], ValueError), (x.double(), TypeError), (x.cpu(), _cabi.QzError), (x.int(), TypeError)):
        with pytest.raises(error):
            optim.orthogonalize(bad)
    for steps in (0, 17, -1):
        with pytest.raises(ValueError):
            optim.orthogonalize(x, steps=steps)
    p = torch.nn.Parameter(x.clone())
    p.grad = torch.zeros((4, 5), device=gpu_device)
    opt = optim.Muon([p], lr=torch.tensor(0.1, device=gpu_device, dtype=torch.float64))
    with pytest.raises(ValueError):
        opt.step()
    opt = optim.Muon([p])
    opt.state[p]["momentum_buffer"] = torch.zeros((5, 4), device=gpu_device)
    with pytest.raises(ValueError):
        opt.step()
