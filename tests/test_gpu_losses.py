"""GPU parity of the policy losses (losses.py, csrc/qz_policy.hip) against their definitions in float64.

Tolerances.  u = 2^-24.  A row's sum of exponentials is a chain of at most 40 float32 additions per thread and tree plus 1 ulp per
exponential and logarithm, so s is good to 64 u relative; lse, z - lse and the action's log-probability add the rounding of values
of size max|z|: delta = 64 u (1 + max|z|) bounds the absolute error of a log-probability.  A probability is then good to
2 delta relative, a ratio to delta, and a gradient entry w [c (d - p) + beta (p - q) + eta p (log p + H)] to
2 delta w [ (|c| + |beta| + |eta| (|log p| + H + 2)) (p + q) + |c| d ], plus half a step of its own type.  In KL, sum q f(x), an
error of x counts with |p - q|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def pack(legal):
    n, a = legal.shape
    w = (torch.nn.functional.pad(legal, (0, -a % 32)).view(n, -1, 32).long() << torch.arange(32)).sum(2)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def make(n, a, dtype, seed, legal_share=0.6, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn((n, a), generator=g) * spread).to(dtype)
    legal = torch.rand((n, a), generator=g) < legal_share
    actions = torch.randint(0, a, (n,), generator=g)
    legal[torch.arange(n), actions] = True
    d = {"z": z, "legal": legal, "actions": actions, "adv": torch.randn(n, generator=g), "old": torch.randn(n, generator=g) * 0.2 - 2.0,
         "w": torch.rand(n, generator=g), "ref": (z.float() + 0.3 * torch.randn((n, a), generator=g)).to(dtype), "ref_logp": torch.randn(n, generator=g) * 0.3 - 2.0}
    return d


def definition(d, masked, kl, clip, kl_coef, ent_coef):
    """float64, on the CPU; with the elementwise tolerances"""
    z, ok = d["z"].double(), d["legal"] if masked else torch.ones_like(d["legal"])
    n, a = z.shape
    acts = d["actions"]
    inr = (acts >= 0) & (acts < a)
    at = acts.clamp(0, a - 1)
    live = inr & ok[torch.arange(n), at] & (z[torch.arange(n), at] != -math.inf)
    zm = torch.where(ok, z, torch.full_like(z, -math.inf))
    safe = torch.where(live[:, None], zm, torch.zeros_like(zm))
    lp = torch.log_softmax(safe, 1)
    p = torch.exp(lp)
    lp0 = torch.where(p > 0, lp, torch.zeros_like(lp))
    h = -(p * lp0).sum(1)
    logp = lp[torch.arange(n), at]
    w = d["w"].double()
    out = {}
    top = torch.where(torch.isfinite(safe), safe.abs(), torch.zeros_like(safe)).max(1).values
    delta = 64 * U * (1 + top)
    adv = d["adv"].double()
    r = torch.exp(logp - d["old"].double())
    held = r.clamp(1 - clip[0], 1 + clip[1]) * adv
    loss = -torch.minimum(r * adv, held)
    c = torch.where(held < r * adv, torch.zeros_like(r), -r * adv)
    q, klv, cols_tol = torch.zeros_like(p), torch.zeros(n, dtype=torch.float64), 0.0
    if kl == "full":
        zq = torch.where(live[:, None], torch.where(ok, d["ref"].double(), torch.full_like(z, -math.inf)), torch.zeros_like(z))
        lq = torch.log_softmax(zq, 1)
        q = torch.exp(lq)
        klv = torch.where(q > 0, q * (torch.where(q > 0, lq, 0.0) - lp), torch.zeros_like(q)).sum(1)
        cols_tol = 3 * delta * (p - q).abs().sum(1) + 64 * U * klv
    elif kl == "taken":
        x = d["ref_logp"].double() - logp
        klv = torch.exp(x) - 1 - x
        c = c - kl_coef * (torch.exp(x) - 1)
        cols_tol = delta * (torch.exp(x) - 1).abs() + 16 * U * (1 + klv)
    onehot = torch.zeros_like(p)
    onehot[torch.arange(n), at] = 1.0
    beta = kl_coef if kl == "full" else 0.0
    grad = w[:, None] * (c[:, None] * (onehot - p) + beta * (p - q) + ent_coef * p * (lp0 + h[:, None]))
    cdel = (c.abs() + (kl_coef if kl == "taken" else 0.0))[:, None]
    tol = 2 * (delta * w)[:, None] * ((cdel + abs(beta) + abs(ent_coef) * (lp0.abs() + h[:, None] + 2)) * (p + q) + cdel * onehot)
    row = w * (loss + kl_coef * klv - ent_coef * h)
    row = torch.where(live & (w != 0), row, torch.zeros_like(row))
    row_tol = torch.where(live, w * (delta * (c.abs() + ent_coef * 2) + kl_coef * cols_tol + 16 * U * (loss.abs() + h + klv)), torch.zeros_like(w))
    zero = torch.zeros_like(h)
    grad = torch.where((live & (w != 0))[:, None] & ok, grad, torch.zeros_like(grad))
    out = {"loss": row.sum(), "loss_tol": row_tol.sum() + 2 * U * row.sum().abs(), "logp": torch.where(live, logp, torch.where(acts < 0, 0.0, -math.inf)),
           "logp_tol": delta, "entropy": torch.where(live, h, zero), "entropy_tol": 2 * delta * (1 + h), "kl": torch.where(live, klv, zero), "kl_tol": cols_tol,
           "grad": grad, "grad_tol": tol, "live": live, "p": p, "lp": lp0, "h": h, "ok": ok}
    return out


def close(got, want, tol, what):
    got, want = got.double().cpu(), want
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    d = torch.where(same, torch.zeros_like(want), (got - want).abs())
    assert not torch.isnan(d).any(), what
    worst = (d - tol).max() if d.numel() else torch.tensor(-1.0)
    assert worst <= 0, "%s: off by %.3g past the tolerance (largest error %.3g)" % (what, float(worst), float(d.max()))


def stored(want, dtype):
    """A value past a type's largest one by half a step or more is rounded to infinity (float16: 65,520)."""
    edge = torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4)
    return torch.where(want.abs() >= edge, torch.full_like(want, math.inf) * torch.sign(want), want)


def grad_tolerance(e, dtype):
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half * 2
    return e["grad_tol"] * (1 + half) + half * e["grad"].abs() + tiny


WIDTHS = (1, 2, 3, 31, 32, 33, 63, 64, 65, 140, 191, 193, 255, 257, 511, 1000, 1024, 1025, 2048, 2051, 4096, 5001, 8192, 16387, 32768, 40003)


@pytest.mark.parametrize("a", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES, ids=("f32", "bf16", "f16"))
def test_loss_and_gradient_against_the_definition(gpu_device, a, dtype):
    from alphazero_quoridor_amd import losses

    n = 5 if a > 4096 else 37
    for k, (kind, kl, clip) in enumerate((("none", "full", (0.2, 0.2)), ("bits", "taken", (0.1, 0.3)), ("bytes", "full", (0.2, 0.28)), ("none", "none", (0.2, 0.2)),
                                          ("bits", "full", (1.0, 0.0)))):
        d = make(n, a, dtype, 100 * k + a)
        d["w"][0] = 0.0
        if n > 3:
            d["actions"][1], d["actions"][2] = -1, a  # padding; out of range
            d["legal"][3, d["actions"][3]] = False    # an illegal action
            d["legal"][4] = False                     # nothing legal
        e = definition(d, kind != "none", kl, clip, 0.05, 0.02)
        dev = {key: v.to(gpu_device) for key, v in d.items()}
        legal = None if kind == "none" else dev["legal"] if kind == "bytes" else pack(d["legal"]).to(gpu_device)
        z = dev["z"].clone()
        if kind != "none":  # what illegal columns hold is never used
            z[~dev["legal"]] = float("nan")
        z.requires_grad_(True)
        out = losses.clipped_policy_loss(z, dev["actions"], dev["adv"], dev["old"], legal=legal, weights=dev["w"], ref_logits=dev["ref"] if kl == "full" else None,
                                         ref_logp=dev["ref_logp"] if kl == "taken" else None, clip=clip, kl_coef=0.05, entropy_coef=0.02)
        out.loss.backward()
        what = "%s %s a=%d" % (kind, kl, a)
        close(out.loss.detach(), e["loss"], e["loss_tol"], what + " loss")
        close(out.logp, e["logp"], e["logp_tol"], what + " logp")
        close(out.entropy, e["entropy"], e["entropy_tol"], what + " entropy")
        close(out.kl, e["kl"], e["kl_tol"], what + " kl")
        close(z.grad, e["grad"], grad_tolerance(e, dtype), what + " grad")
        plain = losses.clipped_policy_loss(z.detach(), dev["actions"], dev["adv"], dev["old"], legal=legal, weights=dev["w"], ref_logits=dev["ref"] if kl == "full" else None,
                                           ref_logp=dev["ref_logp"] if kl == "taken" else None, clip=clip, kl_coef=0.05, entropy_coef=0.02)
        assert torch.equal(plain.logp, out.logp) and torch.equal(plain.entropy, out.entropy)
        close(plain.loss, e["loss"], e["loss_tol"], what + " loss without a gradient")


@pytest.mark.parametrize("a", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES, ids=("f32", "bf16", "f16"))
def test_action_logp_and_its_gradient(gpu_device, a, dtype):
    from alphazero_quoridor_amd import losses

    n = 3 if a > 4096 else 41
    for k, kind in enumerate(("none", "bits", "bytes")):
        d = make(n, a, dtype, 7 * k + a)
        d["actions"][0] = -100
        if n > 3:
            d["actions"][1], d["legal"][3] = a + 7, False
        e = definition(d, kind != "none", "none", (0.2, 0.2), 0.0, 0.0)
        dev = {key: v.to(gpu_device) for key, v in d.items()}
        legal = None if kind == "none" else dev["legal"] if kind == "bytes" else pack(d["legal"]).to(gpu_device)
        z = dev["z"].clone().requires_grad_(True)
        logp, ent = losses.action_logp(z, dev["actions"], legal=legal, entropy=True)
        close(logp.detach(), e["logp"], e["logp_tol"], "%s logp" % kind)
        close(ent.detach(), e["entropy"], e["entropy_tol"], "%s entropy" % kind)
        g, hh = dev["adv"], dev["old"]
        torch.autograd.backward((logp, ent), (g, hh))
        g64, h64, p, lp, h = d["adv"].double(), d["old"].double(), e["p"], e["lp"], e["h"]
        onehot = torch.zeros_like(p)
        onehot[torch.arange(n), d["actions"].clamp(0, a - 1)] = 1.0
        want = g64[:, None] * (onehot - p) - h64[:, None] * p * (lp + h[:, None])
        on = e["live"][:, None] & e["ok"]
        want = torch.where(on, want, torch.zeros_like(want))
        tol = 2 * e["logp_tol"][:, None] * ((g64.abs()[:, None] + h64.abs()[:, None] * (lp.abs() + h[:, None] + 2)) * p) + 4 * U * g64.abs()[:, None] * onehot
        half = torch.finfo(dtype).eps / 2
        close(z.grad, want, tol * (1 + half) + half * want.abs() + torch.finfo(dtype).smallest_normal * half * 2, "%s grad" % kind)
        assert torch.equal(losses.action_logp(z.detach(), dev["actions"], legal=legal), logp.detach())
        # only one of the two outputs takes part
        z2 = dev["z"].clone().requires_grad_(True)
        losses.action_logp(z2, dev["actions"], legal=legal).sum().backward()
        z3 = dev["z"].clone().requires_grad_(True)
        losses.action_logp(z3, dev["actions"], legal=legal, entropy=True)[0].sum().backward()
        assert torch.equal(z2.grad, z3.grad)


@pytest.mark.parametrize("n,a,dtype", ((70, 66003, torch.bfloat16), (70, 66003, torch.float32), (65, 33001, torch.float16), (65, 33001, torch.float32), (64, 131072, torch.bfloat16),
                                       (1, 131071, torch.float32), (1030, 1500, torch.bfloat16), (1030, 8200, torch.float32)), ids=str)
def test_many_and_few_wide_rows(gpu_device, n, a, dtype):
    """The forms that go by the number of rows as well: rows past the registers, few rows split over workgroups, many wide ones."""
    from alphazero_quoridor_amd import losses

    d = make(n, a, dtype, n + a)
    if n > 2:
        d["actions"][1], d["legal"][2] = -1, False
    dev = {key: v.to(gpu_device) for key, v in d.items()}
    for kind, kl in (("bits", "full"), ("none", "taken")):
        e = definition(d, kind != "none", kl, (0.2, 0.2), 0.05, 0.02)
        legal = pack(d["legal"]).to(gpu_device) if kind == "bits" else None
        kw = dict(ref_logits=dev["ref"]) if kl == "full" else dict(ref_logp=dev["ref_logp"])
        out, grad = losses.policy_loss_and_grad(dev["z"], dev["actions"], dev["adv"], dev["old"], legal=legal, weights=dev["w"], kl_coef=0.05, entropy_coef=0.02, **kw)
        for name in ("loss", "logp", "entropy", "kl"):
            close(getattr(out, name), e[name], e[name + "_tol"], "%s %s" % (kind, name))
        close(grad, stored(e["grad"], dtype), grad_tolerance(e, dtype), "%s grad" % kind)
        z = dev["z"].clone().requires_grad_(True)
        logp, ent = losses.action_logp(z, dev["actions"], legal=legal, entropy=True)
        close(logp.detach(), e["logp"], e["logp_tol"], "%s action_logp" % kind)
        close(ent.detach(), e["entropy"], e["entropy_tol"], "%s action entropy" % kind)
        torch.autograd.backward((logp, ent), (dev["adv"], dev["old"]))
        g64, h64 = d["adv"].double(), d["old"].double()
        onehot = torch.zeros_like(e["p"])
        onehot[torch.arange(n), d["actions"].clamp(0, a - 1)] = 1.0
        want = g64[:, None] * (onehot - e["p"]) - h64[:, None] * e["p"] * (e["lp"] + e["h"][:, None])
        want = torch.where(e["live"][:, None] & e["ok"], want, torch.zeros_like(want))
        tol = 2 * e["logp_tol"][:, None] * ((g64.abs()[:, None] + h64.abs()[:, None] * (e["lp"].abs() + e["h"][:, None] + 2)) * e["p"]) + 4 * U * g64.abs()[:, None] * onehot
        half = torch.finfo(dtype).eps / 2
        close(z.grad, want, tol * (1 + half) + half * want.abs() + torch.finfo(dtype).smallest_normal * half * 2, "%s action_logp grad" % kind)


def test_gradient_against_differences(gpu_device):
    """d loss / d z_j against central differences of the kernel's own loss.  Step h = 2^-6: the truncation is below
    h^2 / 6 |L'''| <= 4.1e-5 (|L'''| <= 1 here: weights sum to 1, |A| r <= 3 ... bounded with room by 8 max|w c|), the rounding of the two
    losses below 2 loss_tol / (2 h)."""
    from alphazero_quoridor_amd import losses

    d = make(6, 9, torch.float32, 3)
    d["w"] = torch.full((6,), 1.0 / 6)
    e = definition(d, True, "full", (1.0, 9.0), 0.3, 0.1)  # a range that no ratio leaves: the loss is smooth
    dev = {k: v.to(gpu_device) for k, v in d.items()}
    kw = dict(legal=dev["legal"], weights=dev["w"], ref_logits=dev["ref"], clip=(1.0, 9.0), kl_coef=0.3, entropy_coef=0.1)

    def run(z):
        return losses.policy_loss_and_grad(z, dev["actions"], dev["adv"], dev["old"], **kw)

    base, grad = run(dev["z"])
    h = 2.0 ** -6
    r = torch.exp(e["logp"] - d["old"].double())
    bound = 8 * (d["w"].double() * ((r * d["adv"].double()).abs() + 0.3 + 0.1 * 6)).max()
    tol = h * h / 6 * bound + e["loss_tol"] / h
    for i in range(6):
        for j in range(9):
            up, down = dev["z"].clone(), dev["z"].clone()
            up[i, j] += h
            down[i, j] -= h
            diff = (float(run(up)[0].loss) - float(run(down)[0].loss)) / (float(up[i, j]) - float(down[i, j]))
            assert abs(diff - float(grad[i, j])) <= float(tol), (i, j, diff, float(grad[i, j]), float(tol))


def test_small_kl_keeps_its_digits(gpu_device):
    """KL of two nearly equal policies (1e-7 .. 1e-3): every term q (e^x - 1 - x) is >= 0 and taken from the series, so the sum is good
    to 64 u relative plus the logits' own rounding: x = (z - zq) - (lse - lseq) has an absolute error delta_x <= 8 u max|z| per
    column apart from the common one, and counts with sum |p - q| <= sqrt(2 KL)."""
    from alphazero_quoridor_amd import losses

    for a in (140, 3000, 20000):
        for eps in (1e-3, 1e-2):
            g = torch.Generator().manual_seed(a)
            z = torch.randn((9, a), generator=g) * 2
            ref = z + eps * torch.randn((9, a), generator=g)
            lp, lq = torch.log_softmax(z.double(), 1), torch.log_softmax(ref.double(), 1)
            want = (torch.exp(lq) * (lq - lp)).sum(1)
            act = torch.zeros(9, dtype=torch.int64, device=gpu_device)
            o = torch.zeros(9, device=gpu_device)
            got = losses.clipped_policy_loss(z.to(gpu_device), act, o, o, ref_logits=ref.to(gpu_device), kl_coef=1.0).kl
            top = z.abs().max()
            # the common error c of lse - lseq enters as (sum p - sum q) c = 0 up to c^2 / 2
            common = 128 * U * (1 + float(top))
            tol = 64 * U * want + 8 * U * float(top) * torch.sqrt(2 * want) + common * common
            close(got, want, tol, "a=%d eps=%g" % (a, eps))


def test_infinite_and_lowest_logits(gpu_device):
    """-inf logits have no probability; a mask of the type's lowest value leaves a uniform row where it covers all; a NaN or +inf among
    the legal columns makes that row NaN and no other."""
    from alphazero_quoridor_amd import losses

    for a in (5, 140, 3000, 33000):
        n = 6
        z = torch.randn((n, a), generator=torch.Generator().manual_seed(a))
        z[0, 1:] = -math.inf                      # one column left
        z[1, :] = torch.finfo(torch.float32).min  # a mask of the lowest value over everything
        z[2, :] = -math.inf                       # nothing left: the action's logit is -inf
        z[3, a - 1] = math.nan
        z[4, a - 1] = math.inf
        act = torch.zeros(n, dtype=torch.int64)
        zg = z.to(gpu_device).requires_grad_(True)
        adv, old = torch.ones(n, device=gpu_device), torch.zeros(n, device=gpu_device)
        w = torch.tensor([1.0, 1.0, 1.0, 0.0, 0.0, 1.0], device=gpu_device)
        out = losses.clipped_policy_loss(zg, act.to(gpu_device), adv, old, weights=w, entropy_coef=0.5)
        out.loss.backward()
        logp, ent = out.logp.cpu(), out.entropy.cpu()
        assert logp[0] == 0 and ent[0] == 0 and (zg.grad[0] == 0).all()
        assert abs(float(logp[1]) + math.log(a)) <= 64 * U * (1 + math.log(a)) and abs(float(ent[1]) - math.log(a)) <= 64 * U * (1 + math.log(a))
        assert logp[2] == -math.inf and ent[2] == 0 and (zg.grad[2] == 0).all()
        assert torch.isnan(logp[3]) and torch.isnan(ent[3]) and torch.isnan(logp[4])
        assert torch.isfinite(out.loss) and torch.isfinite(logp[5]) and torch.isfinite(zg.grad[5]).all()
        assert (zg.grad[3:5] == 0).all()          # weight 0: left out of the loss
        w[3] = 1.0
        z2 = z.to(gpu_device).requires_grad_(True)
        bad = losses.clipped_policy_loss(z2, act.to(gpu_device), adv, old, weights=w)
        bad.loss.backward()
        assert torch.isnan(bad.loss) and torch.isnan(z2.grad[3]).any() and torch.isfinite(z2.grad[5]).all()
        lp, en = losses.action_logp(z.to(gpu_device), act.to(gpu_device), entropy=True)
        assert torch.equal(torch.nan_to_num(lp), torch.nan_to_num(out.logp)) and torch.equal(torch.nan_to_num(en), torch.nan_to_num(out.entropy))
        # the frozen policy may hold -inf: where both do, the column has no term; where only pi does, KL is infinite
        ref = torch.zeros((2, a))
        zz = torch.zeros((2, a))
        ref[0, -1] = zz[0, -1] = -math.inf
        zz[1, -1] = -math.inf
        k = losses.clipped_policy_loss(zz.to(gpu_device), act[:2].to(gpu_device), adv[:2], old[:2], ref_logits=ref.to(gpu_device), kl_coef=0.1).kl.cpu()
        assert abs(float(k[0])) <= 1e-6 and k[1] == math.inf


def test_strides_shapes_and_broadcast(gpu_device):
    from alphazero_quoridor_amd import losses

    g = torch.Generator().manual_seed(0)
    for dtype in TYPES:
        big = torch.randn((4, 6, 77), generator=g).to(dtype).to(gpu_device)
        legal = (torch.rand((77,), generator=g) < 0.5).to(gpu_device)
        legal[3] = True
        act = torch.full((3, 5), 3, dtype=torch.int32, device=gpu_device)
        ref = losses.action_logp(big[:3, 1:, :].contiguous(), act.long(), legal=legal.expand(3, 5, 77).contiguous())
        assert torch.equal(losses.action_logp(big[:3, 1:, :], act, legal=legal), ref)  # rows with gaps, one legal set for all
        t = big[0, :5].t().contiguous().t()  # columns first
        assert torch.equal(losses.action_logp(t, act[0], legal=legal), losses.action_logp(big[0, :5], act[0], legal=legal))
        one = big[0, :1].clone().requires_grad_(True)
        many = one.expand(5, 77)             # one row for five decisions: its gradient is the sum of theirs
        losses.action_logp(many, act[0], legal=legal).sum().backward()
        single = big[0, :1].clone().requires_grad_(True)
        losses.action_logp(single, act[0, :1], legal=legal).sum().backward()
        half = torch.finfo(dtype).eps / 2
        assert ((one.grad.double() - 5 * single.grad.double()).abs() <= 16 * half * 5 * single.grad.double().abs() + 1e-6).all()
        z = big[:, 1:].clone().requires_grad_(True)
        adv = torch.randn((4, 5), generator=g).to(gpu_device)
        out = losses.clipped_policy_loss(z, act[:1].expand(4, 5), adv, torch.zeros_like(adv), legal=legal)
        assert out.logp.shape == (4, 5) and out.loss.shape == ()
        out.loss.backward()
        loss2, grad2 = losses.policy_loss_and_grad(z.detach().reshape(20, 77), act[:1].expand(4, 5).reshape(20), adv.reshape(20), torch.zeros(20, device=gpu_device),
                                                   legal=legal)
        assert torch.equal(loss2.loss, out.loss.detach()) and torch.equal(grad2.reshape(4, 5, 77), z.grad)
        # rows that start at every alignment
        base = torch.randn(40 * 1031 + 16, generator=g).to(dtype).to(gpu_device)
        a2 = torch.arange(40, device=gpu_device)
        for off in range(0, 9):
            v = base[off:off + 40 * 1031].view(40, 1031)
            assert torch.equal(losses.action_logp(v, a2), losses.action_logp(v.clone(), a2))
            l1, g1 = losses.policy_loss_and_grad(v, a2, torch.ones(40, device=gpu_device), torch.zeros(40, device=gpu_device), ref_logits=v.flip(0).contiguous(), kl_coef=0.1)
            l2, g2 = losses.policy_loss_and_grad(v.clone(), a2, torch.ones(40, device=gpu_device), torch.zeros(40, device=gpu_device), ref_logits=v.flip(0), kl_coef=0.1)
            assert torch.equal(g1, g2) and torch.equal(l1.loss, l2.loss)


def test_no_rows(gpu_device):
    from alphazero_quoridor_amd import losses

    z = torch.zeros((0, 140), device=gpu_device, requires_grad=True)
    e = torch.zeros(0, device=gpu_device)
    out = losses.clipped_policy_loss(z, torch.zeros(0, dtype=torch.int64, device=gpu_device), e, e)
    out.loss.backward()
    assert float(out.loss.detach()) == 0.0 and z.grad.shape == (0, 140)
    assert losses.action_logp(z, torch.zeros(0, dtype=torch.int64, device=gpu_device)).shape == (0,)


@pytest.mark.parametrize("n,a", ((200, 140), (9, 3000), (5, 70000)))
def test_upstream_factors_and_a_second_backward(gpu_device, n, a):
    """A factor on the loss gives the gradient computed with that factor, not the rounded gradient times it: under a loss scale of
    65536 float16 gradients that underflow at 1 are kept."""
    from alphazero_quoridor_amd import losses

    d = make(n, a, torch.float16, 5)
    d["w"] = torch.full((n,), 1e-4 / n)
    dev = {k: v.to(gpu_device) for k, v in d.items()}
    z = dev["z"].clone().requires_grad_(True)
    out = losses.clipped_policy_loss(z, dev["actions"], dev["adv"], dev["old"], weights=dev["w"], kl_coef=0.1, ref_logits=dev["ref"])
    (out.loss * 65536.0).backward(retain_graph=True)
    scaled = z.grad.clone()
    d2 = dict(d, w=d["w"] * 65536.0)
    e = definition(d2, False, "full", (0.2, 0.2), 0.1, 0.0)
    close(scaled, e["grad"], grad_tolerance(e, torch.float16), "scaled")
    z.grad = None
    out.loss.backward(retain_graph=True)  # the buffer of the forward pass is gone: computed again, and for a factor of 1
    first = z.grad.clone()
    z.grad = None
    out.loss.backward()
    assert torch.equal(first, z.grad)
    z2 = dev["z"].clone().requires_grad_(True)
    losses.clipped_policy_loss(z2, dev["actions"], dev["adv"], dev["old"], weights=dev["w"], kl_coef=0.1, ref_logits=dev["ref"]).loss.backward()
    assert torch.equal(first, z2.grad)
    z2.grad = None
    out = losses.clipped_policy_loss(z2, dev["actions"], dev["adv"], dev["old"], weights=dev["w"])
    with torch.no_grad():
        z2.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.loss.backward()


def test_no_second_derivative(gpu_device):
    """create_graph would make autograd take the gradient for a constant: refused."""
    from alphazero_quoridor_amd import losses

    d = {k: v.to(gpu_device) for k, v in make(4, 12, torch.float32, 1).items()}
    z = d["z"].requires_grad_(True)
    for loss in (lambda: losses.clipped_policy_loss(z, d["actions"], d["adv"], d["old"]).loss, lambda: losses.action_logp(z, d["actions"]).sum()):
        with pytest.raises(RuntimeError, match="once only"):
            torch.autograd.grad(loss(), z, create_graph=True)
        torch.autograd.grad(loss(), z)
        out = loss()
        out.backward()
        with pytest.raises(RuntimeError, match="second time"):  # the graph was given up
            out.backward()
        z.grad = None


def test_two_calls_on_two_streams_and_a_captured_call(gpu_device):
    from alphazero_quoridor_amd import losses

    sets = [{k: v.to(gpu_device) for k, v in make(300, 140, torch.float32, s).items()} for s in (1, 2)]

    def run(d):
        return losses.policy_loss_and_grad(d["z"], d["actions"], d["adv"], d["old"], legal=d["legal"], weights=d["w"], ref_logits=d["ref"], kl_coef=0.1)

    want = [run(d) for d in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, d in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(run(d))
        torch.cuda.synchronize()
        for (a, ga), (b, gb) in zip(want, got):
            assert torch.equal(ga, gb) and all(torch.equal(x, y) for x, y in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    static = {k: v.clone() for k, v in sets[0].items()}
    with torch.cuda.graph(graph):
        out, grad = run(static)
        lp = losses.action_logp(static["z"], static["actions"], legal=static["legal"])
    for k in (1, 0, 1):
        for key in static:
            static[key].copy_(sets[k][key])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, want[k][1]) and torch.equal(out.loss, want[k][0].loss) and torch.equal(lp, want[k][0].logp)
        run(sets[1 - k])  # eager work between the replays
        torch.cuda.synchronize()


def test_training_step_captured_into_a_graph(gpu_device):
    """Forward and backward through a layer inside a capture (logits that are no leaves), replayed; a leaf is refused there."""
    from alphazero_quoridor_amd import losses

    d = {k: v.to(gpu_device) for k, v in make(64, 140, torch.float32, 4).items()}
    x = torch.randn((64, 16), device=gpu_device)
    w = torch.randn((16, 140), device=gpu_device, requires_grad=True)

    def step():
        out = losses.clipped_policy_loss(x @ w, d["actions"], d["adv"], d["old"], legal=d["legal"])
        return torch.autograd.grad(out.loss, w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step().clone()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
        with pytest.raises(RuntimeError, match="inside a graph capture"):
            losses.clipped_policy_loss(d["z"].requires_grad_(True), d["actions"], d["adv"], d["old"])
        d["z"].requires_grad_(False)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_results_repeat_bit_for_bit(gpu_device):
    from alphazero_quoridor_amd import losses

    for n, a in ((4000, 140), (3, 60001), (300, 9000)):
        d = {k: v.to(gpu_device) for k, v in make(n, a, torch.bfloat16, 8).items()}
        runs = [losses.policy_loss_and_grad(d["z"], d["actions"], d["adv"], d["old"], weights=d["w"], ref_logits=d["ref"], kl_coef=0.1, entropy_coef=0.1) for _ in range(3)]
        for o, g in runs[1:]:
            assert torch.equal(g, runs[0][1]) and all(torch.equal(p, q) for p, q in zip(o, runs[0][0]))


def test_refusals_on_the_device(gpu_device):
    from alphazero_quoridor_amd import _cabi, losses

    z = torch.zeros((4, 10), device=gpu_device)
    a, f = torch.zeros(4, dtype=torch.int64, device=gpu_device), torch.zeros(4, device=gpu_device)
    ok = dict(logits=z, actions=a, advantages=f, old_logp=f)
    losses.clipped_policy_loss(**ok)
    for change, error in ((dict(actions=a[:3]), ValueError), (dict(actions=f), TypeError), (dict(advantages=f[:2]), ValueError), (dict(old_logp=f.long()), TypeError),
                          (dict(legal=torch.ones((4, 9), dtype=torch.bool, device=gpu_device)), ValueError), (dict(legal=torch.ones((4, 10), device=gpu_device)), TypeError),
                          (dict(legal=torch.ones((4, 2), dtype=torch.int32, device=gpu_device)), ValueError), (dict(ref_logits=z.half()), ValueError),
                          (dict(ref_logits=z, ref_logp=f), ValueError), (dict(clip=-0.1), ValueError), (dict(clip=(1.5, 0.2)), ValueError),
                          (dict(logits=z.double()), TypeError), (dict(logits=z[:, :0]), ValueError), (dict(weights=f.clone().requires_grad_(True)), ValueError),
                          (dict(old_logp=f.clone().requires_grad_(True)), ValueError), (dict(actions=a.cpu()), _cabi.QzError), (dict(logits=z.cpu()), _cabi.QzError),
                          (dict(clip=float("nan")), ValueError), (dict(advantages=None), TypeError)):
        with pytest.raises(error):
            losses.clipped_policy_loss(**dict(ok, **change))


def test_rows_too_long_to_index_are_refused(gpu_device):
    """More columns than 32 bits count would wrap to another number: refused before anything is read or copied."""
    from alphazero_quoridor_amd import losses

    a, f = torch.zeros(1, dtype=torch.int64, device=gpu_device), torch.zeros(1, device=gpu_device)
    for cols in (2 ** 30 + 1, 2 ** 32 + 5):
        z = torch.zeros((1, 1), device=gpu_device).expand(1, cols)
        for call in (lambda: losses.action_logp(z, a), lambda: losses.clipped_policy_loss(z, a, f, f), lambda: losses.policy_loss_and_grad(z, a, f, f)):
            with pytest.raises(ValueError, match="at most 2\\^30"):
                call()
