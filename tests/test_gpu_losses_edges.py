"""Policy losses (losses.py, csrc/qz_policy.hip) where a frozen policy forbids what the other one does, in every form that a row's width
and number choose, against the definitions in float64.  Definitions and tolerances: tests/test_gpu_losses.py."""
import math

import pytest
import torch
from test_gpu_losses import close, definition, grad_tolerance, make, pack, stored

pytestmark = pytest.mark.gpu

# a wave per row; a workgroup per row in registers, of 256 and of 1,024; read twice; few rows split over workgroups
FORMS = ((5, 140, torch.float32, "bits"), (5, 3000, torch.bfloat16, "none"), (5, 50001, torch.bfloat16, "bytes"), (70, 66003, torch.float16, "none"), (5, 70000, torch.float32, "none"))


def call(d, device, kind, kl, kl_coef, ent_coef=0.02, **kw):
    """-> (result, gradient) through autograd, after the same through policy_loss_and_grad"""
    from alphazero_quoridor_amd import losses

    dev = {k: v.to(device) for k, v in d.items()}
    legal = None if kind == "none" else dev["legal"] if kind == "bytes" else pack(d["legal"]).to(device)
    args = dict(legal=legal, weights=dev["w"], ref_logits=dev["ref"] if kl == "full" else None, ref_logp=dev["ref_logp"] if kl == "taken" else None,
                kl_coef=kl_coef, entropy_coef=ent_coef, **kw)
    z = dev["z"].clone().requires_grad_(True)
    out = losses.clipped_policy_loss(z, dev["actions"], dev["adv"], dev["old"], **args)
    out.loss.backward()
    raw, grad = losses.policy_loss_and_grad(dev["z"], dev["actions"], dev["adv"], dev["old"], **args)
    assert torch.equal(grad, z.grad) and torch.equal(raw.logp, out.logp)
    return out, z.grad


@pytest.mark.parametrize("n,a,dtype,kind", FORMS, ids=str)
def test_a_frozen_policy_that_forbids_the_action_taken(gpu_device, n, a, dtype, kind):
    """KL estimated from ref_logp = -inf, or a mask's lowest value: an infinite or huge term, whose gradient is that of -x: the
    derivative e^x - 1 of e^x - 1 - x is -1 there."""
    d = make(n, a, dtype, 17 + a)
    d["ref_logp"][:5] = torch.tensor([-math.inf, -torch.finfo(torch.float32).max, -1e9, -3e7, -2.0])
    e = definition(d, kind != "none", "taken", (0.2, 0.2), 0.05, 0.02)
    assert torch.isfinite(e["grad"]).all()
    out, grad = call(d, gpu_device, kind, "taken", 0.05)
    close(out.kl, e["kl"], e["kl_tol"], "kl")
    assert float(out.loss.detach()) == math.inf
    close(grad, stored(e["grad"], dtype), grad_tolerance(e, dtype), "grad")


@pytest.mark.parametrize("kl", ("taken", "full"))
@pytest.mark.parametrize("n,a,dtype,kind", FORMS, ids=str)
def test_a_term_with_the_factor_zero_takes_no_part(gpu_device, n, a, dtype, kind, kl):
    """kl_coef = 0 only watches KL: where it is infinite (or, a legal frozen logit being NaN, undefined), loss and gradient are those
    without a frozen policy."""
    d = make(n, a, dtype, 23 + a)
    d["ref_logp"][0] = -math.inf
    other = (d["actions"] + 1) % a  # legal, and given no probability by the policy in row 1, none by the frozen one in row 2
    d["legal"][torch.arange(n), other] = True
    d["z"][1, other[1]] = -math.inf
    d["ref"][2, other[2]] = -math.inf
    d["ref"][3, other[3]] = math.nan
    e = definition(d, kind != "none", "none", (0.2, 0.2), 0.0, 0.02)
    out, grad = call(d, gpu_device, kind, kl, 0.0)
    assert math.isinf(float(out.kl[0 if kl == "taken" else 1]))
    assert kl == "taken" or math.isnan(float(out.kl[3]))
    close(out.loss.detach(), e["loss"], e["loss_tol"], "loss")
    close(out.logp, e["logp"], e["logp_tol"], "logp")
    close(out.entropy, e["entropy"], e["entropy_tol"], "entropy")
    close(grad, e["grad"], grad_tolerance(e, dtype), "grad")


def test_forward_mode_is_refused(gpu_device):
    """A dual tensor requires no gradient: its tangent must not be dropped in silence, in the logits or in what is constant otherwise."""
    import torch.autograd.forward_ad as fwd
    from alphazero_quoridor_amd import losses

    d = {k: v.to(gpu_device) for k, v in make(6, 20, torch.float32, 1).items()}

    def both(**change):
        a = dict(dict(logits=d["z"], actions=d["actions"], advantages=d["adv"], old_logp=d["old"]), **change)
        return (lambda: losses.clipped_policy_loss(**a)), (lambda: losses.policy_loss_and_grad(**a))

    want = losses.clipped_policy_loss(d["z"], d["actions"], d["adv"], d["old"]).loss
    with fwd.dual_level():
        calls = []
        for name, key in (("logits", "z"), ("advantages", "adv"), ("old_logp", "old"), ("weights", "w"), ("ref_logits", "ref"), ("ref_logp", "ref_logp")):
            calls += both(**{name: fwd.make_dual(d[key], torch.ones_like(d[key]))})
        dual = fwd.make_dual(d["z"], torch.ones_like(d["z"]))
        calls += [lambda: losses.action_logp(dual, d["actions"]), lambda: losses.action_logp(dual.view(2, 3, 20), d["actions"].view(2, 3), entropy=True),
                  lambda: losses.action_logp(dual.clone().requires_grad_(True) * 1, d["actions"])]
        for k, f in enumerate(calls):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
                pytest.fail("call %d went through" % k)
        primal = fwd.unpack_dual(dual).primal
        assert torch.equal(losses.clipped_policy_loss(primal, d["actions"], d["adv"], d["old"]).loss, want)
    assert torch.equal(losses.clipped_policy_loss(d["z"], d["actions"], d["adv"], d["old"]).loss, want)


@pytest.mark.parametrize("factor", (1.0, 3.0))
def test_a_captured_backward_pass_of_an_eager_forward_pass(gpu_device, factor):
    """The graph holds the backward pass alone: every replay computes the gradient of the logits as they are by then, also after the last
    one's gradient was changed in place."""
    from alphazero_quoridor_amd import losses

    sets = [{k: v.to(gpu_device) for k, v in make(50, 140, torch.float32, s).items()} for s in (1, 2)]
    fixed = {k: v for k, v in sets[0].items() if k != "z"}

    def want(z):
        return losses.policy_loss_and_grad(z, fixed["actions"], fixed["adv"], fixed["old"], legal=fixed["legal"], weights=fixed["w"] * factor)[1]

    side, leaf = torch.cuda.Stream(), torch.zeros((50, 140), device=gpu_device, requires_grad=True)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = leaf + sets[0]["z"]
        out = losses.clipped_policy_loss(z, fixed["actions"], fixed["adv"], fixed["old"], legal=fixed["legal"], weights=fixed["w"])
    torch.cuda.synchronize()
    graph, up = torch.cuda.CUDAGraph(), torch.tensor(factor, device=gpu_device)
    with torch.cuda.graph(graph, stream=side):
        grad = torch.autograd.grad(out.loss, z, up, retain_graph=True)[0]
        grad.mul_(0.5)
    for k in (0, 0, 1, 1, 0):
        z.detach().copy_(sets[k]["z"])
        e = 0.5 * want(z.detach())
        graph.replay()
        torch.cuda.synchronize()
        assert float((grad - e).abs().max()) <= 8 * 2.0 ** -24 * (1 + float(e.abs().max())), k  # (the weights carry the factor there: one rounding each)
        (grad + 1).sum()  # eager work between the replays
    # the forward pass captured too, in a graph of its own
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first, stream=side):
        z2 = leaf + sets[0]["z"]
        out2 = losses.clipped_policy_loss(z2, fixed["actions"], fixed["adv"], fixed["old"], legal=fixed["legal"], weights=fixed["w"])
    with torch.cuda.graph(second, stream=side):
        grad2 = torch.autograd.grad(out2.loss, z2, up, retain_graph=True)[0]
        grad2.mul_(0.5)
    first.replay()
    e = 0.5 * want(sets[0]["z"])
    for _ in range(3):
        second.replay()
        torch.cuda.synchronize()
        assert float((grad2 - e).abs().max()) <= 8 * 2.0 ** -24 * (1 + float(e.abs().max()))


def test_which_divergence_the_kl_terms_are(gpu_device):
    """Over the logits: KL(frozen || pi).  From ref_logp: terms whose mean over actions drawn from pi is KL(pi || frozen).  Every action of one
    distribution is a decision here, so that the mean is a sum; each term is good to 16 u (1 + |x| + e^x)."""
    from alphazero_quoridor_amd import losses

    g = torch.Generator().manual_seed(9)
    z, zq = torch.randn(40, generator=g), torch.randn(40, generator=g)
    lp, lq = torch.log_softmax(z.double(), 0), torch.log_softmax(zq.double(), 0)
    rows = dict(logits=z.expand(40, 40).contiguous().to(gpu_device), actions=torch.arange(40, device=gpu_device), advantages=torch.zeros(40, device=gpu_device),
                old_logp=lp.float().to(gpu_device), kl_coef=1.0)
    over = losses.clipped_policy_loss(ref_logits=zq.expand(40, 40).contiguous().to(gpu_device), **rows).kl.double().cpu()
    taken = losses.clipped_policy_loss(ref_logp=lq.float().to(gpu_device), **rows).kl.double().cpu()
    tol = 16 * 2.0 ** -24 * float((lp.exp() * (1 + (lq - lp).abs() + (lq - lp).exp())).sum())
    assert float((over - (lq.exp() * (lq - lp)).sum()).abs().max()) <= 8 * tol
    assert abs(float((lp.exp() * taken).sum() - (lp.exp() * (lp - lq)).sum())) <= tol


def test_negated_views(gpu_device):
    """The imaginary part of a conjugate is a view whose memory holds the other sign; a single element, or a single column, of one counts as
    contiguous."""
    from alphazero_quoridor_amd import losses

    c = torch.randn((1, 8), dtype=torch.complex64, generator=torch.Generator().manual_seed(2)).to(gpu_device).conj()
    z, v = c.real.contiguous(), c[:, 3].imag
    assert v.is_neg() and v.is_contiguous()
    act = torch.tensor([2], device=gpu_device)
    args = dict(advantages=v, old_logp=c[:, 4].imag, weights=c[:, 5].imag, ref_logp=c[:, 6].imag, kl_coef=0.1)
    plain = {k: x.clone().resolve_neg() if torch.is_tensor(x) else x for k, x in args.items()}
    for a, b in zip(losses.policy_loss_and_grad(z, act, **args)[0], losses.policy_loss_and_grad(z, act, **plain)[0]):
        assert torch.equal(a, b)
    many = torch.randn((4, 8), dtype=torch.complex64, generator=torch.Generator().manual_seed(3)).to(gpu_device).conj().imag
    for logits in (many, many.t(), torch._neg_view(z.expand(4, 8).contiguous())):
        a = torch.arange(logits.shape[0], device=gpu_device) % logits.shape[1]
        assert logits.is_neg() and torch.equal(losses.action_logp(logits, a), losses.action_logp(logits.resolve_neg().contiguous(), a))
    # upstream gradients
    x = z.clone().requires_grad_(True)
    for f, up in ((lambda: losses.action_logp(x, act), c[:, 1].imag), (lambda: losses.clipped_policy_loss(x, act, c.real[:, 1], c.real[:, 2]).loss, c[0, 1].imag)):
        assert up.is_neg()
        assert torch.equal(torch.autograd.grad(f(), x, up)[0], torch.autograd.grad(f(), x, up.resolve_neg().clone())[0])
