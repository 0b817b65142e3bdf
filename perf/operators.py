"""What the training operators of this package are measured on.

Four operators: the log-probability of the action taken under a legal-move mask (``losses.action_logp``), the clipped
policy loss with its KL and entropy terms and its gradient (``losses.clipped_policy_loss``), the Newton-Schulz
orthogonalisation of updates (``optim.orthogonalize``) and the optimiser step built on it (``optim.Muon``).
``own = False`` computes them from elementary tensor operations in float32; ``own = True`` calls the package."""
import functools
import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NS = (3.4445, -4.7750, 2.0315)      # quintic Newton-Schulz coefficients of the Muon optimiser
NS_STEPS, NS_FLOOR = 5, 1e-7
MOMENTUM, LR, DECAY = 0.95, 0.02, 0.01
CLIP, KL_COEF, ENT_COEF = 0.2, 0.02, 0.01
# the hidden matrices of this package's policy-value net: conv1, the ten trunk convolutions, the head convolutions, fc1
NETWORK = "64x234 " + "64x576 " * 10 + "4x576 2x576 128x324"


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one training minibatch of the policy-value net (batch_size 128, 140 moves, the legal sets of the boards)
        {"name": "loss minibatch", "op": "loss", "rows": 128, "cols": 140, "type": "f32", "legal": "bits", "kl": "full"},
        # the whole replay buffer as one batch
        {"name": "loss buffer", "op": "loss", "rows": 10000, "cols": 140, "type": "f32", "legal": "bits", "kl": "full"},
        # policy tuning of a sequence model: a batch of tokens over a vocabulary, KL to a frozen policy's logits
        {"name": "loss tokens", "op": "loss", "rows": 8192, "cols": 32768, "type": "bf16", "legal": "none", "kl": "full"},
        # an odd vocabulary (rows that start unaligned) with a byte mask, KL estimated from the frozen policy's log-probabilities
        {"name": "loss odd vocabulary", "op": "loss", "rows": 2047, "cols": 50001, "type": "bf16", "legal": "bytes", "kl": "taken"},
        # the moves that a full set of concurrent self-play boards has just played
        {"name": "logp boards", "op": "logp", "rows": 13312, "cols": 140, "type": "f32", "legal": "bits", "grad": False},
        # one sampled token of one sequence
        {"name": "logp one token", "op": "logp", "rows": 1, "cols": 32000, "type": "bf16", "legal": "none", "grad": False},
        # log-probabilities with their gradient for a loss that the user writes
        {"name": "logp tokens", "op": "logp", "rows": 4096, "cols": 32000, "type": "bf16", "legal": "none", "grad": True},
        # the hidden matrices of the policy-value net
        {"name": "orthogonalize network", "op": "ortho", "shapes": NETWORK, "type": "f32"},
        # a wide and a tall matrix in 16 bits
        {"name": "orthogonalize wide tall", "op": "ortho", "shapes": "1024x4096 4096x1024", "type": "bf16"},
        # one large square matrix
        {"name": "orthogonalize square", "op": "ortho", "shapes": "4096x4096", "type": "f32"},
        # one optimiser step of the policy-value net
        {"name": "muon network", "op": "muon", "shapes": NETWORK, "type": "f32"},
        # one optimiser step of four attention projections and a feed-forward pair
        {"name": "muon block", "op": "muon", "shapes": "1024x1024 1024x1024 1024x1024 1024x1024 4096x1024 1024x4096", "type": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("loss", "loss", "logp", "ortho", "muon"))
    if op in ("loss", "logp"):
        cols = _log(rng, 2, 131072)
        rows = _log(rng, 1, max(1, min(40000, (8192 * 32768 // 2) // cols)))
        c = {"op": op, "rows": rows, "cols": cols, "type": rng.choice(("f32", "bf16", "f16")), "legal": rng.choice(("none", "bits", "bytes"))}
        if op == "loss":
            c["kl"] = rng.choice(("none", "full", "taken"))
        else:
            c["grad"] = rng.random() < 0.5
        return c
    count = rng.choice((1, 1, 2, 3, 5))
    shapes = []
    for _ in range(count):
        m = _log(rng, 1, 2048)
        n = min(8192, max(1, _log(rng, max(1, m // 8), m * 8)))
        shapes.append("%dx%d" % ((m, n) if rng.random() < 0.5 else (n, m)))
    return {"op": op, "shapes": " ".join(shapes), "type": rng.choice(("f32", "bf16", "f16")) if op == "ortho" else "f32"}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split()]


def work(case):
    if case["op"] in ("loss", "logp"):
        n, a = case["rows"], case["cols"]
        e = 4 if case["type"] == "f32" else 2
        grad = case["op"] == "loss" or case["grad"]
        full = case.get("kl") == "full"
        mask = {"none": 0, "bits": 4 * ((a + 31) // 32), "bytes": a}[case["legal"]]
        per_row = n * (a * e * (1 + int(full) + int(grad)) + mask)
        return {"bytes": per_row + n * (8 + 4 * 6), "flops": n * a * (8 + 8 * int(full) + 4 * int(grad))}
    e = 4 if case["type"] == "f32" else 2
    # per step: X X^T and its square (symmetric: half of each), and the product with X
    flops = sum(NS_STEPS * (min(s) ** 2 * max(s) + min(s) ** 3 + 2 * min(s) ** 2 * max(s)) for s in _shapes(case))
    size = sum(m * n for m, n in _shapes(case))
    return {"bytes": size * (2 * e if case["op"] == "ortho" else 5 * 4), "flops": flops}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


def _gradient(shape, g, device):
    """A gradient as training meets it: a few decaying directions and the noise of the minibatch."""
    m, n = shape
    r = max(1, min(m, n) // 8)
    u = torch.randn((m, r), generator=g, device=device) * torch.exp(-3.0 * torch.arange(r, device=device) / r)
    signal, noise = u @ torch.randn((r, n), generator=g, device=device), torch.randn((m, n), generator=g, device=device)
    return 1e-3 * (signal / signal.norm() + 0.3 * noise / noise.norm()) * math.sqrt(m * n)


def _pack_bits(legal):
    n, a = legal.shape
    bits = F.pad(legal, (0, -a % 32)).view(n, -1, 32).to(torch.int64)
    words = (bits << torch.arange(32, device=legal.device)).sum(2)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _policy_inputs(case, seed, device="cuda"):
    g = _gen(seed, device)
    n, a, dt = case["rows"], case["cols"], DTYPES[case["type"]]
    logits = (torch.randn((n, a), generator=g, device=device) * 2.0).to(dt)
    d = {"logits": logits, "legal": None, "legal_mask": None}
    if case["legal"] != "none":
        legal = torch.rand((n, a), generator=g, device=device) < 0.7
        legal[:, 0] |= ~legal.any(1)
        d["legal_mask"] = legal
        d["legal"] = legal if case["legal"] == "bytes" else _pack_bits(legal)
    # actions sampled from the policy among the legal ones (Gumbel maximum)
    noise = -torch.log(-torch.log(torch.rand((n, a), generator=g, device=device).clamp_(1e-7, 1 - 1e-7)))
    score = logits.float() + noise
    if d["legal_mask"] is not None:
        score.masked_fill_(~d["legal_mask"], -math.inf)
    d["actions"] = score.argmax(1)
    del noise, score
    # float16 gradients are trained with a loss scale: without one they underflow
    scale = min(4096, n) if dt == torch.float16 else 1
    if case["op"] == "logp":
        d["dlogp"] = torch.randn(n, generator=g, device=device) * (scale / n)
        d["dentropy"] = torch.randn(n, generator=g, device=device) * (0.01 * scale / n)
        return d
    z = logits.double()
    if d["legal_mask"] is not None:
        z.masked_fill_(~d["legal_mask"], -math.inf)
    logp = (z.gather(1, d["actions"][:, None]) - torch.logsumexp(z, 1, keepdim=True)).squeeze(1)
    del z
    # ratios around one, a third of them past the clip range, none within 1e-3 of its borders
    log_ratio = torch.randn(n, generator=g, device=device, dtype=torch.float64) * 0.2
    for border in (math.log(1 - CLIP), math.log(1 + CLIP)):
        near = (log_ratio - border).abs() < 1e-3
        log_ratio = torch.where(near, torch.full_like(log_ratio, border - 2e-3), log_ratio)
    d["old_logp"] = (logp - log_ratio).float()
    d["advantages"] = torch.randn(n, generator=g, device=device)
    live = torch.rand(n, generator=g, device=device) < 0.95  # the rest is padding: weight 0
    live[0] = True
    d["weights"] = live.float() * scale / live.sum()
    d["ref_logits"] = d["ref_logp"] = None
    if case["kl"] == "full":
        d["ref_logits"] = (logits.float() + 0.3 * torch.randn((n, a), generator=g, device=device)).to(dt)
    elif case["kl"] == "taken":
        d["ref_logp"] = (logp + 0.3 * torch.randn(n, generator=g, device=device)).float()
    return d


def _matrix_inputs(case, seed, device="cuda"):
    g = _gen(seed, device)
    dt = DTYPES[case["type"]]
    d = {"grads": [_gradient(s, g, device).to(dt) for s in _shapes(case)]}
    if case["op"] == "muon":
        d["momenta"] = [_gradient(s, g, device) for s in _shapes(case)]
        d["params"] = [torch.randn(s, generator=g, device=device) / math.sqrt(s[1]) for s in _shapes(case)]
    return d


def prepare(case, seed):
    if case["op"] in ("loss", "logp"):
        d = _policy_inputs(case, seed)
        d["logits"].requires_grad_(case["op"] == "loss" or case["grad"])
    else:
        d = _matrix_inputs(case, seed)
        if own and case["op"] == "muon":
            from alphazero_quoridor_amd.optim import Muon

            d["params"] = [torch.nn.Parameter(p) for p in d["params"]]
            opt = Muon(d["params"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, ns_steps=NS_STEPS)
            for p, grad, buf in zip(d["params"], d["grads"], d["momenta"]):
                p.grad = grad
                opt.state[p]["momentum_buffer"] = buf
            d["optimizer"] = opt
    d["case"] = dict(case)
    return d


# ------------------------------------------------------------------------------------------------ plain forms, float32
def _log_softmax(z, legal):
    z = z.float()
    if legal is not None:
        z = z.masked_fill(~legal, -math.inf)
    z = z - z.max(1, keepdim=True).values
    return z - torch.log(torch.exp(z).sum(1, keepdim=True))


def _finite(x, legal):
    return x if legal is None else x.masked_fill(~legal, 0.0)


def _plain_logp(d):
    case, legal, a = d["case"], d["legal_mask"], d["actions"][:, None]
    logits = d["logits"].detach()
    logp = _log_softmax(logits, legal)
    p = torch.exp(logp)
    logp = _finite(logp, legal)
    taken, entropy = logp.gather(1, a).squeeze(1), -(p * logp).sum(1)
    if not case["grad"]:
        return {"logp": taken, "entropy": entropy}
    grad = -p * (d["dlogp"][:, None] + d["dentropy"][:, None] * (logp + entropy[:, None]))
    grad.scatter_add_(1, a, d["dlogp"][:, None])
    return {"logp": taken, "entropy": entropy, "grad": _finite(grad, legal).to(logits.dtype)}


def _plain_loss(d):
    legal, a = d["legal_mask"], d["actions"][:, None]
    logits = d["logits"].detach()
    logp = _log_softmax(logits, legal)
    p = torch.exp(logp)
    logp = _finite(logp, legal)
    taken, entropy = logp.gather(1, a).squeeze(1), -(p * logp).sum(1)
    ratio, adv = torch.exp(taken - d["old_logp"]), d["advantages"]
    free, held = ratio * adv, ratio.clamp(1 - CLIP, 1 + CLIP) * adv
    pull = torch.where(free <= held, -adv * ratio, torch.zeros_like(ratio))  # d(-surrogate)/d logp
    kl = torch.zeros_like(taken)
    diff = None
    if d["ref_logits"] is not None:
        ref = _log_softmax(d["ref_logits"], legal)
        q = torch.exp(ref)
        x = logp - _finite(ref, legal)
        kl = (q * (torch.expm1(x) - x)).sum(1)  # = sum q (log q - log p): both sum to one
        diff = p - q
    elif d["ref_logp"] is not None:
        x = d["ref_logp"] - taken
        kl = torch.expm1(x) - x
        pull = pull - KL_COEF * torch.expm1(x)
    w = d["weights"]
    loss = (w * (-torch.minimum(free, held) + KL_COEF * kl - ENT_COEF * entropy)).sum()
    grad = p * (ENT_COEF * (logp + entropy[:, None]) - pull[:, None])
    if diff is not None:
        grad = grad + KL_COEF * diff
    grad.scatter_add_(1, a, pull[:, None])
    grad = _finite(grad * w[:, None], legal).to(logits.dtype)
    return {"loss": loss, "logp": taken, "kl": kl, "entropy": entropy, "grad": grad}


def _ns_step(x):
    a = x @ x.t()
    return NS[0] * x + (NS[1] * a + NS[2] * (a @ a)) @ x


def _plain_orthogonalize(u):
    x = u.float() if u.shape[0] <= u.shape[1] else u.float().t()
    x = x / x.norm().clamp(min=NS_FLOOR)
    x = functools.reduce(lambda y, _: _ns_step(y), range(NS_STEPS), x)
    return (x if u.shape[0] <= u.shape[1] else x.t()).contiguous().to(u.dtype)


def _plain_muon(p, grad, buf):
    buf.lerp_(grad, 1 - MOMENTUM)
    o = _plain_orthogonalize(torch.lerp(grad, buf, MOMENTUM))
    p.mul_(1 - LR * DECAY).sub_(LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * o)
    return p


def run(d):
    op = d["case"]["op"]
    if not own:
        if op == "logp":
            return _plain_logp(d)
        if op == "loss":
            return _plain_loss(d)
        if op == "ortho":
            return [_plain_orthogonalize(g) for g in d["grads"]]
        return {"params": [_plain_muon(*t) for t in zip(d["params"], d["grads"], d["momenta"])], "momenta": d["momenta"]}
    from alphazero_quoridor_amd import losses, optim

    if op == "logp":
        logits = d["logits"]
        logits.grad = None
        logp, entropy = losses.action_logp(logits, d["actions"], legal=d["legal"], entropy=True)
        if not d["case"]["grad"]:
            return {"logp": logp, "entropy": entropy}
        torch.autograd.backward((logp, entropy), (d["dlogp"], d["dentropy"]))
        return {"logp": logp.detach(), "entropy": entropy.detach(), "grad": logits.grad}
    if op == "loss":
        logits = d["logits"]
        logits.grad = None
        out = losses.clipped_policy_loss(logits, d["actions"], d["advantages"], d["old_logp"], legal=d["legal"], weights=d["weights"],
                                         ref_logits=d["ref_logits"], ref_logp=d["ref_logp"], clip=CLIP, kl_coef=KL_COEF, entropy_coef=ENT_COEF)
        out.loss.backward()
        return {"loss": out.loss.detach(), "logp": out.logp, "kl": out.kl, "entropy": out.entropy, "grad": logits.grad}
    if op == "ortho":
        return optim.orthogonalize(d["grads"], steps=NS_STEPS)
    d["optimizer"].step()
    return {"params": [p.detach() for p in d["params"]], "momenta": d["momenta"]}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_distribution(z, legal):
    z = z.double()
    if legal is not None:
        z = torch.where(legal, z, torch.full_like(z, -1e300))
    return torch.log_softmax(z, 1)


def exact(case, seed):
    if case["op"] in ("loss", "logp"):
        d = _policy_inputs(case, seed)
        legal, a = d["legal_mask"], d["actions"][:, None]
        z = d["logits"].double().requires_grad_(True)
        logp = _exact_distribution(z, legal)
        p = torch.exp(logp)
        inside = torch.ones_like(p, dtype=torch.bool) if legal is None else legal
        plogp = torch.where(inside, p * torch.where(inside, logp, torch.zeros_like(logp)), torch.zeros_like(p))
        taken, entropy = logp.gather(1, a)[:, 0], -plogp.sum(1)
        if case["op"] == "logp":
            if not case["grad"]:
                return {"logp": taken.detach(), "entropy": entropy.detach()}
            (grad,) = torch.autograd.grad((taken * d["dlogp"].double()).sum() + (entropy * d["dentropy"].double()).sum(), z)
            return {"logp": taken.detach(), "entropy": entropy.detach(), "grad": grad}
        ratio, adv, w = torch.exp(taken - d["old_logp"].double()), d["advantages"].double(), d["weights"].double()
        per_row = -torch.minimum(ratio * adv, torch.clamp(ratio, 1 - CLIP, 1 + CLIP) * adv)
        kl = torch.zeros_like(taken)
        if d["ref_logits"] is not None:
            ref = _exact_distribution(d["ref_logits"], legal)
            kl = torch.where(inside, torch.exp(ref) * (ref - logp), torch.zeros_like(ref)).sum(1)
        elif d["ref_logp"] is not None:
            x = d["ref_logp"].double() - taken
            kl = torch.exp(x) - 1 - x
        loss = (w * (per_row + KL_COEF * kl - ENT_COEF * entropy)).sum()
        (grad,) = torch.autograd.grad(loss, z)
        return {"loss": loss.detach(), "logp": taken.detach(), "kl": kl.detach(), "entropy": entropy.detach(), "grad": grad}
    d = _matrix_inputs(case, seed)

    def polynomial(u):
        x = u.double() / torch.clamp(torch.linalg.vector_norm(u.double()), min=NS_FLOOR)
        tall = x.shape[0] > x.shape[1]
        for _ in range(NS_STEPS):  # odd polynomial of the singular values, from whichever side is shorter
            g = x.mT @ x if tall else x @ x.mT
            q = NS[1] * g + NS[2] * torch.mm(g, g)
            q.diagonal().add_(NS[0])
            x = x @ q if tall else q @ x
        return x

    if case["op"] == "ortho":
        return [polynomial(g) for g in d["grads"]]
    params, momenta = [], []
    for p, g, m in zip(d["params"], d["grads"], d["momenta"]):
        m = MOMENTUM * m.double() + (1 - MOMENTUM) * g.double()
        scale = max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        params.append(p.double() * (1 - LR * DECAY) - LR * scale * polynomial((1 - MOMENTUM) * g.double() + MOMENTUM * m))
        momenta.append(m)
    return {"params": params, "momenta": momenta}
