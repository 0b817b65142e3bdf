"""More decisions than the work-items of one launch (2^32 a dimension) hold at a wave or a workgroup each: the policy losses' rows
(losses.py, csrc/qz_policy.hip) go to several launches.  One row of logits stands for all of them (stride 0), so that only the
results take memory.

Tolerance: a log-probability is good to 64 u (1 + max|z|), u = 2^-24 (tests/test_gpu_losses.py)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def setup(n, a, dtype, device):
    g = torch.Generator().manual_seed(a)
    row = (torch.randn(a, generator=g) * 2.0).to(dtype)
    actions = (torch.arange(n, device=device) * 7) % a
    want = torch.log_softmax(row.double(), 0)
    return row.to(device)[None].expand(n, a), actions, want.to(device), 64 * U * (1 + float(row.abs().max()))


def off(got, want, actions):
    return max(float((got[i:i + (1 << 24)].double() - want[actions[i:i + (1 << 24)]]).abs().max()) for i in range(0, got.numel(), 1 << 24))


# past 2^26 rows of a wave each; past 2^24 rows of a workgroup of 256 each
@pytest.mark.parametrize("n,a,dtype", (((1 << 26) + 5, 2, torch.bfloat16), ((1 << 24) + 9, 1100, torch.bfloat16)), ids=str)
def test_log_probabilities(gpu_device, n, a, dtype):
    from alphazero_quoridor_amd import losses

    z, actions, want, delta = setup(n, a, dtype, gpu_device)
    assert off(losses.action_logp(z, actions), want, actions) <= delta


@pytest.mark.parametrize("n,a,dtype", (((1 << 26) + 5, 2, torch.bfloat16), ((1 << 24) + 9, 600, torch.float16)), ids=str)
def test_loss(gpu_device, n, a, dtype):
    from alphazero_quoridor_amd import losses

    z, actions, want, delta = setup(n, a, dtype, gpu_device)
    old = want.float()[actions]
    with torch.no_grad():
        out = losses.clipped_policy_loss(z, actions, torch.ones(n, device=gpu_device), old, weights=torch.full((n,), 2.0 ** -24, device=gpu_device))
    assert off(out.logp, want, actions) <= delta
    # every ratio is within delta and old's rounding of 1, every advantage 1, the weights add up to n 2^-24
    assert abs(float(out.loss) + n * 2.0 ** -24) <= n * 2.0 ** -24 * 2 * (delta + 16 * U)


def test_gradient_of_log_probabilities(gpu_device):
    """(160 MB of logits: 20 million decisions over two moves)"""
    from alphazero_quoridor_amd import losses

    n = 20_000_000
    g = torch.Generator(device=gpu_device).manual_seed(1)
    z = torch.randn((n, 2), generator=g, device=gpu_device).requires_grad_(True)
    actions = torch.arange(n, device=gpu_device) % 2
    up = torch.rand(n, generator=g, device=gpu_device)
    losses.action_logp(z, actions).backward(up)
    with torch.no_grad():
        taken = z.double().gather(1, actions[:, None])[:, 0]
        other = z.double().gather(1, 1 - actions[:, None])[:, 0]
        q = up.double() / (1 + torch.exp(taken - other))  # g (1 - p) for the action, -g (1 - p) for the other
        tol = 4 * 64 * U * (1 + float(z.abs().max()))
        assert float((z.grad.gather(1, actions[:, None])[:, 0] - q).abs().max()) <= tol
        assert float((z.grad.gather(1, 1 - actions[:, None])[:, 0] + q).abs().max()) <= tol


def test_loss_with_its_gradient(gpu_device):
    """(17 GB of gradient, of which a block at either end and around the first launch's last row is looked at)"""
    from alphazero_quoridor_amd import losses

    n, a = (1 << 24) + 9, 520
    z, actions, want, delta = setup(n, a, torch.bfloat16, gpu_device)
    old = want.float()[actions]
    adv = torch.ones(n, device=gpu_device)
    out, grad = losses.policy_loss_and_grad(z, actions, adv, old, weights=adv)
    assert grad.shape == (n, a)
    p = torch.exp(want)
    for i in (0, (1 << 21) - 8, (1 << 24) - 8, n - 16):
        rows = torch.arange(i, i + 16, device=gpu_device)
        w = p[None].repeat(16, 1)  # -r (delta - p) with r = 1
        w[torch.arange(16), actions[rows]] -= 1.0
        assert bool(((grad[rows].double() - w).abs() <= 4 * delta + 2.0 ** -8 * w.abs()).all()), i
