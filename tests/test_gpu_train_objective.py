"""The training operators as the pipeline uses them: the clipped objective on self-play data with the boards' legal sets, the Muon
optimiser over the net's hidden matrices, and both together for an update."""
import contextlib
import io

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def quiet():
    return contextlib.redirect_stdout(io.StringIO())


@pytest.fixture(scope="module")
def shard(tmp_path_factory):
    from alphazero_quoridor_amd.train import TrainPipeline

    torch.manual_seed(3)
    play = TrainPipeline(n_boards=64, seed=4)
    play.n_playout = 2
    with quiet():
        play.collect_selfplay_data(3)
    path = tmp_path_factory.mktemp("shard") / "games.qzr"
    play.data_buffer.save_shard(path)
    return path


def pipeline(shard, **kw):
    from alphazero_quoridor_amd.train import TrainPipeline

    torch.manual_seed(7)
    tp = TrainPipeline(n_boards=64, seed=5, **kw)
    tp.data_buffer.load_shard(shard)
    tp.batch_size, tp.epochs = 32, 3
    return tp


@pytest.mark.parametrize("objective,optimizer", (("clipped", "adam"), ("clipped", "muon"), ("mcts", "muon")))
def test_policy_update(gpu_device, shard, objective, optimizer):
    tp = pipeline(shard, objective=objective, optimizer=optimizer)
    net = tp.policy_value_net.policy_value_net
    before = {n: p.detach().clone() for n, p in net.named_parameters()}
    with quiet():
        loss, entropy = tp.policy_update()
    assert np.isfinite(loss) and np.isfinite(entropy) and 0 < tp.last_update["optimizer_steps"] <= 3 and np.isfinite(tp.last_update["kl"])
    for n, p in net.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n
    if optimizer == "muon":
        muon = tp.policy_value_net.optimizer.optimizers[0]
        assert len(muon.state) == 14 and all(torch.isfinite(s["momentum_buffer"]).all() for s in muon.state.values())


def test_clipped_step_gradient_equals_the_composed_operations(gpu_device, shard):
    """policy_step_t's gradients against autograd through elementary float64 operations on the head's log-probabilities, carried back
    through the same network.  The loss's own gradient is good to 2 delta relative (tests/test_gpu_losses.py), delta <= 64 u (1 + 30);
    the network's backward pass is linear in it, so a parameter's gradient may be off by that share of the sum of the
    magnitudes that make it up: rows' contributions are summed with their signs, and 32 rows' magnitudes bound it."""
    from alphazero_quoridor_amd import losses, rules

    tp = pipeline(shard, objective="clipped")
    pvn = tp.policy_value_net
    boards, pi, z = tp.data_buffer.gather(list(range(32)))
    states, legal = rules.encode(boards), rules.movegen(boards)
    with torch.no_grad():
        old, old_v = pvn.policy_value_net(states)
    moves = pi.argmax(1)
    bits = ((legal.long()[:, :, None] >> torch.arange(32, device=gpu_device)) & 1).reshape(32, -1)[:, :140].bool()
    assert bits.gather(1, moves[:, None]).all()  # the search only visits legal moves
    noise = 0.1 * torch.randn(32, generator=torch.Generator().manual_seed(1)).to(gpu_device)
    move_logp, adv = losses.action_logp(old, moves, legal=legal) + noise, z - old_v.view(-1)
    ref = (old + 0.1).detach()
    logp, v = pvn.policy_value_net(states)
    logp.retain_grad()
    out = losses.clipped_policy_loss(logp, moves, adv, move_logp, legal=legal, ref_logits=ref, kl_coef=0.02, entropy_coef=0.01)
    (torch.nn.functional.mse_loss(v.view(-1), z) + out.loss).backward()
    got = logp.grad.double()
    x = logp.detach().double().requires_grad_(True)
    lp = torch.log_softmax(torch.where(bits, x, torch.full_like(x, -1e300)), 1)
    lq = torch.log_softmax(torch.where(bits, ref.double(), torch.full_like(x, -1e300)), 1)
    p, q = lp.exp(), lq.exp()
    taken = lp.gather(1, moves[:, None])[:, 0]
    r, a64 = torch.exp(taken - move_logp.double()), adv.double()
    kl = torch.where(bits, q * (lq - lp), 0.0).sum(1)
    h = -torch.where(bits, p * lp, 0.0).sum(1)
    want = torch.autograd.grad((-torch.minimum(r * a64, r.clamp(0.8, 1.2) * a64) + 0.02 * kl - 0.01 * h).mean(), x)[0]
    delta = 64 * 2.0 ** -24 * (1 + float(logp.detach().abs().max()))
    tol = 2 * delta / 32 * ((r * a64).abs() + 0.02 + 0.01 * 12)[:, None]
    assert ((got - want).abs() <= tol + 2.0 ** -24 * want.abs()).all()
    assert (got[~bits] == 0).all()
    # and the step itself: the same gradients in the parameters as a backward pass by hand
    grads = {n: w.grad.clone() for n, w in pvn.policy_value_net.named_parameters()}
    with torch.no_grad():
        w0 = [w.clone() for w in pvn.policy_value_net.parameters()]
    loss, ent = pvn.policy_step_t(states, moves, adv, move_logp, z, 1e-3, legal=legal, ref_logits=ref, kl_coef=0.02, entropy_coef=0.01)
    assert loss.is_cuda and loss.dim() == 0 and abs(float(ent) - float(out.entropy.mean())) < 1e-6
    for n, w in pvn.policy_value_net.named_parameters():
        scale = float(grads[n].abs().max())
        assert float((w.grad - grads[n]).abs().max()) <= 1e-3 * scale, n  # (the library's convolution gradients add in any order)
    assert all(not torch.equal(a, b) for a, b in zip(w0, pvn.policy_value_net.parameters()))


def test_refusals(gpu_device):
    from alphazero_quoridor_amd.policy_value_net import PolicyValueNet
    from alphazero_quoridor_amd.train import TrainPipeline

    with pytest.raises(ValueError):
        TrainPipeline(objective="other")
    with pytest.raises(ValueError):
        PolicyValueNet(optimizer="other")
    with pytest.raises(ValueError):
        PolicyValueNet(use_gpu=False, optimizer="muon")
