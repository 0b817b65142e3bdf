"""The clipped objective's first ratio: the policy before the update is the net itself, whatever probability it holds a move at."""
import contextlib
import io

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_first_ratio_is_one_for_moves_that_the_net_holds_next_to_impossible(gpu_device, monkeypatch):
    """Half of the moves are held at e^-40 or so; the search's distribution is put on legal ones among them.  Both log-probabilities come
    from the same float32 net on the same states, about 40 in size: they agree to far less than 0.01, where a floor of 1e-10 under the
    probability (e^-23) would put them 17 apart."""
    from alphazero_quoridor_amd import losses, rules
    from alphazero_quoridor_amd.train import TrainPipeline

    torch.manual_seed(3)
    tp = TrainPipeline(n_boards=64, seed=4, objective="clipped")
    tp.n_playout = 2
    with contextlib.redirect_stdout(io.StringIO()):
        tp.collect_selfplay_data(3)
    tp.batch_size, tp.epochs = 32, 2
    with torch.no_grad():
        tp.policy_value_net.policy_value_net.fc3.bias[0::2] -= 40.0
    boards, pi, z = tp.data_buffer.gather(list(range(32)))
    legal = rules.movegen(boards)
    bits = ((legal.long()[:, :, None] >> torch.arange(32, device=gpu_device)) & 1).reshape(32, -1)[:, :140].bool()
    bits[:, 1::2] = False
    assert bits.any(1).all()
    moves = bits.long().argmax(1)
    one_hot = torch.zeros_like(pi).scatter_(1, moves[:, None], 1.0)
    monkeypatch.setattr(tp.data_buffer, "gather", lambda idx: (boards, one_hot, z))
    seen = []
    whole = losses.clipped_policy_loss

    def watched(logits, actions, advantages, old_logp, **kw):
        out = whole(logits, actions, advantages, old_logp, **kw)
        seen.append((actions, old_logp, out.logp, kw["ref_logits"], logits.detach()))
        return out

    monkeypatch.setattr(losses, "clipped_policy_loss", watched)
    with contextlib.redirect_stdout(io.StringIO()):
        tp.policy_update()
    actions, old, now, ref, logits = seen[0]
    assert torch.equal(actions, moves) and int((now < -30.0).sum()) >= 16  # (where all legal moves are held so, theirs among each other count)
    assert float((now - old).abs().max()) < 0.01
    assert float((ref - logits).abs().max()) < 0.01  # and KL is to that policy
