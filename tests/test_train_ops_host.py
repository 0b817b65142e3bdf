"""The training operators' checks of arguments that need no GPU: the C entry points refuse bad arguments before they touch a
device, and the Python ones refuse tensors on the CPU (there is no CPU path)."""
import ctypes as C

import pytest
import torch

from alphazero_quoridor_amd import _cabi


def lib():
    import os

    if not os.path.exists(_cabi.LIB_PATH):
        _cabi.build()
    return _cabi.load()


def rows(**kw):
    d = dict(logits=1 << 20, ld=140, n=4, n_actions=140, dtype=0, actions=1 << 20, legal=0, legal_ld=0, legal_kind=0)
    d.update(kw)
    return _cabi.qz_policy_rows(*[d[f] for f, _ in _cabi.qz_policy_rows._fields_])


def terms(**kw):
    d = dict(advantages=1 << 20, old_logp=1 << 20, ref_logp=0, weights=0, ref_logits=0, ref_ld=0, clip_low=0.2, clip_high=0.2, kl_coef=0.0, entropy_coef=0.0)
    d.update(kw)
    return _cabi.qz_policy_terms(*[d[f] for f, _ in _cabi.qz_policy_terms._fields_])


BIG = 1 << 30


def test_policy_entry_points_refuse_bad_arguments():
    L, p = lib(), 1 << 20

    def loss(r, t, loss=p, logp=p, grad=p, ld=140, ws=p, size=BIG):
        return L.qz_policy_loss(C.byref(r), C.byref(t), loss, logp, p, p, grad, ld, ws, size, None)

    for r in (rows(n=-1), rows(n=1 << 31), rows(n_actions=0), rows(dtype=3), rows(dtype=-1), rows(legal_kind=3), rows(legal_kind=1), rows(logits=0), rows(actions=0),
              rows(ld=-140)):
        assert loss(r, terms()) == _cabi.E_INVALID, _cabi.load().qz_last_error()
        assert L.qz_action_logp(C.byref(r), p, None, None, p, BIG, None) == _cabi.E_INVALID
        assert L.qz_action_logp_backward(C.byref(r), p, None, p, None, p, 140, None) == _cabi.E_INVALID
    for t in (terms(advantages=0), terms(old_logp=0), terms(ref_logits=p, ref_logp=p), terms(clip_low=-0.1), terms(clip_low=1.1), terms(clip_high=-0.5),
              terms(clip_low=float("nan")), terms(clip_high=float("nan"))):
        assert loss(rows(), t) == _cabi.E_INVALID
    assert L.qz_policy_loss(None, C.byref(terms()), p, p, p, p, p, 140, p, BIG, None) == _cabi.E_INVALID
    assert L.qz_policy_loss(C.byref(rows()), None, p, p, p, p, p, 140, p, BIG, None) == _cabi.E_INVALID
    need = L.qz_policy_workspace(4, 140)
    assert need > 0 and loss(rows(), terms(), size=need - 1) == _cabi.E_INVALID and loss(rows(), terms(), ws=0) == _cabi.E_INVALID
    assert b"workspace" in L.qz_last_error()
    assert L.qz_policy_workspace(-1, 140) == 0 and L.qz_policy_workspace(4, 0) == 0


def test_rows_too_long_to_index_are_refused():
    L, p = lib(), 1 << 20
    for a in ((1 << 30) + 1, (1 << 31) - 1):
        r = rows(n=1, n_actions=a)
        assert L.qz_policy_loss(C.byref(r), C.byref(terms()), p, p, p, p, p, 140, p, BIG, None) == _cabi.E_INVALID
        assert L.qz_action_logp(C.byref(r), p, None, None, p, BIG, None) == _cabi.E_INVALID


def test_matrix_entry_points_refuse_bad_arguments():
    L, p = lib(), 1 << 20

    def mat(rows=8, cols=9, update=p, ld=9, out=p, out_ld=9, momentum=p, param=p, scale=1.0):
        return _cabi.qz_matrix(rows, cols, update, ld, out, out_ld, momentum, param, scale)

    def ortho(m, count=1, dtype=0, steps=5, ws=p, size=BIG):
        arr = (_cabi.qz_matrix * 1)(m)
        return L.qz_orthogonalize(arr, count, dtype, steps, ws, size, None)

    def muon(m, opts=True, steps=5):
        arr = (_cabi.qz_matrix * 1)(m)
        o = _cabi.qz_muon_opts(0.1, 0.9, 0.0, 1, 0)
        return L.qz_muon_step(arr, 1, 0, steps, C.byref(o) if opts else None, p, BIG, None)

    for m in (mat(rows=-1), mat(cols=-1), mat(rows=(1 << 20) + 1), mat(rows=1 << 20, cols=1 << 20), mat(update=0), mat(ld=-1)):
        assert ortho(m) == _cabi.E_INVALID and muon(m) == _cabi.E_INVALID
    assert ortho(mat(out=0)) == _cabi.E_INVALID and ortho(mat(out_ld=8)) == _cabi.E_INVALID
    assert muon(mat(momentum=0)) == _cabi.E_INVALID and muon(mat(param=0)) == _cabi.E_INVALID and muon(mat(), opts=False) == _cabi.E_INVALID
    for kw in (dict(count=-1), dict(dtype=3)):
        assert ortho(mat(), **kw) == _cabi.E_INVALID
    assert L.qz_orthogonalize(None, 1, 0, 5, p, BIG, None) == _cabi.E_INVALID
    assert L.qz_orthogonalize_workspace(None, 3) == 0
    arr = (_cabi.qz_matrix * 2)(mat(), mat(rows=0))
    one = L.qz_orthogonalize_workspace(arr, 1)
    assert one > 0 and L.qz_orthogonalize_workspace(arr, 2) == one  # an empty matrix takes nothing
    if not torch.cuda.is_available():  # past the arguments: no device
        assert ortho(mat()) == _cabi.E_NO_DEVICE and muon(mat()) == _cabi.E_NO_DEVICE


def test_no_cpu_path():
    from alphazero_quoridor_amd import losses, optim

    z, a, f = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    for call in (lambda: losses.action_logp(z, a), lambda: losses.clipped_policy_loss(z, a, f, f), lambda: losses.policy_loss_and_grad(z, a, f, f),
                 lambda: optim.orthogonalize(z), lambda: optim.orthogonalize([z])):
        with pytest.raises(_cabi.QzError) as e:
            call()
        assert e.value.code == _cabi.E_NO_DEVICE
    p = torch.nn.Parameter(z)
    p.grad = torch.zeros(3, 5)
    with pytest.raises(_cabi.QzError):
        optim.Muon([p]).step()


def test_muon_refuses_bad_options():
    from alphazero_quoridor_amd import optim

    p = torch.nn.Parameter(torch.zeros(3, 5))
    for kw in (dict(lr=-1.0), dict(lr=float("nan")), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0), dict(ns_steps=0), dict(ns_steps=17),
               dict(adjust_lr="other")):
        with pytest.raises(ValueError):
            optim.Muon([p], **kw)
    for bad in (torch.zeros(5), torch.zeros(3, 5).half(), torch.zeros(5, 3).t(), torch.zeros(3, 5, dtype=torch.float64)):
        with pytest.raises(ValueError):
            optim.Muon([torch.nn.Parameter(bad)])


def test_muon_refuses_a_parameter_twice_and_checks_later_groups():
    from alphazero_quoridor_amd import optim

    p, q = (torch.nn.Parameter(torch.zeros(3, 5)) for _ in range(2))
    with pytest.raises(ValueError), pytest.warns(UserWarning):
        optim.Muon([p, p])
    opt = optim.Muon([p])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [p]})
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4))]})
    opt = optim.Muon([p])
    opt.add_param_group({"params": [q], "lr": 0.5})
    assert opt.param_groups[1]["lr"] == 0.5 and opt.param_groups[1]["momentum"] == 0.95


def test_chained_optimisers_step_and_keep_their_state():
    from alphazero_quoridor_amd import optim

    ps = [torch.nn.Parameter(torch.ones(2)), torch.nn.Parameter(torch.ones(3))]
    both = optim.Chained(torch.optim.SGD([ps[0]], lr=0.1), torch.optim.Adam([ps[1]], lr=0.2))
    assert [g["lr"] for g in both.param_groups] == [0.1, 0.2]
    for g in both.param_groups:
        g["lr"] = 0.5
    for p in ps:
        p.grad = torch.ones_like(p)
    both.step()
    assert torch.equal(ps[0], torch.full((2,), 0.5)) and (ps[1] < 1).all()
    state = both.state_dict()
    both.zero_grad()
    assert ps[0].grad is None
    again = optim.Chained(torch.optim.SGD([ps[0]], lr=0.1), torch.optim.Adam([ps[1]], lr=0.2))
    again.load_state_dict(state)
    assert again.param_groups[1]["lr"] == 0.5 and len(again.optimizers[1].state) == 1
    with pytest.raises(ValueError):
        again.load_state_dict({"optimizers": []})


def test_negative_strides_are_refused():
    """A negative stride of the legal set's bytes or of the frozen policy's logits would read before their start."""
    L, p = lib(), 1 << 20
    for r, t in ((rows(legal=p, legal_kind=2, legal_ld=-140), terms()), (rows(legal=p, legal_kind=1, legal_ld=-5), terms()), (rows(), terms(ref_logits=p, ref_ld=-140))):
        assert L.qz_policy_loss(C.byref(r), C.byref(t), p, p, p, p, p, 140, p, BIG, None) == _cabi.E_INVALID, _cabi.load().qz_last_error()
        assert L.qz_policy_loss_backward(C.byref(r), C.byref(t), p, 0, p, 140, p, BIG, None) == _cabi.E_INVALID
        assert b"stride" in L.qz_last_error()
    r = rows(legal=p, legal_kind=2, legal_ld=-140)
    assert L.qz_action_logp(C.byref(r), p, None, None, p, BIG, None) == _cabi.E_INVALID
    assert L.qz_action_logp_backward(C.byref(r), p, None, p, None, p, 140, None) == _cabi.E_INVALID


def test_the_workspace_of_a_matrix_out_of_range_is_refused():
    """A caller that allocates what it is told must not be told terabytes for a matrix that the call itself refuses (or what is left of
    a size past 64 bits)."""
    L = lib()
    for rows_, cols in ((1 << 31, 1), (1, (1 << 20) + 1), (1 << 20, 1 << 20), (1 << 62, 1 << 62), (-1, 5)):
        arr = (_cabi.qz_matrix * 2)(_cabi.qz_matrix(8, 9), _cabi.qz_matrix(rows_, cols))
        assert L.qz_orthogonalize_workspace(arr, 2) == _cabi.E_INVALID and b"out of range" in L.qz_last_error()


def test_python_asks_for_no_memory_for_a_matrix_out_of_range(monkeypatch):
    from alphazero_quoridor_amd import optim

    monkeypatch.setattr(torch, "empty", lambda *a, **k: pytest.fail("allocated"))
    with pytest.raises(_cabi.QzError) as e:
        optim._List([1 << 31, 1, 1 << 20, 1, 1 << 20, 1, 0, 0, 0], torch.device("cpu"))
    assert e.value.code == _cabi.E_INVALID
