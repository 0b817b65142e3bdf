"""Policy losses (losses.py, csrc/qz_policy.hip) on many wide rows, against the definitions in float64 of tests/test_gpu_losses.py.

Tolerance: the definitions' tolerances are linear in 64 u, the relative error of a row's sums of exponentials (u = 2^-24).  A thread that
adds k columns, then joins 8 times at most with a rescaled sum (3 roundings each), its exponentials off by at most 4 u (the argument's
scaling, the instruction, the difference to the maximum), is within (k + 24 + 4) u: the tolerances are taken times that over 64."""
import pytest
import torch
from test_gpu_losses import close, definition, grad_tolerance, make, pack, stored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,a,dtype,kind,kl,per_thread", (
    # mask and frozen logits together, the widest rows that stay in registers: 512 threads of 8 chunks
    (300, 32768, torch.bfloat16, "bits", "full", 64), (300, 20003, torch.float16, "bytes", "full", 64), (300, 16384, torch.float32, "bytes", "full", 32),
    (300, 9001, torch.float32, "bits", "full", 32),
    # more rows than 256, read twice by 256 threads each
    (260, 131072, torch.bfloat16, "none", "full", 512)), ids=str)
def test_many_wide_rows(gpu_device, n, a, dtype, kind, kl, per_thread):
    from alphazero_quoridor_amd import losses

    d = make(n, a, dtype, n + a)
    d["actions"][1], d["legal"][2] = -1, False
    d["w"][4] = 0.0
    e = definition(d, kind != "none", kl, (0.2, 0.2), 0.05, 0.02)
    k = max(1.0, (per_thread + 28) / 64)
    dev = {key: v.to(gpu_device) for key, v in d.items()}
    legal = None if kind == "none" else dev["legal"] if kind == "bytes" else pack(d["legal"]).to(gpu_device)
    out, grad = losses.policy_loss_and_grad(dev["z"], dev["actions"], dev["adv"], dev["old"], legal=legal, weights=dev["w"], ref_logits=dev["ref"], kl_coef=0.05,
                                            entropy_coef=0.02)
    for name in ("loss", "logp", "entropy", "kl"):
        close(getattr(out, name), e[name], k * e[name + "_tol"], name)
    e["grad_tol"] *= k
    close(grad, stored(e["grad"], dtype), grad_tolerance(e, dtype), "grad")
    logp, ent = losses.action_logp(dev["z"], dev["actions"], legal=legal, entropy=True)
    k = max(1.0, (a / 256 + 28) / 64)  # (256 threads, whatever the width)
    close(logp, e["logp"], k * e["logp_tol"], "action_logp")
    close(ent, e["entropy"], k * e["entropy_tol"], "action entropy")
