"""The sequence operators on the GPU at the edges of their ranges: positions without a target beside a
reference.  Tolerances as in test_seq_ops_gpu.py."""
import numpy as np
import pytest
import torch

from oracle import seq as S
from test_seq_ops_gpu import TYPES, U, close, e_of, f64, randn

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------- positions without a target
@pytest.mark.parametrize("lens", [([2, 4, 3], [3, 0, 5]), ([5] * 70, [3] * 70)])  # one workgroup, and many
@pytest.mark.parametrize("smooth", [0.0, 0.2])
def test_preference_loss_leaves_positions_without_a_target_out(cuda, lens, smooth):
    """A logp of +0 (no target) takes no part whatever the reference holds there; -0 (a certain item) does."""
    from FoodRec.engine import ops
    rng = np.random.default_rng(41)
    off = np.concatenate([[0], np.cumsum(lens[0] + lens[1])])
    n = off[-1] + 3
    lp, rf = rng.normal(size=n) * 5 - 6, rng.normal(size=n) * 5 - 6
    lost = rng.random(n) < 0.3
    lost[[0, off[-2]]] = True
    lp[lost] = 0.0
    rf[0], rf[off[-2]] = np.nan, -np.inf
    lp[1] = -0.0
    lost[1] = False
    logp = torch.tensor(lp, dtype=torch.float32, device=cuda).requires_grad_()
    ref = torch.tensor(rf, dtype=torch.float32, device=cuda)
    loss = ops.preference_loss(logp, ref, torch.from_numpy(off).to(cuda), 0.3, smooth)
    # the same lists with the positions without a target taken out of them
    kept = np.concatenate([[0], np.cumsum([(~lost[a:b]).sum() for a, b in zip(off[:-1], off[1:])])])
    want, grad = S.preference_loss(f64(logp)[:off[-1]][~lost[:off[-1]]], f64(ref)[:off[-1]][~lost[:off[-1]]], kept, 0.3,
                                   smooth)
    m = 0.3 * 2 * max((np.abs(lp) + np.abs(np.where(lost, 0, rf)))[a:b].sum() for a, b in zip(off[:-1], off[1:]))
    close(loss, want, (12 + 2 * m) * U * (1 + abs(want)))
    (got,) = torch.autograd.grad(loss, logp)
    full = np.zeros(n)
    full[:off[-1]][~lost[:off[-1]]] = grad
    close(got, full, (20 + 2 * m) * U * 0.3 / len(lens[0]))
    assert not got[torch.from_numpy(lost)].any()


@pytest.mark.parametrize("dt", list(TYPES))
def test_lost_items_beside_a_reference_that_knows_them(cuda, dt):
    """Items outside the policy's table, with a value from the reference's larger one: loss and gradients are those
    of the lists without them.  Roundings as in test_operators_together, and for bf16 those of its gradients."""
    from FoodRec.engine import ops
    t = TYPES[dt]
    rng = np.random.default_rng(42)
    n, v, d, pairs = 224, 1500, 64, 16
    H, W = randn(rng, (n, d), t, cuda, 0.5).requires_grad_(), randn(rng, (v, d), t, cuda, 0.5).requires_grad_()
    ids = rng.integers(0, v, n)
    lost = rng.random(n) < 0.05
    ids[lost] = np.where(rng.random(n) < 0.5, -1, v + 3)[lost]
    assert lost.sum() > 3
    ref = torch.tensor(rng.normal(size=n) * 2 - 9, dtype=torch.float32, device=cuda)
    off = torch.arange(0, n + 1, 7, device=cuda)
    assert len(off) == 2 * pairs + 1
    lp = ops.item_log_probs(H, W, torch.from_numpy(ids).to(cuda))
    loss = ops.preference_loss(lp, ref, off, 0.1, 0.05)
    gH, gW = torch.autograd.grad(loss, (H, W))
    h, w = (torch.from_numpy(f64(x)).requires_grad_() for x in (H, W))
    ok = torch.from_numpy(~lost)
    val = torch.log_softmax(h @ w.t(), 1)[torch.arange(n), torch.from_numpy(ids).clamp(0, v - 1)] - ref.double().cpu()
    s = torch.where(ok, val, torch.zeros((), dtype=torch.float64)).view(2 * pairs, 7).sum(1)
    m = 0.1 * (s[:pairs] - s[pairs:])
    want = (0.95 * torch.nn.functional.softplus(-m) + 0.05 * torch.nn.functional.softplus(m)).mean()
    close(loss, want.item(), 2000 * U)
    for g, x in zip((gH, gW), torch.autograd.grad(want, (h, w))):
        close(g, x.numpy(), (2000 * U + (2 * e_of(t) if t != torch.float32 else 0)) * x.abs().max().item())


@pytest.mark.parametrize("dt", list(TYPES))
def test_item_log_probs_of_targets_are_never_plus_zero(cuda, dt):
    """+0 marks a position without a target: a certain item's value is -0, also where the scores are so large that the
    difference to the log-sum rounds to nothing."""
    from FoodRec.engine import ops
    t = TYPES[dt]
    n, v = 200, 40
    rng = np.random.default_rng(43)
    H = torch.zeros(n, 16, device=cuda)
    H[:, 0] = torch.tensor(2.0 ** rng.uniform(3, 30, n), dtype=torch.float32)
    H[:, 1] = torch.tensor(2.0 ** rng.uniform(0, 7, n), dtype=torch.float32)
    W = torch.zeros(v, 16, device=cuda)
    W[:, 0] = -1.0
    W[:2, 0] = 1.0
    W[1, 1] = -1.0  # the second item's score is a little below the first one's
    H, W = H.to(t).requires_grad_(), W.to(t).requires_grad_()
    for first in (0, 1):
        ids = torch.full((n,), first, dtype=torch.int64, device=cuda)
        ids[3] = -1
        real = ids >= 0
        with torch.no_grad():
            plain = ops.item_log_probs(H, W, ids)
        for lp in (plain, ops.item_log_probs(H, W, ids)):
            assert torch.signbit(lp[real]).all()
            assert lp[3] == 0 and not torch.signbit(lp[3])
