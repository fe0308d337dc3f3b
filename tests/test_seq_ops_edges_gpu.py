"""The sequence operators on the GPU at the edges of their ranges: positions without a target beside a
reference, masked and outlying rows.  Tolerances as in test_seq_ops_gpu.py."""
import numpy as np
import pytest
import torch

from oracle import seq as S
from test_seq_ops_gpu import TYPES, U, close, e_of, f64, randn, strided

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


# ------------------------------------------------------------------------ masked and outlying rows
def own_bounds(H, W, ids, scale, up, t):
    """logp_bounds of test_seq_ops_gpu.py, where a score's error is that of its own terms: d products (twice, see
    there), 12 u of two 11-bit parts, and for fp32 2^-22 for what such parts leave of entries far below the largest of
    their 32 rows; scores far below a row's log-sum have no part in it whatever their size.  exp2 gives 0 below 2^-126,
    so a probability may be off by that much.  A score beyond fp32's range in units of log 2 is that range's end."""
    n, d = H.shape
    v = len(W)
    ok = (ids >= 0) & (ids < v)
    Hc, W = np.where(ok[:, None], H, 0.0), np.maximum(W, -1e300)  # -inf as a number: 0 times it is 0 in a row without target
    with np.errstate(all="ignore"):
        logp, z, lse = S.item_log_probs(Hc, W, ids, scale)
        logp = np.where(logp < -1e200, -np.inf, np.maximum(logp, -np.log(2) * np.finfo(np.float32).max))
        f32 = t == torch.float32
        own = np.where(np.isfinite(z), np.abs(Hc) @ np.abs(W).T, 0.0)
        dz = ((2 * (d + 2) + 12 * f32) * U * own + 2 * U * np.where(np.isfinite(z), np.abs(z), 0) / scale) * scale
        dz += 2.0 ** -22 * f32
        at = (np.arange(n), np.where(ok, ids, 0))
        dzt, zt = dz[at], np.where(np.isfinite(z[at]), np.abs(z[at]), 0)
        live = z + dz > lse[:, None] - 150
        dz = np.where(live, dz, 0.0)
        p = np.where(live, np.exp(z - lse[:, None]), 0.0)
        top = np.maximum(np.abs(np.where(live, z, 0.0)).max(1), np.abs(lse))
        dlse = 1.01 * (p * dz).sum(1) + (v / 2 + 100) * U + 6 * U * top
        dlogp = np.where(ok, dzt + dlse + 4 * U * (top + zt), 0.0)
        dH, dW, g = S.item_log_probs_grad(H, W, ids, scale, up)
        c = np.where(ok, np.abs(up) * scale, 0.0)
        e = 0.0 if f32 else e_of(t)
        rel = dz + dlse[:, None] + 4 * U * (top[:, None] + 1) + 4 * U
        dg = c[:, None] * (p * rel + 2.0 ** -126) + np.abs(g) * (4 * U + e)
        tH = dg @ np.abs(W) + 2 * (v / 16 + 64) * U * np.abs(g) @ np.abs(W) + (e_of(t) + 4 * U) * np.abs(dH)
        if not f32:
            dg += c[:, None] * p * 2 * (d + 2) * U * np.abs(lse)[:, None]
        tW = dg.T @ np.abs(Hc) + 2 * (n / 2 + 64) * U * np.abs(g).T @ np.abs(Hc) + (e_of(t) + 4 * U) * np.abs(dW)
    return logp, dlogp, dH, tH, dW, tW


def check_scores(ops, H, W, ids, t, scale=1.0, columns=None, upstream=1.0):
    """Values without and with gradients and both gradients against float64 (the gradients' first `columns`)."""
    n, v = len(H), len(W)
    up = torch.linspace(-1, 1, n, device=H.device) * upstream
    it = torch.from_numpy(ids).to(H.device)
    want, tol, dH, tH, dW, tW = own_bounds(f64(H), f64(W), ids, scale, f64(up), t)
    fin = np.isfinite(want)
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            lp = ops.item_log_probs(H, W, it, scale)
        assert (f64(lp)[~fin] == want[~fin]).all(), grad
        close(f64(lp)[fin], want[fin], tol[fin], ("logp", grad))
    gH, gW = torch.autograd.grad(lp, (H, W), up)
    close(f64(gH)[:, :columns], dH[:, :columns], tH[:, :columns], "dH")
    close(f64(gW), dW, tW, "dW")


MASKS = [-1e4, -1e9, -1e30, "lowest", -np.inf]


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("d", [33, 64, 100, 256])
@pytest.mark.parametrize("mask", MASKS)
def test_item_log_probs_of_masked_items(cuda, mask, d, dt):
    """Items taken out through a column that is 1 in every user row: their neighbours in the table keep their bits."""
    from FoodRec.engine import ops
    t = TYPES[dt]
    value = torch.finfo(t).min if mask == "lowest" else mask
    rng = np.random.default_rng(d)
    n, v = 150, 333
    s = 1.2 / d ** 0.25
    H, W = randn(rng, (n, d), t, cuda, s), randn(rng, (v, d), t, cuda, s)
    out = np.zeros(v, bool)
    out[[0, 5, 31, 40, 331]] = True
    out[96:170] = True  # whole blocks of rows, too
    out[rng.integers(200, v, 12)] = True
    H[:, -1] = 1.0
    W[:, -1] = torch.where(torch.from_numpy(out).to(cuda), torch.tensor(value, dtype=t, device=cuda), torch.zeros((), dtype=t, device=cuda))
    ids = rng.choice(np.flatnonzero(~out), n)
    ids[:3] = 4, 6, 332  # beside masked rows
    ids[9], ids[10], ids[11] = 5, -1, v  # a masked target, and none
    with torch.no_grad():
        H[10] = float("nan")
    # (0 times an infinite entry: dH has no number in its column)
    check_scores(ops, H.requires_grad_(), W.requires_grad_(), ids, t, columns=d - 1 if mask == -np.inf else None)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("d", [64, 100, 256])
def test_item_log_probs_of_items_masked_by_the_users(cuda, d, dt):
    """The other way round: the users' rows hold the mask's value, in a column that only masked items have."""
    from FoodRec.engine import ops
    t = TYPES[dt]
    rng = np.random.default_rng(d + 1)
    n, v = 150, 333
    s = 1.2 / d ** 0.25
    H, W = randn(rng, (n, d), t, cuda, s), randn(rng, (v, d), t, cuda, s)
    out = torch.from_numpy(rng.random(v) < 0.1).to(cuda)
    W[:, 3] = out.to(t)
    for value in (-1e9, -1e30):
        H[:, 3] = value
        ids = rng.choice(np.flatnonzero(~out.cpu().numpy()), n)
        check_scores(ops, H.clone().requires_grad_(), W.clone().requires_grad_(), ids, t)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("d", [64, 100])
def test_item_log_probs_beside_an_outlying_user(cuda, d, dt):
    """One user's row 1e12 times the others': its neighbours keep their bits, it is certain of one item."""
    from FoodRec.engine import ops
    t = TYPES[dt]
    rng = np.random.default_rng(d + 2)
    H, W = randn(rng, (150, d), t, cuda, 0.4), randn(rng, (333, d), t, cuda, 0.4)
    H[37] *= 1e12
    check_scores(ops, H.requires_grad_(), W.requires_grad_(), rng.integers(0, 333, 150), t)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("size", [3.0, 30.0])
@pytest.mark.parametrize("d", [64, 256])
def test_item_log_probs_of_large_scores(cuda, d, size, dt):
    """Even rows whose scores are in the hundreds and thousands."""
    from FoodRec.engine import ops
    t = TYPES[dt]
    rng = np.random.default_rng(d + 3)
    H, W = randn(rng, (150, d), t, cuda, size), randn(rng, (333, d), t, cuda, size)
    check_scores(ops, H.requires_grad_(), W.requires_grad_(), rng.integers(0, 333, 150), t)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("mask", [-1e30, "lowest"])
@pytest.mark.parametrize("d,v", [(16, 50), (64, 700), (100, 1), (256, 300)])
def test_item_log_probs_where_all_items_are_masked_alike(cuda, d, v, mask, dt):
    """Every score of a row the same huge negative number: every item as likely as any other, in the gradients, too.
    Roundings: the sum of v ones, one exp2 and log2; g rounded to the type, sums of n and of v products of it."""
    from FoodRec.engine import ops
    t = TYPES[dt]
    rng = np.random.default_rng(d)
    n = 130
    H, W = torch.zeros(n, d, device=cuda, dtype=t), randn(rng, (v, d), t, cuda)
    H[:, -1], W[:, -1] = 1.0, torch.finfo(t).min if mask == "lowest" else mask
    H, W = H.requires_grad_(), W.requires_grad_()
    ids = rng.integers(0, v, n)
    ids[7] = -1
    it, up = torch.from_numpy(ids).to(cuda), torch.linspace(-1, 1, n, device=cuda)
    want = np.where(ids >= 0, -np.log(v), 0.0)
    with torch.no_grad():
        close(ops.item_log_probs(H, W, it), want, (v + 60) * U * (1 + np.log(v)))
    lp = ops.item_log_probs(H, W, it)
    close(lp, want, (v + 60) * U * (1 + np.log(v)))
    gH, gW = torch.autograd.grad(lp, (H, W), up)
    a, w = np.where(ids >= 0, f64(up), 0.0), f64(W)[:, :-1]
    e = 0.0 if t == torch.float32 else e_of(t)
    dH = a[:, None] * (w[ids] - w.mean(0))
    size = np.abs(a)[:, None] * (np.abs(w[ids]) + np.abs(w).mean(0))
    close(f64(gH)[:, :-1], dH, (e + (2 * v + 60) * U) * size + e_of(t) * np.abs(dH))
    hit = np.zeros((v, n))
    hit[ids, np.arange(n)] = 1.0
    dW, size = (hit - 1 / v) @ a, (hit + 1 / v) @ np.abs(a)
    close(f64(gW)[:, -1], dW, (e + (2 * v + 2 * n + 60) * U) * size + e_of(t) * np.abs(dW))
    assert not gW[:, :-1].any()


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("scale", [1e-38, 3e-36])
def test_item_log_probs_of_vanishing_scale(cuda, scale, dt):
    """A temperature so high that the log-sum in the scores' units leaves fp32's range."""
    from FoodRec.engine import ops
    t = TYPES[dt]
    rng = np.random.default_rng(51)
    H, W = randn(rng, (150, 64), t, cuda, 0.4), randn(rng, (700, 64), t, cuda, 0.4)
    check_scores(ops, H.requires_grad_(), W.requires_grad_(), rng.integers(0, 700, 150), t, scale, upstream=1e30)


@pytest.mark.parametrize("dt", list(TYPES))
def test_item_log_probs_where_the_mask_leaves_nothing(cuda, dt):
    """Every score -inf: there is no distribution, and the value is NaN, as log_softmax has it; other rows keep theirs."""
    from FoodRec.engine import ops
    t = TYPES[dt]
    for d, v in ((16, 50), (100, 1), (64, 700)):
        H, W = torch.ones(40, d, device=cuda, dtype=t), torch.zeros(v, d, device=cuda, dtype=t)
        H[20:, 1] = 0.0
        W[:, 1] = torch.finfo(t).min
        H[:20, 1] = 4.0  # overflows to -inf; 0 in the others' rows leaves a score of 0
        H, W = H.requires_grad_(), W.requires_grad_()
        ids = torch.arange(40, device=cuda) % v
        ids[4] = -1
        with torch.no_grad():
            plain = ops.item_log_probs(H, W, ids)
        for lp in (plain, ops.item_log_probs(H, W, ids)):
            assert lp[4] == 0
            gone = torch.arange(20, device=cuda) != 4
            assert torch.isnan(lp[:20][gone]).all()
            close(lp[20:], np.full(20, -np.log(v)), 60 * U * (1 + np.log(v)))


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("d", [50, 64])
def test_item_log_probs_of_masked_items_layouts(cuda, d, dt):
    """The same rows at any stride and alignment."""
    from FoodRec.engine import ops
    t = TYPES[dt]
    rng = np.random.default_rng(d + 4)
    H, W = randn(rng, (140, d), t, cuda, 0.4), randn(rng, (333, d), t, cuda, 0.4)
    H[:, 0], W[:, 0] = 1.0, torch.where(torch.arange(333, device=cuda) % 9 == 2, -1e9, 0.0).to(t)
    ids, up = torch.arange(140, device=cuda) * 9 % 333, torch.linspace(-1, 1, 140, device=cuda)

    def both(h, w):
        h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
        lp = ops.item_log_probs(h, w, ids)
        return lp, *torch.autograd.grad(lp, (h, w), up)
    for got in (both(strided(H), strided(W)), both(H.t().contiguous().t(), W.t().contiguous().t())):
        assert all(torch.equal(a, b) for a, b in zip(got, both(H, W)))


@pytest.mark.parametrize("pairs", [2, 70])
def test_preference_loss_of_infinite_margins(cuda, pairs):
    """A rejected item that the policy cannot choose (logp -inf): no loss and no gradient without smoothing."""
    from FoodRec.engine import ops
    n = 2 * pairs
    logp = torch.full((n,), -2.0, device=cuda)
    logp[pairs] = -float("inf")
    logp.requires_grad_()
    off = torch.arange(n + 1, device=cuda)
    loss = ops.preference_loss(logp, None, off, 0.5)
    want = (pairs - 1) * np.log(2) / pairs
    close(loss, want, 20 * U)
    (g,) = torch.autograd.grad(loss, logp)
    slope = np.full(pairs, -0.25 / pairs)
    slope[0] = 0.0
    close(g, np.concatenate([slope, -slope]), 20 * U)
    assert ops.preference_loss(logp, None, off, 0.5, 0.1).item() == float("inf")
    low = torch.tensor([-2.0, -float("inf"), -1.0], device=cuda).requires_grad_()
    assert ops.preference_loss(low, None, torch.tensor([1, 2, 3], device=cuda), 0.5).item() == float("inf")


def test_forward_mode_and_traces_are_refused(cuda):
    import torch.autograd.forward_ad as fwd
    from FoodRec.engine import native, ops
    x, w = torch.randn(6, 8, device=cuda), torch.randn(20, 8, device=cuda)
    i, c = torch.arange(6, device=cuda), torch.zeros(1, dtype=torch.int64, device=cuda)
    lp, off = torch.randn(6, device=cuda), torch.tensor([0, 3, 6], device=cuda)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.embedding_scaled(i, fwd.make_dual(w, w), 2.0), lambda: ops.dropout(d, 0.1, 1, c),
                     lambda: ops.dropout(x, 0.1, 1, c, residual=d), lambda: ops.rms_norm(d), lambda: ops.rms_norm(x, d[0]),
                     lambda: ops.add_rms_norm(x, d), lambda: ops.add_rms_norm_quant(x, d),
                     lambda: ops.item_log_probs(d, w, i), lambda: ops.item_log_probs(x, fwd.make_dual(w, w), i),
                     lambda: ops.preference_loss(fwd.make_dual(lp, lp), None, off),
                     lambda: ops.preference_loss(lp, fwd.make_dual(lp, lp), off)):
            with pytest.raises(native.EngineError, match="forward-mode"):
                call()
        assert torch.equal(ops.rms_norm(x), ops.rms_norm(fwd.unpack_dual(d).primal))
    with pytest.raises(native.EngineError, match="traced"):
        torch.jit.trace(lambda a: ops.rms_norm(a), x)


# ------------------------------------------------------------------------------- 8-bit norm
@pytest.mark.parametrize("d", [64, 50, 2048])
def test_add_rms_norm_quant_of_tiny_rows(cuda, d):
    """Rows whose largest value is subnormal: the scale is still positive and no value leaves the 8 bits' range."""
    from FoodRec.engine import ops
    rng = np.random.default_rng(d)
    tops = [2.0 ** -149, 3 * 2.0 ** -149, 447 * 2.0 ** -149, 671 * 2.0 ** -149, 449 * 2.0 ** -149, 1e-41, 1e-39, 1e-36]
    x = torch.ones(len(tops), d, device=cuda)
    w = torch.tensor(rng.uniform(-1, 1, (len(tops), d)), dtype=torch.float64)
    w[:, 3] = 1.0
    for k, top in enumerate(tops):
        wk = (w[k] * top).float().to(cuda)
        q, s, _ = ops.add_rms_norm_quant(x[k:k + 1], None, wk, 0.0)
        y = f64(wk)  # rows of ones: rstd is 1 to rounding, and its step is far below one of a subnormal number
        val = f64(q.float())[0] * f64(s)[0]
        assert np.isfinite(val).all() and f64(s)[0] > 0
        # s is rounded to a step of 2^-149 or up to the next; e4m3 as in test_add_rms_norm_quant
        assert abs(f64(s)[0] - top / 448) <= 2.0 ** -149 + 64 * U * top / 448
        assert (np.abs(val - y) <= (2.0 ** -4 + (d + 40) * U) * np.abs(y) + f64(s)[0] * 2.0 ** -10 + 2.0 ** -149).all()
