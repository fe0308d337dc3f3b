"""The edges of the sequence operators' ranges that need no GPU: the oracle there, and refusals."""
import numpy as np
import pytest

from oracle import seq as S


@pytest.mark.parametrize("smooth", [0.0, 0.2])
def test_preference_oracle_leaves_positions_without_a_target_out(smooth):
    """Loss and gradient are those of the lists without the positions whose logp is +0; -0 is a value."""
    r = np.random.default_rng(1)
    off = np.array([0, 3, 5, 5, 9, 12, 13, 20, 21])
    lp, ref = r.normal(size=23) - 5, r.normal(size=23) - 5
    lost = np.isin(np.arange(23), [0, 4, 9, 10, 11, 22])
    lp[lost], lp[6], ref[4], ref[9] = 0.0, -0.0, np.nan, np.inf
    loss, grad = S.preference_loss(lp, ref, off, 0.4, smooth)
    kept = np.concatenate([[0], np.cumsum([(~lost[a:b]).sum() for a, b in zip(off[:-1], off[1:])])])
    want, g = S.preference_loss(np.where(lost, -1, lp)[~lost], ref[~lost], kept, 0.4, smooth)
    assert abs(loss - want) < 1e-14
    assert np.allclose(grad[~lost], g, atol=1e-15) and not grad[lost].any()
    # without a reference there is nothing to leave out: the same loss with either zero
    a, _ = S.preference_loss(lp, None, off, 0.4, smooth)
    b, _ = S.preference_loss(np.where(lost, -0.0, lp), None, off, 0.4, smooth)
    assert a == b
