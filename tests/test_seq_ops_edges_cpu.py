"""The edges of the sequence operators' ranges that need no GPU: the oracle there, and refusals."""
import numpy as np
import pytest
import torch

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


def _calls(ops, x, w, lp, i, c):
    return {"embedding_scaled": lambda: ops.embedding_scaled(i, w, 2.0), "dropout": lambda: ops.dropout(x, 0.1, 1, c),
            "rms_norm": lambda: ops.rms_norm(x), "add_rms_norm": lambda: ops.add_rms_norm(x, x),
            "add_rms_norm_quant": lambda: ops.add_rms_norm_quant(x, x),
            "item_log_probs": lambda: ops.item_log_probs(x, w, i),
            "preference_loss": lambda: ops.preference_loss(lp, None, i)}


def _inputs():
    return (torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3), torch.zeros(3, dtype=torch.int64),
            torch.zeros(1, dtype=torch.int64))


def test_forward_mode_is_refused():
    """A tangent would be dropped: its primal asks for no gradient, so the kernels would be called directly."""
    import torch.autograd.forward_ad as fwd
    from FoodRec.engine import native, ops
    x, w, lp, i, c = _inputs()
    with fwd.dual_level():
        dx, dw, dl = (fwd.make_dual(t, torch.ones_like(t)) for t in (x, w, lp))
        for name, call in _calls(ops, dx, dw, dl, i, c).items():
            with pytest.raises(native.EngineError, match=name + ".*forward-mode"):
                call()
        for call in (lambda: ops.item_log_probs(x, dw, i), lambda: ops.rms_norm(x, dx[0]),  # any argument's
                     lambda: ops.dropout(x, 0.1, 1, c, residual=dx), lambda: ops.preference_loss(lp, dl, i)):
            with pytest.raises(native.EngineError, match="forward-mode"):
                call()
        for name, call in _calls(ops, x, w, lp, i, c).items():  # without a tangent: the usual refusal of CPU tensors
            with pytest.raises(native.EngineError, match="GPU"):
                call()


def test_tracing_is_refused():
    from FoodRec.engine import native, ops
    x, w, lp, i, c = _inputs()
    for name in _calls(ops, x, w, lp, i, c):
        with pytest.raises(native.EngineError, match=name + ".*traced"):
            torch.jit.trace(lambda a, b, v: _calls(ops, a, b, v, i, c)[name](), (x, w, lp))


class _OnGpu:
    """A stand-in for a device tensor, as far as layers.Dropout looks at one before any kernel."""
    is_cuda, dtype, device = True, torch.float32, torch.device("cpu")


def test_dropout_layer_refuses_its_first_forward_in_a_capture(monkeypatch):
    """The counter would be zeroed by every replay.  With a counter made before, the forward goes on."""
    from FoodRec.engine import layers, native, ops
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    seen = []
    monkeypatch.setattr(ops, "dropout", lambda x, p, seed, counter, residual=None: seen.append((seed, int(counter))))
    layer = layers.Dropout(0.5)
    with pytest.raises(native.EngineError, match="cannot be captured"):
        layer(_OnGpu())
    assert "_fr_dropout" not in layer.__dict__
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    layer(_OnGpu())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    layer(_OnGpu())
    assert [s for _, s in seen] == [0, 1] and seen[0][0] == seen[1][0]


def test_dropout_layer_mask_state(monkeypatch):
    """A resumed layer goes on where the saved one stopped; copies, attributes set by a model or not, do not repeat it."""
    import copy
    from FoodRec.engine import layers, ops
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    seen = []
    monkeypatch.setattr(ops, "dropout", lambda x, p, seed, counter, residual=None: seen.append((seed, int(counter))))
    layer = layers.Dropout(0.5)
    layer.__dict__["_fr_salt"] = 0
    assert layer.mask_state() is None
    for _ in range(3):
        layer(_OnGpu())
    state = layer.mask_state()
    assert state == {"seed": seen[0][0], "step": 3}
    copy.deepcopy(layer)(_OnGpu())
    assert seen[-1][0] != state["seed"] and seen[-1][1] == 0
    resumed = layers.Dropout(0.5)
    resumed.load_mask_state(state, "cpu")
    resumed(_OnGpu())
    layer(_OnGpu())
    assert seen[-1] == seen[-2] == (state["seed"], 3)
    resumed.load_mask_state(None, "cpu")
    resumed(_OnGpu())
    assert seen[-1][0] != state["seed"]


def test_tensors_without_memory_are_refused():
    """Wrappers of torch.func's transforms and sparse tensors have no rows for a kernel to read."""
    from FoodRec.engine import native, ops
    x, w, lp, i, c = _inputs()
    for call in (lambda: torch.vmap(lambda a: ops.rms_norm(a))(x),
                 lambda: torch.func.grad(lambda a: ops.embedding_scaled(i, a).sum())(w),
                 lambda: torch.func.grad(lambda a: ops.item_log_probs(x, a, i).sum())(w),
                 lambda: torch.func.grad(lambda a: ops.dropout(x, 0.5, 1, c, residual=a).sum())(x),
                 lambda: ops.rms_norm(x.to_sparse()), lambda: ops.preference_loss(lp.to_sparse(), None, i)):
        with pytest.raises(native.EngineError, match="dense tensor"):
            call()
