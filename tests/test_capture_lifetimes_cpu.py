"""What lives and dies around a captured training step, on the CPU with stand-ins for the graph: a graph that is no
longer used goes at once, and none is destroyed by the garbage collector in the middle of another one's capture (its
destruction and its memory pool's release are calls into the GPU runtime)."""
import contextlib
import gc
import types
import weakref

import pytest
import torch

from FoodRec.common import trainer as T


class _Graph:
    def __init__(self):
        self.replays = 0

    def replay(self):
        self.replays += 1

    def pool(self):
        return None


class _Feed:
    on_stage = None

    def fill(self, u, p, n, feats):
        return None


class _Sampler:
    batch_size = 4

    def device_feed(self):
        self.feed = _Feed()
        return self.feed


class _Trainer:
    device = "cpu"
    optimizer = types.SimpleNamespace(zero_grad=lambda: None)

    def _features(self):
        return types.SimpleNamespace(ssl=True, batch=lambda u, p, n, pre=None: None)

    def train_step(self, batch, idx, state, accumulate=True):
        for _ in range(200):  # a step makes objects enough for a collection of the youngest ones
            a, b = [], []
            a.append(b), b.append(a)
        state["acc"] = torch.zeros(1, dtype=torch.float64) if state.get("acc") is None else state["acc"]
        return torch.zeros(())


@pytest.fixture
def capture_log(monkeypatch):
    """Collections while a (stand-in) capture is open, and the graphs that died meanwhile."""
    log = types.SimpleNamespace(open=0, collections=0, captures=0)

    @contextlib.contextmanager
    def graph(g, *a, **k):
        log.open, log.captures = log.open + 1, log.captures + 1
        yield
        log.open -= 1

    @contextlib.contextmanager
    def stream(s):
        yield
    side = types.SimpleNamespace(wait_stream=lambda s: None)
    monkeypatch.setattr(torch.cuda, "graph", graph)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", _Graph)
    monkeypatch.setattr(torch.cuda, "Stream", lambda: side)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: side)
    monkeypatch.setattr(torch.cuda, "stream", stream)

    def note(phase, info):
        log.collections += phase == "start" and log.open > 0
    gc.callbacks.append(note)
    yield log
    gc.callbacks.remove(note)


def _step():
    sampler = _Sampler()
    step = T.GraphedStep(_Trainer(), 4, warmup=1, unroll=2)
    step.attach_feed(sampler)
    return sampler, step


def _run(step, calls):
    for k in range(calls):
        step(*step.inputs, k, step.state)


def test_a_graphed_step_goes_with_its_last_user(capture_log):
    sampler, step = _step()
    _run(step, 4)
    assert step.graph is not None and step.graph_n is not None and sampler.feed.on_stage is not None
    graphs = weakref.ref(step.graph), weakref.ref(step.graph_n)
    gc.disable()
    try:
        del step
        assert graphs[0]() is None and graphs[1]() is None
        sampler.feed.on_stage()  # nothing pending any more
    finally:
        gc.enable()


def test_no_garbage_is_collected_inside_a_capture(capture_log):
    old = gc.get_threshold()
    gc.set_threshold(50, 1, 1)
    try:
        doomed = types.SimpleNamespace(graph=_Graph())  # an unused graph in a cycle of its owner's
        doomed.itself, gone = doomed, weakref.ref(doomed.graph)
        del doomed
        _, step = _step()
        _run(step, 4)
    finally:
        gc.set_threshold(*old)
    assert capture_log.captures == 2 and capture_log.collections == 0
    assert gone() is None and gc.isenabled()


def test_a_failed_capture_turns_the_collector_on_again(capture_log):
    with pytest.raises(ValueError), T._capture(_Graph()):
        assert not gc.isenabled()
        raise ValueError
    assert gc.isenabled()
    gc.disable()
    try:
        with T._capture(_Graph()):
            pass
        assert not gc.isenabled()  # as the caller had it
    finally:
        gc.enable()


def test_flush_is_still_called_when_an_epoch_is_staged(capture_log):
    sampler, step = _step()
    _run(step, 4)
    assert step.pending == 1
    sampler.feed.on_stage()
    assert step.pending == 0 and step.graph.replays == 1
