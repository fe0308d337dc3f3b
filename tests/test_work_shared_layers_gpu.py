"""layers.Dropout in graph captures and over a checkpoint, on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_dropout_layer_first_used_in_a_capture(cuda):
    """Refused while its counter would be made by the graph; after a forward outside, replays draw new masks."""
    from FoodRec.engine import layers, native, ops
    layer, x = layers.Dropout(0.5), torch.ones(70, 33, device=cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = x * 2
        with pytest.raises(native.EngineError, match="cannot be captured"):
            layer(x)
    graph.replay()
    assert torch.equal(y, 2 * x)
    layer(x)
    state = layer.mask_state()
    assert state["step"] == 1
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = layer(x)
    seen = []
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.dropout(x, 0.5, state["seed"], torch.tensor([1 + k], device=cuda)))
        seen.append(y.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
    layer.load_mask_state(state, cuda)  # the graph goes on from there, too
    graph.replay()
    assert torch.equal(y, seen[0])
    resumed = layers.Dropout(0.5)
    resumed.load_mask_state(layer.mask_state(), cuda)
    assert torch.equal(resumed(x), layer(x))
