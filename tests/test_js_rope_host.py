"""RotaryEmbedding on the Node.js host without a GPU (tests/js/fake_native.js in place of the addon): layouts, batches, and what is refused."""
import numpy as np
import pytest

import node_runner
import rope_models
from webdnn_amd import modelgen


def run(tmp_path, data, inputs, **kw):
    (tmp_path / "model.onnx").write_bytes(data)
    return node_runner.run_model(str(tmp_path), inputs, "hip", strict=True, fake_native=True, **kw)


@pytest.mark.parametrize("case", rope_models.MODELS)
def test_rotary_embedding(tmp_path, case):
    data, x, y, bound = rope_models.model(*case)
    outs, rep = run(tmp_path, data, [x], runs=2)
    batch, three = case[0], case[7]
    assert rep["nodes"] == 1 and list(rep["stats"]["nodesByBackend"]) == ["hip"]
    assert rep["nativeCalls"]["rope"] == 2 * (1 if three else batch)
    assert rep["liveBuffers"] == rep["initializerCopies"]
    assert outs[0].shape == y.shape and np.all(np.abs(outs[0] - y) <= bound)


@pytest.mark.parametrize("shape,heads,rotary,table,ids,needle", [
    ([2, 6], 0, 0, [4, 3], None, "3 or 4 dimensions"),
    ([1, 4, 12], 0, 0, [1, 4, 3], None, "num_heads"),
    ([1, 4, 12], 5, 0, [1, 4, 3], None, "num_heads"),
    ([1, 2, 4, 6], 0, 5, [1, 4, 3], None, "5 rotated elements of 6"),
    ([1, 2, 4, 6], 0, 8, [1, 4, 4], None, "8 rotated elements of 6"),
    ([1, 2, 4, 7], 0, 0, [1, 4, 3], None, "7 rotated elements of 7"),
    ([1, 2, 4, 6], 0, 0, [1, 4, 2], None, "[1, 4, 3]"),
    ([1, 2, 4, 6], 0, 0, [4, 3], None, "[1, 4, 3]"),
    ([1, 2, 4, 6], 0, 0, [1, 4, 3], [1, 4], "[positions, 3]"),
    ([1, 2, 4, 6], 0, 0, [9, 3], [4], "position_ids"),
    ([1, 2, 4, 6], 0, 0, [9, 3], [1, 5], "position_ids"),
])
def test_what_rotary_embedding_refuses(tmp_path, shape, heads, rotary, table, ids, needle):
    g = modelgen.GraphBuilder(0)
    g.const("c", np.ones(table, np.float32))
    inputs = ["x", "c", "c"]
    if ids:
        g.const("ids", np.zeros(ids, np.int64))
        inputs.append("ids")
    g.op("RotaryEmbedding", inputs, "y", num_heads=heads, rotary_embedding_dim=rotary)
    with pytest.raises(RuntimeError) as err:
        run(tmp_path, g.finish([("x", shape)], [("y", shape)], opset=23), [np.zeros(shape, np.float32)])
    assert needle in str(err.value)


def test_position_ids_are_whole_numbers(tmp_path):
    g = modelgen.GraphBuilder(0)
    g.const("c", np.ones((9, 3), np.float32))
    g.const("ids", np.zeros((1, 4), np.float32))
    g.op("RotaryEmbedding", ["x", "c", "c", "ids"], "y")
    with pytest.raises(RuntimeError) as err:
        run(tmp_path, g.finish([("x", [1, 2, 4, 6])], [("y", [1, 2, 4, 6])], opset=23), [np.zeros((1, 2, 4, 6), np.float32)])
    assert "position_ids must be int32" in str(err.value)
