"""Root-mean-square norms and 8-bit linear layers on the Node.js host without a GPU (tests/js/fake_native.js in place of the addon):
operators, the fusion of Add and norm, 8-bit initializers, and what is refused."""
import json
import os
import subprocess

import numpy as np
import pytest

import fp8_models
import fp8_ref as F
import node_runner
from util import assert_bit_exact
from webdnn_amd import modelgen

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(tmp_path, data, inputs, **kw):
    (tmp_path / "model.onnx").write_bytes(data)
    return node_runner.run_model(str(tmp_path), inputs, "hip", strict=True, fake_native=True, **kw)


def test_a_block_with_8_bit_weights(tmp_path):
    data, compute = fp8_models.block_model()
    rng = np.random.default_rng(1)
    x, r = (rng.standard_normal((1, 7, 72)).astype(np.float32) for _ in range(2))
    outs, rep = run(tmp_path, data, [x, r], runs=2)
    assert rep["nodes"] == 4 and list(rep["stats"]["nodesByBackend"]) == ["hip"]
    calls = rep["nativeCalls"]
    assert calls["rmsnorm"] == 4 and calls["gemmFp8"] == 4 and calls["quantizeFp8"] == 4 and "binary" not in calls
    assert rep["liveBuffers"] == rep["initializerCopies"]
    plain, rep = run(tmp_path, data, [x, r], fuse=False)
    assert rep["nodes"] == 6 and rep["nativeCalls"]["binary"] == 2
    y, s2 = compute(x, r)
    for got, other, want in zip(outs, plain, (y, s2)):
        assert_bit_exact(got, other, "fused and not")
        assert np.max(np.abs(got - want)) <= fp8_models.FLIPS * np.max(np.abs(want))


def test_a_broadcasting_addend_goes_through_the_add_kernel(tmp_path):
    g = modelgen.GraphBuilder(0)
    g.const("row", np.arange(6, dtype=np.float32))
    g.const("g", np.linspace(0.5, 2, 6).astype(np.float32))
    g.op("Add", ["x", "row"], "s")
    g.op("RMSNormalization", ["s", "g"], "y")
    data = g.finish([("x", [3, 6])], [("y", [3, 6]), ("s", [3, 6])], opset=23)
    x = np.random.default_rng(2).standard_normal((3, 6)).astype(np.float32)
    outs, rep = run(tmp_path, data, [x])
    assert rep["nodes"] == 1 and rep["nativeCalls"]["binary"] == 1 and rep["nativeCalls"]["rmsnorm"] == 1
    s = x + np.arange(6, dtype=np.float32)
    assert np.array_equal(outs[1], s)
    want = F.rms(s.astype(np.float64), np.linspace(0.5, 2, 6).astype(np.float32).astype(np.float64), 1e-5)
    assert np.all(np.abs(outs[0] - want) <= 3.01 * 2.0 ** -24 * np.abs(want))


def test_fusion_takes_the_norms_whose_scale_is_known():
    code = """
const { fuseAddRMSNorm } = require("./webdnn_amd/js/core/modelTransform");
const nd = (opType, input, output) => ({ opType, input, output, name: output[0], attribute: [] });
const init = (name) => ({ name, dims: [4], dataType: 1, floatData: [0, 0, 0, 0] });
const graph = {
  node: [nd("Add", ["x", "r"], ["s"]), nd("Relu", ["s"], ["q"]), nd("RMSNormalization", ["s", "g"], ["n"]),
         nd("RMSNormalization", ["s", "g"], ["again"]), nd("Add", ["n", "q"], ["t"]), nd("Relu", ["q"], ["late"]),
         nd("RMSNormalization", ["t", "late"], ["u"]), nd("RMSNormalization", ["x", "g"], ["v"])],
  initializer: [init("g")], input: [{ name: "x" }, { name: "r" }], output: [{ name: "u" }],
};
const count = fuseAddRMSNorm(graph);
console.log(JSON.stringify([count, graph.node.map((n) => [n.opType, n.input.join(), n.output.join()])]));
"""
    out = subprocess.run(["node", "-e", code], cwd=ROOT, stdout=subprocess.PIPE, text=True, check=True).stdout
    count, nodes = json.loads(out.strip().splitlines()[-1])
    assert count == 1 and nodes == [
        ["WebDNNHipAddRMSNorm", "x,r,g", "s,n"], ["Relu", "s", "q"], ["RMSNormalization", "s,g", "again"], ["Add", "n,q", "t"],
        ["Relu", "q", "late"], ["RMSNormalization", "t,late", "u"], ["RMSNormalization", "x,g", "v"]]


@pytest.mark.parametrize("change, needle", [
    (dict(w=np.zeros((10, 8), np.float32)), "float8e4m3fn"),
    (dict(c=np.zeros((2, 1), np.float32)), "one scale for each"),
    (dict(w=np.zeros((10, 9), np.uint8)), "inner dimensions"),
    (dict(b=np.zeros(9, np.float32)), "bias"),
    (dict(activation="Gelu"), "activation"),
])
def test_what_an_8_bit_layer_refuses(tmp_path, change, needle):
    g = modelgen.GraphBuilder(0)
    g.const("w", change.get("w", np.zeros((10, 8), np.uint8)))
    g.const("c", change.get("c", np.ones((1, 1), np.float32)))
    g.const("b", change.get("b", np.zeros(10, np.float32)))
    g.op("WebDNNHipMatMulFp8", ["x", "w", "c", "b"], "y", activation=change.get("activation", ""))
    data = g.finish([("x", [3, 8])], [("y", [3, 10])], opset=23)
    with pytest.raises(RuntimeError) as err:
        run(tmp_path, data, [np.zeros((3, 8), np.float32)])
    assert needle in str(err.value)


def test_e4m3_of_the_stand_in_is_the_restatements(tmp_path):
    """Every e4m3 value passes through an 8-bit layer's weights as itself, and rows are quantised alike."""
    w = np.arange(256, dtype=np.uint8)[np.arange(256) & 127 != 127].reshape(1, 254)
    x = np.random.default_rng(3).standard_normal((4, 254)).astype(np.float32)
    g = modelgen.GraphBuilder(0)
    g.const("w", w)
    g.const("c", np.array([[0.5, 2.0]], np.float32))
    g.op("WebDNNHipMatMulFp8", ["x", "w", "c"], "y")
    outs, _ = run(tmp_path, g.finish([("x", [4, 254])], [("y", [4, 1])], opset=23), [x])
    q, c = fp8_models.quantize_rows(x.astype(np.float64))
    want, size = F.product(q, c, w, np.array([[0.5, 2.0]], np.float32))
    assert np.all(np.abs(outs[0] - want) <= 2.0 ** -23 * size)
