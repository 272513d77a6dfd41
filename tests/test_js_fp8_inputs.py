"""8-bit weights as a graph input that lives on the device: run node by node, recorded and replayed (Node.js host, without a GPU)."""
import os
import subprocess

import numpy as np

import fp8_ref as F
from webdnn_amd import modelgen

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
const fs = require("fs");
const WebDNN = require("./webdnn_amd/js");
const native = require("./tests/js/fake_native.js");
// ranges of copies as the library checks them
const sizes = new Map(), alloc = native.alloc, copy = native.copy;
native.alloc = (bytes) => { const h = alloc.call(native, bytes); sizes.set(h, bytes); return h; };
native.copy = (dst, doff, src, soff, bytes) => {
  if (doff + bytes > sizes.get(dst) || soff + bytes > sizes.get(src)) throw new Error("wdh_copy failed (-2): range exceeds a buffer");
  copy.call(native, dst, doff, src, soff, bytes);
};
(async () => {
  const dir = process.argv[1], runner = await WebDNN.load(dir, { backendOrder: ["hip"], optimized: false, strict: true, backendOptions: { hip: { native } } });
  const f = (name, T) => { const b = fs.readFileSync(`${dir}/${name}`); return new T(b.buffer.slice(b.byteOffset, b.byteOffset + b.length)); };
  const x = new WebDNN.CPUTensor([4, 200], "float32", f("x", Float32Array));
  const c = new WebDNN.CPUTensor([1, 2], "float32", f("c", Float32Array));
  const all = f("w", Uint8Array), hip = runner.backendContexts.hip, out = [];
  let replayed = 0;
  for (let i = 0; i < 6; i++) {
    const w = await hip.moveTensor(new WebDNN.CPUTensor([30, 200], "float8e4m3fn", all.subarray(6000 * i, 6000 * i + 6000)), {});
    out.push(...(await (await runner.run([x, w, c]))[0].getData()));
    if (runner.lastRunStats.graphReplay) replayed++;
    w.dispose();
  }
  fs.writeFileSync(`${dir}/y`, new Uint8Array(new Float32Array(out).buffer));
  console.log(replayed);
})().catch((e) => { console.error(e); process.exit(1); });
"""


def test_8_bit_weights_that_change_between_runs(tmp_path):
    g = modelgen.GraphBuilder(0)
    g.op("WebDNNHipMatMulFp8", ["x", "w", "c"], "y")
    (tmp_path / "model.onnx").write_bytes(g.finish([("x", [4, 200]), ("w", [30, 200]), ("c", [1, 2])], [("y", [4, 30])], opset=23))
    rng = np.random.default_rng(1)
    x, c = rng.standard_normal((4, 200)).astype(np.float32), np.array([[0.5, 0.25]], np.float32)
    w = (rng.integers(0, 127, (6, 30, 200)) | rng.integers(0, 2, (6, 30, 200)) << 7).astype(np.uint8)
    for name, t in (("x", x), ("c", c), ("w", w)):
        t.tofile(tmp_path / name)
    done = subprocess.run(["node", "-e", CODE, str(tmp_path)], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=100)
    assert done.returncode == 0, done.stderr
    assert int(done.stdout.split()[-1]) >= 3
    y = np.fromfile(tmp_path / "y", np.float32).reshape(6, 4, 30)
    # (the stand-in quantises rows of x by its definition, here too)
    scale = (np.maximum(F.finite_amax(F.block_view(x, 1), (1, 3)).astype(np.float32) / np.float32(448), np.float32(F.LEAST))).astype(np.float32)
    q = F.encode(x.astype(np.float64) / F.spread(scale, 1, x.shape))
    for i in range(6):
        want, size = F.product(q, scale, w[i], c)
        assert np.all(np.abs(y[i] - want) <= 2.0 ** -22 * size)
