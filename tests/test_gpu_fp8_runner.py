"""Root-mean-square norms and 8-bit linear layers through the Node.js runner on the GPU, and the cache through the N-API functions."""
import json
import os
import subprocess

import numpy as np
import pytest

import fp8_models
import fp8_ref as F
import node_runner

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("tokens,width,hidden", [(7, 72, 200), (40, 256, 1000)])
def test_a_block_with_8_bit_weights(tmp_path, tokens, width, hidden):
    """Node by node, and recorded and replayed: the same bits; and what the graph computes."""
    data, compute = fp8_models.block_model(tokens, width, hidden)
    (tmp_path / "model.onnx").write_bytes(data)
    rng = np.random.default_rng(1)
    x, r = (rng.standard_normal((1, tokens, width)).astype(np.float32) for _ in range(2))
    outs, rep = node_runner.run_model(str(tmp_path), [x, r], "hip", strict=True, extra=["--no-graph"])
    assert rep["nodes"] == 4
    replayed, _ = node_runner.run_model(str(tmp_path), [x, r], "hip", strict=True, runs=4, extra=["--graph"])
    apart, rep = node_runner.run_model(str(tmp_path), [x, r], "hip", strict=True, fuse=False)
    assert rep["nodes"] == 6
    for got, again, plain, want in zip(outs, replayed, apart, compute(x, r)):
        assert np.array_equal(got, again) and np.array_equal(got, plain)
        assert np.max(np.abs(got - want)) <= fp8_models.FLIPS * np.max(np.abs(want))


def test_the_cache_from_javascript(tmp_path):
    rng = np.random.default_rng(4)
    heads, kv, d, new = 4, 2, 64, [70, 1, 3]
    lens, starts = np.array(new), np.concatenate([[0], np.cumsum(new)])
    table, tokens = np.array([[3, 0], [1, -1], [4, -1]]), int(sum(new))
    k, v = (rng.standard_normal((tokens, kv, d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((tokens, heads, d)).astype(np.float32)
    c = F.Cache(6, kv, d)
    c.append(k, v, table, lens, starts)
    want, bound = c.attention(q, table, lens, starts, 0.125)
    case = dict(heads=heads, kvHeads=kv, d=d, pages=6, maxPages=2, seqs=3, tokens=tokens, alpha=0.125, table=table.ravel().tolist(),
                lens=lens.tolist(), starts=starts.tolist(), q=q.ravel().tolist(),
                kv=np.concatenate([k.reshape(tokens, -1), v.reshape(tokens, -1)], 1).ravel().tolist())
    (tmp_path / "case.json").write_text(json.dumps(case))
    out = tmp_path / "out.bin"
    done = subprocess.run(["node", os.path.join(HERE, "js", "cache_native.js"), str(tmp_path / "case.json"), str(out)], stdout=subprocess.PIPE,
                          stderr=subprocess.STDOUT, text=True, timeout=100)
    assert done.returncode == 0, done.stdout
    assert "head dimension 48" in json.loads(done.stdout.strip().splitlines()[-1])["refused"]
    flat = np.fromfile(out, np.float32)
    got = flat[:q.size].reshape(q.shape)
    assert np.all(np.abs(got - want) <= bound)
    for at, scales in ((q.size, c.ks), (q.size + c.ks.size, c.vs)):
        written = np.isfinite(scales)
        assert np.array_equal(flat[at:at + scales.size].reshape(scales.shape)[written], scales[written])
