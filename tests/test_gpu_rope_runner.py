"""RotaryEmbedding through the Node.js runner on the GPU, and a step with drafted tokens through the N-API functions."""
import json
import os
import subprocess

import numpy as np
import pytest

import drafts_ref as D
import fp8_ref as F
import node_runner
import rope_models

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("case", rope_models.MODELS)
def test_rotary_embedding(tmp_path, case):
    """Node by node, and recorded and replayed: the same bits; and what the graph computes."""
    data, x, y, bound = rope_models.model(*case)
    (tmp_path / "model.onnx").write_bytes(data)
    outs, rep = node_runner.run_model(str(tmp_path), [x], "hip", strict=True, extra=["--no-graph"])
    assert rep["nodes"] == 1
    assert np.all(np.abs(outs[0] - y) <= bound)
    replayed, _ = node_runner.run_model(str(tmp_path), [x], "hip", strict=True, runs=4, extra=["--graph"])
    assert np.array_equal(outs[0], replayed[0])


def test_a_step_with_drafts_from_javascript(tmp_path):
    rng = np.random.default_rng(4)
    heads, kv, d, vocab, past, new = 4, 2, 64, 50, [3, 70], [4, 6]
    starts = np.concatenate([[0], np.cumsum(new)])
    tokens, seqs = int(sum(new)), 2
    table = np.array([[3, 0], [1, 2]])
    cos, sin = D.tables(100, d)
    parents = np.concatenate([D.tree(rng, n, 2) for n in new]).astype(np.int32)
    x = rng.standard_normal((tokens, heads + 2 * kv, d)).astype(np.float32)
    old = rng.standard_normal((sum(past), 2 * kv, d)).astype(np.float32)
    positions = np.concatenate([p + np.arange(n) for p, n in zip(past, new)]).astype(np.int32)
    c = F.Cache(4, kv, d)
    lens = np.array(past)
    c.append(old[:, :kv], old[:, kv:], table, lens, np.concatenate([[0], np.cumsum(past)]))
    sees = [[j == i or is_above(parents[s:], j, i) for j in range(n)] for s, n in zip(starts, new) for i in range(n)]
    q, _ = D.rope(x[:, :heads], None, cos, sin, positions, False, 0.0)
    words = 1
    mask = D.pack(sees, words)
    p = rng.dirichlet(np.ones(vocab), tokens).astype(np.float32)
    drafted = rng.integers(0, vocab, tokens).astype(np.int32)
    uniform = np.full(tokens, 0.001, np.float32)
    next_, count, path = D.verify(p, None, drafted, parents, uniform, starts)
    case = dict(heads=heads, kvHeads=kv, d=d, pages=4, maxPages=2, seqs=seqs, tokens=tokens, vocab=vocab, words=words, alpha=0.125, rows=100,
                table=table.ravel().tolist(), past=past, starts=starts.tolist(), oldStarts=np.concatenate([[0], np.cumsum(past)]).tolist(),
                positions=positions.tolist(), parents=parents.tolist(), drafted=drafted.tolist(),
                mask=np.asarray(mask).view(np.int32).ravel().tolist(), **{k: v.ravel().tolist() for k, v in
                                                                         dict(x=x, old=old, cos=cos, sin=sin, p=p, uniform=uniform).items()})
    (tmp_path / "case.json").write_text(json.dumps(case))
    out = tmp_path / "out.bin"
    done = subprocess.run(["node", os.path.join(HERE, "js", "drafts_native.js"), str(tmp_path / "case.json"), str(out)], stdout=subprocess.PIPE,
                          stderr=subprocess.STDOUT, text=True, timeout=100)
    assert done.returncode == 0, done.stdout
    said = json.loads(done.stdout.strip().splitlines()[-1])
    assert "head dimension 48" in said["refused"]
    assert said["next"] == next_.tolist() and said["count"] == count.tolist() and said["path"] == path.tolist()
    flat = np.fromfile(out, np.float32)
    turned, got = flat[:q.size].reshape(q.shape), flat[q.size:2 * q.size].reshape(q.shape)
    _, bound = D.rope(x[:, :heads], None, cos, sin, positions, False, 0.0)
    assert np.all(np.abs(turned - q) <= bound)
    # the cache takes the keys as the GPU turned them: rounded alike but where a rotation falls on a border, so scales and results are compared, not bytes
    turned_k = flat[2 * q.size:2 * q.size + tokens * kv * d].reshape(tokens, kv, d)
    c.append(turned_k, x[:, heads + kv:], table, np.array(past) + new, starts)
    want, bound = D.attention(c, turned, table, np.array(past) + new, starts, sees, 0.125)
    assert np.all(np.abs(got - want) <= bound)
    D.keep(c, table, np.array(past) + new, starts, path, count)
    scales = flat[2 * q.size + tokens * kv * d:]
    for at, s in ((0, c.ks), (c.ks.size, c.vs)):
        written = np.isfinite(s)
        assert np.array_equal(scales[at:at + s.size].reshape(s.shape)[written], s[written])


def is_above(parents, j, i):
    while i > 0:
        i = parents[i]
        if i == j:
            return True
    return False
