"""The rules of the operators for drafted tokens, without a GPU: verification leaves the target's distribution as it is; masks of trees; the refusals of
the Python and JavaScript bindings."""
import json
import os
import subprocess
import types

import numpy as np
import pytest

import drafts_ref as D
from webdnn_amd import hostops as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HUGE = 2 ** 32 + 5


def distribution_of_first_token(p, q, children):
    """Of the token that comes first when `children` drafts are drawn from q and tested as wdh_verify_drafts tests them, by its formulas: a draft is
    accepted with probability min(1, r / (s q)), and the rest of the probability goes on."""
    out, reach, t, s = np.zeros_like(p), 1.0, 0.0, 1.0
    for _ in range(children):
        r = np.maximum(p - t * q, 0)
        accept = np.minimum(1, np.divide(r, s * q, out=np.ones_like(p), where=q > 0))
        out += reach * q * accept
        reach *= 1 - (q * accept).sum()
        t, s = t + s, np.maximum(p - (t + s) * q, 0).sum()
        if s <= 0:
            return out + reach * p
    r = np.maximum(p - t * q, 0)
    return out + reach * r / r.sum()


@pytest.mark.parametrize("children", [0, 1, 2, 3, 7])
def test_drawn_drafts_leave_the_targets_distribution(children):
    rng = np.random.default_rng(children)
    for _ in range(20):
        p, q = (x / x.sum() for x in rng.gamma(0.4, size=(2, 40)) + 1e-12)
        assert np.abs(distribution_of_first_token(p, q, children) - p).max() < 1e-12


def test_chosen_drafts_leave_the_targets_distribution():
    """accept with p(x) / s, take it out, and the rest by its share: every token comes with p."""
    rng = np.random.default_rng(1)
    p = rng.dirichlet(np.ones(12))
    out, reach, s, left = np.zeros_like(p), 1.0, 1.0, p.copy()
    for x in (3, 7, 0):
        out[x] += reach * left[x] / s
        reach *= 1 - left[x] / s
        s -= left[x]
        left[x] = 0
    assert np.abs(out + reach * left / left.sum() - p).max() < 1e-14


def test_verification_by_many_draws_of_its_numbers():
    """The walk of the reference itself, on a small tree: how often each token comes first."""
    rng = np.random.default_rng(2)
    vocab, turns = 3, 40000
    p = rng.dirichlet(np.ones(vocab), 4).astype(np.float32)
    parents, starts = np.array([-1, 0, 0, 1], np.int32), np.array([0, 4], np.int32)
    by_token = np.stack([p[1], p[2], p[3]])            # what follows a first token, whichever row drafted it
    counts = np.zeros(vocab)
    draft = np.tile(np.array([0.5, 0.2, 0.3], np.float32), (4, 1))
    for _ in range(turns):
        tokens = np.concatenate([[0], rng.choice(vocab, 3, p=draft[0].astype(np.float64) / draft[0].sum(dtype=np.float64))]).astype(np.int32)
        rows = p.copy()
        for r in (1, 2, 3):
            rows[r] = by_token[tokens[r]]
        u = rng.random(4).astype(np.float32)
        token, count, path = D.verify(rows, draft, tokens, parents, u, starts)
        counts[tokens[path[1]] if count[0] else token[0]] += 1
    share = counts / turns
    assert np.all(np.abs(share - p[0]) <= 5 * np.sqrt(p[0] * (1 - p[0]) / turns))   # (five standard deviations of a share)


def test_tree_mask():
    starts = np.array([0, 4, 4, 44])
    parents = np.concatenate([[-1, 0, 0, 2], [-1] + list(range(39))]).astype(np.int32)
    mask = H.tree_mask(parents, starts)
    assert mask.dtype == np.int32 and mask.shape == (44, 2)
    sees = D.unpack(mask, 40)
    assert [np.flatnonzero(r).tolist() for r in sees[:4]] == [[0], [0, 1], [0, 2], [0, 2, 3]]
    assert all(sees[4 + r].tolist() == [True] * (r + 1) + [False] * (64 - r - 1) for r in range(40))
    assert np.array_equal(D.pack(sees, 2), mask)
    for bad in ([-1, 1], [-1, 5], [-2, 0]):
        with pytest.raises(H.OperatorError):
            H.tree_mask(np.array(bad), np.array([0, 2]))


# ---- bindings --------------------------------------------------------------------------------------
def tensor(*dims, data_type="float32"):
    length = 1
    for d in dims:
        length *= d
    return types.SimpleNamespace(dims=list(dims), ndim=len(dims), data_type=data_type, length=length, handle=1)


I32, E4M3 = "int32", "float8e4m3fn"


def cache(pages=2, heads=1, d=32):
    return H.KvCache(None, tensor(pages, heads, 64, d, data_type=E4M3), tensor(pages, heads), tensor(pages, heads, d, 64, data_type=E4M3), tensor(pages, heads))


def i32(*dims):
    return tensor(*dims, data_type=I32)


BAD = {
    "rows": lambda: H.rotary_embedding(None, tensor(3, 64), tensor(9, 16), tensor(9, 16), i32(3), 2, 33),
    "tables": lambda: H.rotary_embedding(None, tensor(3, 64), tensor(9, 16), tensor(9, 15), i32(3), 2, 32),
    "one table": lambda: H.rotary_embedding(None, tensor(3, 64), tensor(9, 16), None, i32(3), 2, 32),
    "wide table": lambda: H.rotary_embedding(None, tensor(3, 64), tensor(9, 17), tensor(9, 17), i32(3), 2, 32),
    "positions": lambda: H.rotary_embedding(None, tensor(3, 64), tensor(9, 16), tensor(9, 16), i32(2), 2, 32),
    "position type": lambda: H.rotary_embedding(None, tensor(3, 64), tensor(9, 16), tensor(9, 16), tensor(3), 2, 32),
    "scale": lambda: H.rotary_embedding(None, tensor(3, 64), tensor(9, 16), tensor(9, 16), i32(3), 2, 32, q_scale=tensor(31)),
    "out rows": lambda: H.rotary_embedding(None, tensor(3, 64), tensor(9, 16), tensor(9, 16), i32(3), 2, 32, out=tensor(4, 64)),
    "out width": lambda: H.rotary_embedding(None, tensor(3, 64), tensor(9, 16), tensor(9, 16), i32(3), 2, 32, out=tensor(3, 63)),
    "e4m3 rows": lambda: H.rotary_embedding(None, tensor(3, 64, data_type=E4M3), tensor(9, 16), tensor(9, 16), i32(3), 2, 32),
    "negative heads": lambda: H.rotary_embedding(None, tensor(3, 64), tensor(9, 16), tensor(9, 16), i32(3), -2, 32),
    "huge rows": lambda: H.rotary_embedding(None, tensor(HUGE, 64), tensor(9, 16), tensor(9, 16), i32(HUGE), 2, 32),
    "huge table": lambda: H.rotary_embedding(None, tensor(3, 64), tensor(HUGE, 16), tensor(HUGE, 16), i32(3), 2, 32, out=tensor(3, 64)),
    "append scale": lambda: H.cache_append_rotary(None, cache(), tensor(3, 32), tensor(3, 32), i32(1, 2), i32(1), i32(2), tensor(9, 16), tensor(9, 16), k_scale=tensor(33)),
    "append table": lambda: H.cache_append_rotary(None, cache(), tensor(3, 32), tensor(3, 32), i32(1, 2), i32(1), i32(2), tensor(9, 17), tensor(9, 17)),
    "append values": lambda: H.cache_append_rotary(None, cache(), tensor(3, 32), tensor(4, 32), i32(1, 2), i32(1), i32(2), tensor(9, 16), tensor(9, 16)),
    "append positions": lambda: H.cache_append_rotary(None, cache(), tensor(3, 32), tensor(3, 32), i32(1, 2), i32(1), i32(2), tensor(9, 16), tensor(9, 16), i32(4)),
    "mask rows": lambda: H.cache_attention_tree(None, cache(), tensor(3, 64), 2, 1.0, i32(1, 2), i32(1), i32(2), i32(2, 1), out=tensor(3, 64)),
    "mask words": lambda: H.cache_attention_tree(None, cache(), tensor(3, 64), 2, 1.0, i32(1, 2), i32(1), i32(2), i32(3, 0), out=tensor(3, 64)),
    "mask type": lambda: H.cache_attention_tree(None, cache(), tensor(3, 64), 2, 1.0, i32(1, 2), i32(1), i32(2), tensor(3, 1), out=tensor(3, 64)),
    "mask heads": lambda: H.cache_attention_tree(None, cache(heads=2), tensor(3, 96), 3, 1.0, i32(1, 2), i32(1), i32(2), i32(3, 1), out=tensor(3, 96)),
    "draft": lambda: H.verify_drafts(None, tensor(3, 9), i32(3), i32(3), tensor(3), i32(2), draft=tensor(3, 8)),
    "tokens": lambda: H.verify_drafts(None, tensor(3, 9), i32(4), i32(3), tensor(3), i32(2)),
    "uniform": lambda: H.verify_drafts(None, tensor(3, 9), i32(3), i32(3), i32(3), i32(2)),
    "starts": lambda: H.verify_drafts(None, tensor(3, 9), i32(3), i32(3), tensor(3), i32(0)),
    "out": lambda: H.verify_drafts(None, tensor(3, 9), i32(3), i32(3), tensor(3), i32(2), out=(i32(2), i32(1), i32(3))),
    "huge vocabulary": lambda: H.verify_drafts(None, tensor(3, HUGE), i32(3), i32(3), tensor(3), i32(2)),
    "path": lambda: H.cache_keep(None, cache(), i32(1, 2), i32(1), i32(2), tensor(3), i32(1)),
    "count": lambda: H.cache_keep(None, cache(), i32(1, 2), i32(1), i32(2), i32(3), i32(2)),
}


@pytest.mark.parametrize("what", sorted(BAD))
def test_python_refuses(what, monkeypatch):
    monkeypatch.setattr(H, "call", lambda name, *args: pytest.fail("%s%r was called" % (name, args)))
    with pytest.raises(H.OperatorError):
        BAD[what]()


def test_javascript_refuses_what_32_bits_do_not_hold():
    code = """
const n = require("./webdnn_amd/lib/webdnn_hip.node"), huge = 2 ** 32 + 5, told = [];
const calls = [["rope", 21, [14, 15, 16, 17, 18, 19]], ["cacheAppendRope", 27, [17, 18, 19, 20, 21, 22, 23, 24, 25]],
               ["cacheAttentionTree", 21, [12, 13, 14, 15, 16, 17, 18, 19]], ["verifyDrafts", 12, [9, 10, 11]], ["cacheKeep", 15, [9, 10, 11, 12, 13, 14]]];
for (const [name, count, places] of calls)
  for (const at of places)
    for (const value of [huge, -huge, 2 ** 31]) {
      const args = Array(count).fill(1);
      args[at] = value;
      try { n[name](...args); told.push("none"); } catch (e) { told.push(e.message); }
    }
console.log(JSON.stringify(told));
"""
    out = subprocess.run(["node", "-e", code], cwd=ROOT, stdout=subprocess.PIPE, text=True, check=True, timeout=60).stdout
    told = json.loads(out.strip().splitlines()[-1])
    assert len(told) == 96 and all("32 bits" in message for message in told), told
