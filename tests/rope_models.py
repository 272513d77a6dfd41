"""ONNX graphs with RotaryEmbedding, and what they compute (64 bits, numpy)."""
import numpy as np

import drafts_ref as D
from webdnn_amd import modelgen

# batch, heads, length, head size, rotated elements (0: all), pairs of neighbours, position ids, X of three dimensions
MODELS = [(1, 3, 5, 8, 0, 0, True, False), (2, 2, 7, 64, 0, 0, True, False), (2, 3, 4, 80, 36, 1, True, True), (3, 2, 6, 20, 10, 0, False, False),
          (2, 4, 9, 128, 0, 1, False, True), (1, 1, 1, 2, 0, 0, False, False), (2, 5, 33, 128, 0, 0, True, True), (3, 1, 3, 16, 6, 1, True, False)]


def model(batch, heads, length, d, rotary, interleaved, ids, three, seed=3):
    """(graph, x, y, bound): X -> RotaryEmbedding -> Y."""
    rng = np.random.default_rng(seed)
    g = modelgen.GraphBuilder(seed)
    half, rows = (rotary or d) // 2, 3 * length
    cos, sin = D.tables(rows if ids else batch * length, 2 * half)
    positions = rng.integers(0, rows, (batch, length)) if ids else np.arange(batch * length).reshape(batch, length)
    g.const("cos", cos if ids else cos.reshape(batch, length, half))
    g.const("sin", sin if ids else sin.reshape(batch, length, half))
    inputs = ["x", "cos", "sin"]
    if ids:
        g.const("ids", positions.astype(np.int64))
        inputs.append("ids")
    g.op("RotaryEmbedding", inputs, "y", interleaved=interleaved, rotary_embedding_dim=rotary, num_heads=heads if three else 0)
    shape = [batch, length, heads * d] if three else [batch, heads, length, d]
    x = rng.standard_normal((batch, length, heads, d)).astype(np.float32)
    place = lambda v: v.reshape(shape) if three else np.ascontiguousarray(np.moveaxis(v.reshape(x.shape), 1, 2))
    y, bound = D.rope(x.reshape(batch * length, heads, d), None, cos, sin, positions.ravel(), bool(interleaved), 0.0)
    return g.finish([("x", shape)], [("y", shape)], opset=23), place(x), place(y), place(bound)
