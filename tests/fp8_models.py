"""ONNX graphs with root-mean-square norms and 8-bit linear layers, and what they compute (64 bits, numpy)."""
import numpy as np

import fp8_ref as F
from webdnn_amd import modelgen


# Of a value that a layer quantises, the fp32 and the 64-bit form (2^-21 apart at most) round to neighbouring e4m3 values about once in 10^5
# values; the step, at most 2^-3 of the value, reaches a result as one term of a sum of 72 to 1000, or spread over the terms of the
# second layer: under 2^-5 of the largest result, while a lost scale, bias or addend is of its size.
FLIPS = 2.0 ** -5


def quantize_rows(x):
    """What the layer does to its input: the e4m3 values and their scales, [rows, ...]."""
    c = np.maximum(F.finite_amax(F.block_view(x, 1), (1, 3)).astype(np.float32) / np.float32(448), np.float32(F.LEAST)).astype(np.float32)
    return F.encode((x / F.spread(c, 1, x.shape)).astype(np.float32)), c


def quantize_weight(w):
    c = (F.finite_amax(F.block_view(w, 128), (1, 3)) / 448).astype(np.float32)
    return F.encode(w / F.spread(c, 128, w.shape)), c


def block_model(tokens=7, width=72, hidden=200, seed=5):
    """x, r -> s = x + r; h = relu(rms(s) W1^T + b1); s2 = s + h W2^T; y = rms(s2): the second half of a decoder block."""
    g = modelgen.GraphBuilder(seed)
    rng = np.random.default_rng(seed)
    w1, c1 = quantize_weight((rng.standard_normal((hidden, width)) * width ** -0.5).astype(np.float32))
    w2, c2 = quantize_weight((rng.standard_normal((width, hidden)) * hidden ** -0.5).astype(np.float32))
    b1 = rng.standard_normal(hidden).astype(np.float32)
    g1, g2 = (rng.uniform(0.5, 1.5, width).astype(np.float32) for _ in range(2))
    for name, a in (("w1", w1), ("c1", c1), ("w2", w2), ("c2", c2), ("b1", b1), ("g1", g1), ("g2", g2)):
        g.const(name, a)
    g.op("Add", ["x", "r"], "s")
    g.op("RMSNormalization", ["s", "g1"], "n", axis=-1, epsilon=1e-6)
    g.op("WebDNNHipMatMulFp8", ["n", "w1", "c1", "b1"], "h", activation="Relu")
    g.op("WebDNNHipMatMulFp8", ["h", "w2", "c2"], "f")
    g.op("Add", ["s", "f"], "s2")
    g.op("RMSNormalization", ["s2", "g2"], "y", axis=-1, epsilon=1e-6)
    data = g.finish([("x", [1, tokens, width]), ("r", [1, tokens, width])], [("y", [1, tokens, width]), ("s2", [1, tokens, width])], opset=23)

    def compute(x, r):
        """(y, s2) in 64 bits but for the two quantisations."""
        s = (x + r).astype(np.float64)[0]
        n8, nc = quantize_rows(F.rms(s, g1.astype(np.float64), 1e-6))
        h = np.maximum(F.product(n8, nc, w1, c1)[0] + b1, 0)
        h8, hc = quantize_rows(h)
        f, _ = F.product(h8, hc, w2, c2)
        s2 = s + f
        return F.rms(s2, g2.astype(np.float64), 1e-6)[None], s2[None]

    return data, compute
