"""The 8-bit serving operators from their definitions, in 64 bits on the CPU (numpy): what their tests compare with."""
import numpy as np

BLOCK, PAGE = 128, 64
LEAST = 2.0 ** -100


def _decode_table():
    v = np.arange(256)
    sign, e, f = np.where(v & 128, -1.0, 1.0), (v >> 3) & 15, v & 7
    x = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    x[(v & 127) == 127] = np.nan
    return sign * x


VALUES = _decode_table()


def decode(q):
    return VALUES[q]


def half_step(x):
    """Half the distance between neighbouring e4m3 values at |x| (of the wider side where x is such a value)."""
    e = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -60)))
    return 2.0 ** (np.maximum(e, -6) - 4)


def encode(x):
    """Nearest e4m3 value (ties to even) as a byte; not finite -> 0x7f."""
    x = np.asarray(x, np.float64)
    fine = np.isfinite(x)
    y = np.where(fine, x, 0.0)
    step = 2 * half_step(y)
    r = np.clip(np.round(y / step) * step, -448, 448)           # np.round: ties to even
    order = np.argsort(VALUES[:127], kind="stable")
    byte = order[np.searchsorted(VALUES[:127], np.abs(r))]
    return np.where(fine, byte | np.where(np.signbit(y), 128, 0), 0x7f).astype(np.uint8)


def same_bytes(a, b):
    """Equal, or both NaN (either sign)."""
    return np.all((a == b) | (((a & 127) == 127) & ((b & 127) == 127)))


def finite_amax(x, axis):
    return np.where(np.isfinite(x), np.abs(x), 0.0).max(axis, initial=0.0)


def block_view(x, block_rows):
    """x [rows, cols] padded with zeros to [row blocks, block_rows, column blocks, 128]."""
    rows, cols = x.shape
    nr, nc = -(-rows // block_rows), -(-cols // BLOCK)
    p = np.zeros((nr * block_rows, nc * BLOCK), x.dtype)
    p[:rows, :cols] = x
    return p.reshape(nr, block_rows, nc, BLOCK)


def spread(scales, block_rows, shape):
    """Block scales to one for each element."""
    return np.repeat(np.repeat(scales.astype(np.float64), block_rows, 0), BLOCK, 1)[:shape[0], :shape[1]]


def check_quantized(q, scales, y, block_rows, eps_y, what=""):
    """q, scales (bytes, fp32) against the 64-bit rows y, which the kernel has to a relative eps_y: the scale is one more rounding
    away (the division by 448), a quotient two (the reciprocal and its product) and the half step of its e4m3 value."""
    e = 2.0 ** -24
    want = np.maximum(finite_amax(block_view(y, block_rows), (1, 3)) / 448, LEAST)
    assert scales.shape == want.shape, (what, scales.shape, want.shape)
    assert np.all(np.abs(scales - want) <= (eps_y + 1.01 * e) * want), what
    c = spread(scales, block_rows, y.shape)
    fine = np.isfinite(y)
    assert np.array_equal((q & 127) == 127, ~fine), what
    x = np.where(fine, y, 0.0) / c
    slack = (eps_y + 3.01 * e) * np.abs(x) + 2.0 ** -149 / c      # (a subnormal y is rounded to steps of 2^-149)
    off = np.abs(np.where(fine, decode(q), 0.0) - x)
    assert np.all(off <= half_step(x * (1 + 2.0 ** -20)) + slack), (what, float(np.max(off - slack)))


def rms(s, gamma, eps):
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + eps)
    return y if gamma is None else y * gamma


def product(a, sa, w, sw):
    """(Y, sum of the terms' sizes) in 64 bits from e4m3 bytes and scales."""
    af, wf = decode(a) * spread(sa, 1, a.shape), decode(w) * spread(sw, BLOCK, w.shape)
    return af @ wf.T, np.abs(af) @ np.abs(wf).T


def page_scale(amax):
    """Least 2^e >= amax / 448, e >= -100."""
    with np.errstate(divide="ignore"):
        e = np.ceil(np.log2(np.asarray(amax, np.float64) / 448))
    return 2.0 ** np.maximum(e, -100)


class Cache:
    """A cache as the operators have it: bytes and fp32 scales; junk everywhere that nobody has written."""

    def __init__(self, pages, heads, d):
        self.k = np.full((pages, heads, PAGE, d), 0x7f, np.uint8)
        self.v = np.full((pages, heads, d, PAGE), 0xff, np.uint8)
        self.ks, self.vs = np.full((pages, heads), np.nan, np.float32), np.full((pages, heads), np.nan, np.float32)
        self.pages, self.heads, self.d = pages, heads, d

    def append(self, k, v, table, lens, starts):
        """k, v: fp32 [tokens, heads, d]."""
        for s in range(len(lens)):
            n = starts[s + 1] - starts[s]
            for x, store, scales, turned in ((k, self.k, self.ks, False), (v, self.v, self.vs, True)):
                at, row = lens[s] - n, starts[s]
                while at < lens[s]:
                    page, slot = table[s][at // PAGE], at % PAGE
                    m = min(PAGE - slot, lens[s] - at)
                    new = x[row:row + m].astype(np.float64).transpose(1, 0, 2)
                    for h in range(self.heads):
                        c = page_scale(finite_amax(new[h], None))
                        view = store[page, h].T if turned else store[page, h]
                        if slot:
                            old = float(scales[page, h])
                            c = max(c, old)
                            if c != old:
                                view[:slot] = encode(decode(view[:slot]) * (old / c))
                        view[slot:slot + m] = encode(new[h] / c)
                        scales[page, h] = c
                    at, row = at + m, row + m

    def tokens(self, table_row, length):
        """(keys, values) of a sequence in 64 bits: [heads, length, d]."""
        p = np.asarray(table_row[:-(-length // PAGE)])
        k = decode(self.k[p]) * self.ks[p].astype(np.float64)[:, :, None, None]
        v = decode(self.v[p]) * self.vs[p].astype(np.float64)[:, :, None, None]
        return (k.transpose(1, 0, 2, 3).reshape(self.heads, -1, self.d)[:, :length],
                v.transpose(1, 0, 3, 2).reshape(self.heads, -1, self.d)[:, :length])

    def attention(self, q, table, lens, starts, alpha):
        """q [tokens, heads of q, d] -> (result in 64 bits, a bound of its error in fp32); rows of no sequence are NaN.

        A key's score is a sum of 3 d exact products (its query in three parts), each addition off by at most 2^-23 (fp32 additions
        of the matrix cores need not round to nearest) of the sizes' sum; a power of two is off by that, the rounding of its
        factor alpha log2(e) scale (3 roundings), of its argument and 2 ulp; the sum of weights is a chain of 16 additions for each page,
        a rescaling included, plus 12 across lanes, wavefronts and parts; the second product has 6 additions of 32 products each
        for each page.  Weights add up to 1, so all of it is relative to the largest |v|."""
        eps, group = 2.0 ** -23, q.shape[1] // self.heads
        out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
        for s in range(len(lens)):
            n, length = starts[s + 1] - starts[s], lens[s]
            if n <= 0:
                continue
            k, v = self.tokens(table[s], length)
            pages = -(-length // PAGE)
            for r in range(n):
                seen = length - n + r + 1
                for h in range(q.shape[1]):
                    kk, vv, qq = k[h // group, :seen], v[h // group, :seen], q[starts[s] + r, h].astype(np.float64)
                    t = (kk @ qq) * alpha
                    size = (np.abs(kk) @ np.abs(qq)).max() * abs(alpha) if seen else 0.0
                    e = np.exp(t - t.max())
                    out[starts[s] + r, h] = (e / e.sum()) @ vv
                    chain = 2 * (3 * self.d + 6) * size + 8 + (17 * pages + 12) + (7 * pages + 32)
                    bound[starts[s] + r, h] = chain * eps * np.abs(vv).max()
        return out, bound
