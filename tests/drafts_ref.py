"""Positions, attention of trees, verification and keeping of drafted tokens from their definitions, in 64 bits on the CPU (numpy): what their
tests compare with."""
import numpy as np

import fp8_ref as F

E = 2.0 ** -24


def tables(rows, rotary, base=10000.0):
    angle = np.arange(rows)[:, None] * base ** (-2.0 * np.arange(rotary // 2) / rotary)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def rope(x, gamma, cos, sin, positions, interleaved, eps):
    """x [tokens, heads, d] -> (result, a bound of its error in fp32).  cos None: no rotation.

    A normed element is 3 roundings away (its factor's, and two products'), a bit more for their products with one another.  A rotated one: the second product is
    rounded, then the sum with the first: 2 more, relative to the two products' sizes.  Elements among the subnormal numbers are rounded to steps of 2^-149."""
    y = x.astype(np.float64)
    slack = 0.0
    if gamma is not None:
        y = F.rms(y, gamma.astype(np.float64), eps)
        slack = 3.01 * E
    out, bound = y.copy(), slack * np.abs(y)
    if cos is not None:
        half = cos.shape[1]
        known = (positions >= 0) & (positions < len(cos))
        for j in range(half):
            a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
            c, s = (np.where(known, t[np.where(known, positions, 0), j].astype(np.float64), np.nan)[:, None] for t in (cos, sin))
            out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
            bound[..., a] = (slack + 2.01 * E) * (np.abs(y[..., a] * c) + np.abs(y[..., b] * s))
            bound[..., b] = (slack + 2.01 * E) * (np.abs(y[..., b] * c) + np.abs(y[..., a] * s))
    return out, bound + 2.0 ** -147


def tree(rng, n, most_children):
    """Parents of a random tree of n rows, parents first."""
    parents, children = [-1], [0]
    for i in range(1, n):
        free = [j for j in range(i) if children[j] < most_children]
        up = free[rng.integers(0, len(free))]
        parents.append(up)
        children[up] += 1
        children.append(0)
    return np.array(parents, np.int32)


def attention(cache, q, table, lens, starts, sees, alpha):
    """Rows [tokens, heads, d] over all tokens before the call's and those of their own sequence that sees[row] (a list of booleans) names:
    (result, bound), as fp8_ref.Cache.attention has them."""
    eps, group = 2.0 ** -23, q.shape[1] // cache.heads
    out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
    for s in range(len(lens)):
        n, length = int(starts[s + 1] - starts[s]), int(lens[s])
        if n <= 0:
            continue
        k, v = cache.tokens(table[s], length)
        pages = -(-length // F.PAGE)
        for r in range(n):
            seen = np.concatenate([np.ones(length - n, bool), np.asarray(sees[starts[s] + r][:n], bool)])
            for h in range(q.shape[1]):
                if not seen.any():
                    out[starts[s] + r, h] = 0
                    continue
                kk, vv, qq = k[h // group][seen], v[h // group][seen], q[starts[s] + r, h].astype(np.float64)
                t = (kk @ qq) * alpha
                size = (np.abs(kk) @ np.abs(qq)).max() * abs(alpha)
                e = np.exp(t - t.max())
                out[starts[s] + r, h] = (e / e.sum()) @ vv
                chain = 2 * (3 * cache.d + 6) * size + 8 + (17 * pages + 12) + (7 * pages + 32)
                bound[starts[s] + r, h] = chain * eps * np.abs(vv).max()
    return out, bound


def pack(sees, words):
    """Rows of booleans as masks of `words` 32-bit words."""
    mask = np.zeros((len(sees), words), np.uint32)
    for r, row in enumerate(sees):
        for j, bit in enumerate(row[:32 * words]):
            if bit:
                mask[r, j // 32] |= np.uint32(1 << (j % 32))
    return mask.view(np.int32)


def unpack(mask, n):
    bits = (mask.view(np.uint32)[:, :, None] >> np.arange(32, dtype=np.uint32)) & 1
    bits = bits.reshape(len(mask), -1).astype(bool)
    return np.pad(bits, ((0, 0), (0, max(0, n - bits.shape[1]))))


def verify(p, draft, tokens, parents, uniform, starts):
    """(next, count, path): the walk as it is told, what is left of a row kept as a row."""
    seqs = len(starts) - 1
    token, count, path = np.full(seqs, -7, np.int32), np.full(seqs, -7, np.int32), np.full(len(tokens), -7, np.int32)
    weigh = lambda x: np.where(x > 0, x.astype(np.float64), 0.0)
    draft = None if draft is None else weigh(draft)
    for s in range(seqs):
        lo, n = int(starts[s]), int(starts[s + 1] - starts[s])
        if n <= 0:
            continue
        node, walk = 0, [0]
        while True:
            row = p[lo + node].astype(np.float64)
            left, mass, follow = weigh(row), 1.0, None
            for child in range(node + 1, n):
                if parents[lo + child] != node:
                    continue
                x = int(tokens[lo + child])
                real = 0 <= x < len(row)
                likely = (float(draft[lo + node, x]) if real else 0.0) if draft is not None else 1.0
                if float(uniform[lo + child]) * mass * likely < (left[x] if real else 0.0):
                    follow = child
                    break
                if draft is not None:
                    left = weigh(left - mass * draft[lo + node])
                    mass = left.sum()
                elif real:
                    mass -= left[x]
                    left[x] = 0
            if follow is None:
                break
            node = follow
            walk.append(node)
        if not left.sum() > 0:
            left = weigh(row)
        upto = np.cumsum(left)
        if upto[-1] > 0 and np.isfinite(upto[-1]):
            token[s] = np.argmax(upto > float(uniform[lo]) * upto[-1])
        else:
            token[s] = -1
        count[s] = len(walk) - 1
        path[lo:lo + n] = -1
        path[lo:lo + len(walk)] = walk
    return token, count, path


def keep(cache, table, lens, starts, path, count):
    """In place, on an fp8_ref.Cache."""
    for store, scales, turned in ((cache.k, cache.ks, False), (cache.v, cache.vs, True)):
        at = lambda position, s: (table[s][position // F.PAGE], position % F.PAGE)
        view = store.transpose(0, 1, 3, 2) if turned else store        # [pages, heads, tokens, d]
        for s in range(len(lens)):
            n = int(starts[s + 1] - starts[s])
            past, kept = int(lens[s]) - n, min(int(count[s]), n - 1) + 1
            if n <= 0 or kept <= 0:
                continue
            for page in range(past // F.PAGE, (past + kept - 1) // F.PAGE + 1):
                lo, hi = max(past, page * F.PAGE), min(past + kept, (page + 1) * F.PAGE)
                here = table[s][page]
                if not 0 <= here < cache.pages:
                    continue
                source = []
                for position in range(lo, hi):
                    j = int(path[starts[s] + position - past])
                    good = position - past < j < n and 0 <= at(past + j, s)[0] < cache.pages
                    source.append(at(past + j, s) if good else at(position, s))
                for h in range(cache.heads):
                    held = [(view[p, h, t].copy(), float(scales[p, h])) for p, t in source]
                    need = max(F.page_scale(F.finite_amax(F.decode(b) * c, None)) for b, c in held)
                    old = float(scales[here, h])
                    c = max(old, need)
                    if c != old:
                        before = view[here, h, :lo - page * F.PAGE]
                        before[:] = F.encode(F.decode(before) * (old / c))
                    for position, (b, was) in zip(range(lo, hi), held):
                        view[here, h, position % F.PAGE] = F.encode(F.decode(b) * (was / c))
                    scales[here, h] = c
