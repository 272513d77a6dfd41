"""Which form attention of trees takes: the library's rule on the host again, so that tests can say which forms their calls reach."""


def form(seqs, tokens, heads, kv, d, max_pages, cus=256):
    """(rows of an item, pages shared out among workgroups)."""
    group = heads // kv
    rows = -(-tokens * group // seqs)
    pages = seqs * -(-rows // 128) * kv * max_pages
    blocks, waves = (1, 8 if d == 128 else 4) if rows <= 32 else (2, 8) if rows <= 64 or pages < 20 * cus else (4, 8)
    item, unit = 32 * blocks, waves // blocks
    items = min(tokens * group // item + seqs, tokens * -(-group // item))
    most_units = -(-max_pages // unit)
    chip = 8 // waves * cus
    likely = seqs * -(-rows // item) * kv
    idle = -(-likely // chip) * chip - likely
    wgs = min(items * most_units, max(chip // kv, 1))
    shared = not (most_units == 1 or most_units * idle <= 4 * chip) and wgs > 1
    return item, shared


# new and earlier tokens of each sequence, heads, heads of the cache: every form there is, for heads of any size
CASES = [([3], [4000], 8, 2), ([4, 2] * 30, [300, 270] * 30, 8, 4), ([40, 50], [3000, 2000], 8, 8), ([50] * 32, list(range(100, 260, 5)), 8, 8),
         ([128, 120], [5600, 5500], 32, 8), ([32] * 32, list(range(1250, 1314, 2)), 32, 8)]


def form_of(new, past, heads, kv, d):
    return form(len(new), sum(new), heads, kv, d, max(-(-(n + p) // 64) for n, p in zip(new, past)))
