"""What a serving step with drafted tokens adds to the 8-bit serving operators, as cases that can be timed: positions (rotation of
queries and keys, after a norm of each head), appending to the cache with both on the way, attention for a tree of drafted tokens over the
cache, verification of the drafts against the target's probabilities, and keeping the accepted tokens in the cache.

A pass is one call as a program in a serving loop makes it: operands lie on the device, results go to buffers that the
program keeps.  `own = False` computes the same from elementary torch operations, in 32 bits or, for sums over a vocabulary, in 64.

Layouts (row-major): rows of heads * d elements; rotation tables [positions, rotary / 2]; cache pages of 64 tokens, keys
[pages, heads, 64, d], values [pages, heads, d, 64] in e4m3, scales [pages, heads]; table [sequences, most pages] of page numbers,
lens [sequences] with the tokens of this call counted, starts [sequences + 1]: which rows of the call belong to which sequence (they
are the last of its lens tokens).  A tree's rows come parents first; parents [rows]: the row's parent as a row of its own sequence,
-1 for the first; mask [rows, words]: bit j of a row is set where it sees row j of its sequence.
"""
import math

import torch

own = False

PAGE, E4M3_MAX, EPS = 64, 448.0, 1e-6


def listed():
    return [
        # one token of each of four conversations through a layer with normed queries and keys: latency is all there is
        dict(name="rope_4x40x128", kind="rope", tokens=4, heads=32, kv_heads=8, d=128, rotary=128, interleaved=False, norm=True),
        # a batch of prompts through the same layer
        dict(name="rope_8192x40x128", kind="rope", tokens=8192, heads=32, kv_heads=8, d=128, rotary=128, interleaved=False, norm=True),
        # heads of an odd size of which a part is rotated, neighbours as pairs, no norm
        dict(name="rope_1001x15x80", kind="rope", tokens=1001, heads=12, kv_heads=3, d=80, rotary=36, interleaved=True, norm=False),
        # one new token for each of 48 sequences
        dict(name="append_48_tokens", kind="append", seqs=48, new=1, spread=0, past=1000, kv_heads=8, d=128, rotary=128, interleaved=False, norm=True),
        # a batch of prompts of different lengths goes into an empty cache
        dict(name="append_6_prompts", kind="append", seqs=6, new=1500, spread=1400, past=0, kv_heads=8, d=128, rotary=128, interleaved=False, norm=True),
        # sixteen conversations of different lengths, a tree of 32 tokens for each
        dict(name="tree_16x32", kind="tree", seqs=16, new=32, spread=0, width=3, past=4500, past_spread=4000, heads=32, kv_heads=8, d=128),
        # one long conversation with a wide tree: the cache of one sequence has to fill the chip
        dict(name="tree_64_behind_100000", kind="tree", seqs=1, new=64, spread=0, width=4, past=100000, past_spread=0, heads=16, kv_heads=2, d=128),
        # many short conversations with small trees of different sizes
        dict(name="tree_64x8", kind="tree", seqs=64, new=8, spread=4, width=2, past=700, past_spread=650, heads=16, kv_heads=4, d=64),
        # four drafted tokens in a row for each of 32 sequences, drawn from a small model's probabilities
        dict(name="verify_32x5_of_128000", kind="verify", seqs=32, new=5, spread=0, width=1, vocab=128000, drawn=True),
        # a tree of a small model's likeliest continuations for one sequence, a vocabulary of odd size
        dict(name="verify_33_of_50001", kind="verify", seqs=1, new=33, spread=0, width=3, vocab=50001, drawn=False),
        # a tree of 32 tokens for each of 16 sequences, of which a path is kept
        dict(name="keep_16x32", kind="keep", seqs=16, new=32, spread=0, width=3, past=4500, past_spread=4000, kv_heads=8, d=128),
        # small trees of many sequences
        dict(name="keep_200x9", kind="keep", seqs=200, new=9, spread=5, width=2, past=300, past_spread=250, kv_heads=4, d=64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "append", "tree", "tree", "tree", "verify", "verify", "keep"])
    norm, interleaved = rng.random() < 0.6, rng.random() < 0.3
    if kind == "rope":
        d = rng.choice([32, 48, 64, 80, 96, 128, 128, 128, 200, 256])
        rotary = d if rng.random() < 0.6 else 2 * rng.randint(1, d // 2)
        heads, kv = rng.randint(1, 48), rng.choice([0, 1, 2, 4, 8])
        return dict(kind=kind, tokens=_log_int(rng, 1, 8192 * 5120 // ((heads + kv) * d)), heads=heads, kv_heads=kv, d=d, rotary=rotary,
                    interleaved=interleaved, norm=norm)
    d, kv = rng.choice([32, 64, 128, 128]), rng.choice([1, 2, 4, 8])
    if kind == "append":
        rotary = d if rng.random() < 0.6 else 2 * rng.randint(1, d // 2)
        if rng.random() < 0.5:
            return dict(kind=kind, seqs=_log_int(rng, 1, 200), new=rng.choice([1, 1, 4]), spread=0, past=_log_int(rng, 1, 2000), kv_heads=kv, d=d,
                        rotary=rotary, interleaved=interleaved, norm=norm)
        seqs = _log_int(rng, 1, 16)
        new = _log_int(rng, 16, 9000 // seqs)
        return dict(kind=kind, seqs=seqs, new=new, spread=new // 2, past=rng.choice([0, 0, 100, 700]), kv_heads=kv, d=d, rotary=rotary,
                    interleaved=interleaved, norm=norm)
    seqs = _log_int(rng, 1, 64)
    if kind == "verify":
        new = _log_int(rng, 2, 64)
        return dict(kind=kind, seqs=seqs, new=new, spread=new // 3, width=rng.choice([1, 1, 2, 3, 4]), drawn=rng.random() < 0.5,
                    vocab=_log_int(rng, 1000, min(160000, 20_000_000 // (seqs * new))))
    if kind == "keep":
        new = _log_int(rng, 2, 130)
        past = _log_int(rng, 1, 4000)
        return dict(kind=kind, seqs=seqs, new=new, spread=new // 3, width=rng.choice([1, 2, 3]), past=past, past_spread=past // 2, kv_heads=kv, d=d)
    heads = kv * rng.choice([1, 2, 4, 8])
    new = _log_int(rng, 2, 130 if seqs < 8 else 40)
    past = _log_int(rng, 1, max(64, min(100000, 3_000_000 // (seqs * new))))
    return dict(kind=kind, seqs=seqs, new=new, spread=new // 3, width=rng.choice([1, 2, 3, 4]), past=past, past_spread=past // 2,
                heads=min(heads, 32), kv_heads=kv, d=d)


# ---- the cache's 8-bit form, in plain torch --------------------------------------------------
def _finite_amax(x, dims):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dims)


def _to_e4m3(x):
    """Nearest e4m3 value; what is not finite becomes NaN."""
    return torch.where(torch.isfinite(x), x.clamp(-E4M3_MAX, E4M3_MAX), torch.full_like(x, math.nan)).to(torch.float8_e4m3fn)


def _power_of_two_scale(amax):
    """The least 2^e with amax <= 448 * 2^e, and e >= -100 (448 is 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), torch.clamp(torch.where(m <= 0.875, e - 9, e - 8), min=-100))


# ---- inputs --------------------------------------------------------------------------------
def _counts(c):
    """How many rows of the call each sequence has, and how many tokens lie before them."""
    steps = torch.linspace(-1, 1, c["seqs"]) if c["seqs"] > 1 else torch.zeros(1)
    new = (c["new"] + (steps * c["spread"]).round()).int().clamp(min=1)
    return new, (c.get("past", 0) + (steps.flip(0) * c.get("past_spread", 0)).round()).int()


def _tree(new, width):
    """Parents of trees in which a token has `width` continuations, and for each row its sequence and its place there."""
    seq = torch.repeat_interleave(torch.arange(len(new)), new.long())
    place = torch.arange(len(seq)) - (torch.cumsum(new, 0) - new)[seq]
    return torch.where(place > 0, (place - 1) // width, -1).int(), seq, place


def _tables(rows, rotary, device):
    """cos and sin of position * 10000^(-2j/rotary), the angles in 64 bits."""
    j = torch.arange(rotary // 2, dtype=torch.float64, device=device)
    angle = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * torch.pow(10000.0, -2 * j / rotary)
    return angle.cos().float(), angle.sin().float()


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    uniform = lambda lo, hi, *shape: torch.rand(shape, generator=g, device="cuda") * (hi - lo) + lo
    s = {}
    if c["kind"] == "rope":
        # rows of a projection: queries, keys, and the values behind them, which are left alone
        s["cos"], s["sin"] = _tables(9000, c["rotary"], "cuda")
        s["x"] = normal(c["tokens"], (c["heads"] + 2 * c["kv_heads"]) * c["d"]) * torch.exp(normal(1, (c["heads"] + 2 * c["kv_heads"]) * c["d"]) * 0.5)
        first = int(torch.randint(0, 500, (1,), generator=cpu))
        s["positions"] = (first + torch.arange(c["tokens"], device="cuda") % (9000 - first)).int()
        if c["norm"]:
            s["q_gamma"], s["k_gamma"] = uniform(0.5, 1.5, c["d"]), uniform(0.5, 1.5, c["d"])
        return s
    new, past = _counts(c)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(new, 0)]).int()
    tokens = int(starts[-1])
    s["starts"] = starts.cuda()
    parents, seq, place = _tree(new, c.get("width", 1))
    if c["kind"] == "verify":
        s["parents"] = parents.cuda()
        logits = normal(tokens, c["vocab"]) * 2.5
        s["p"] = torch.softmax(logits, 1)
        draft = torch.softmax(logits + normal(tokens, c["vocab"]) * 0.7, 1)
        above = (starts[:-1].long()[seq] + parents.clamp(min=0)).cuda()
        if c["drawn"]:
            token = torch.searchsorted(torch.cumsum(draft[above].double(), 1), uniform(0, 0.999999, tokens, 1).double(), right=True)[:, 0]
            s["draft"] = draft
        else:  # the likeliest ones, the first child's token first
            best = torch.topk(draft, c["width"], 1).indices
            token = best[above, ((place - 1).clamp(min=0) % c["width"]).cuda()]
        s["tokens"] = token.clamp(max=c["vocab"] - 1).int()
        s["uniform"] = uniform(0, 1, tokens).clamp(max=1 - 2.0 ** -24)
        return s
    # on which pages the sequences lie
    lens = past + new
    count = (lens + PAGE - 1) // PAGE
    pages, most = int(count.sum()) + 3, int(count.max())
    order = torch.randperm(pages, generator=cpu).int()
    first = torch.cumsum(count, 0) - count
    column = torch.arange(most)
    table = torch.where(column < count[:, None], order[(first[:, None] + column).clamp(max=pages - 1)], torch.zeros((), dtype=torch.int32))
    s.update(table=table.cuda(), lens=lens.cuda())
    kv, d = c["kv_heads"], c["d"]
    keys, values = normal(pages, kv, PAGE, d), normal(pages, kv, d, PAGE)
    if c["kind"] == "keep":  # (pages whose scales differ)
        keys, values = (x * torch.exp2(torch.randint(-1, 2, (pages, kv, 1, 1), generator=g, device="cuda").float()) for x in (keys, values))
    for name, x in (("k", keys), ("v", values)):
        scale = _power_of_two_scale(x.abs().amax((2, 3)))
        s[name + "_pages"], s[name + "_scales"] = _to_e4m3(x / scale[:, :, None, None]), scale
    del keys, values, x
    if c["kind"] == "append":
        s["cos"], s["sin"] = _tables(int(lens.max()) + 1, c["rotary"], "cuda")
        s["positions"] = (past[seq] + place).int().cuda()
        # keys and values are the ends of a projection's rows; now and then a token outgrows what its page held so far
        s["kv"] = normal(tokens, 2 * kv * d) * torch.where(uniform(0, 1, tokens, 1) < 0.1, 3.0, 1.0)
        if c["norm"]:
            s["k_gamma"] = uniform(0.5, 1.5, d)
    elif c["kind"] == "tree":
        s["q"] = normal(tokens, c["heads"] * d)
        words = (int(new.max()) + 31) // 32
        sees = torch.zeros((tokens, 32 * words), dtype=torch.int64)
        row, at = torch.arange(tokens), place.clone()
        while bool((at >= 0).any()):
            sees[row[at >= 0], at[at >= 0]] = 1
            at = torch.where(at >= 0, parents[(starts[:-1].long()[seq] + at.clamp(min=0))].long(), at)
        bits = (sees.view(tokens, words, 32) << torch.arange(32)).sum(2)
        s["mask"] = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).int().cuda()
    else:  # a path from each tree's first row on
        path, kept = torch.full((tokens,), -1, dtype=torch.int32), torch.zeros(c["seqs"], dtype=torch.int32)
        for i in range(c["seqs"]):
            node, n = 0, 0
            while node < int(new[i]):
                path[int(starts[i]) + n] = node
                node, n = node * c["width"] + 1 + int(torch.randint(0, c["width"], (1,), generator=cpu)), n + 1
            kept[i] = n - 1
        s["path"], s["count"] = path.cuda(), kept.cuda()
    return s


def prepare(case, seed):
    c = dict(case)
    s = dict(case=c, **_inputs(c, seed))
    if own:  # (the same inputs, in buffers of the framework)
        s = dict(case=c, device=_Device(c, s))
    return s


class _Device:
    """The same tensors as the framework's own: what a program that serves with it holds, result buffers among them."""

    def __init__(self, c, s):
        from webdnn_amd import hostops

        self.H = hostops
        self.ctx = hostops.HipContext(0).initialize()
        self.tensors, self.views = {}, {}
        for name in s:
            if name != "case":
                self.take(name, s[name])
        if c["kind"] in ("append", "tree", "keep"):
            self.cache = hostops.KvCache(self.ctx, self["k_pages"], self["k_scales"], self["v_pages"], self["v_scales"])
        if c["kind"] == "rope":
            self.empty("y", [c["tokens"], (c["heads"] + c["kv_heads"]) * c["d"]])
        elif c["kind"] == "tree":
            self.empty("y", list(s["q"].shape))
        elif c["kind"] == "verify":
            self.empty("next", [c["seqs"]], "int32")
            self.empty("count", [c["seqs"]], "int32")
            self.empty("path", list(s["tokens"].shape), "int32")
        torch.cuda.synchronize()

    def empty(self, name, shape, data_type="float32"):
        t = self.tensors[name] = self.ctx.empty_tensor(shape, data_type)
        view = torch.as_tensor(t, device="cuda")
        self.views[name] = view.view(torch.float8_e4m3fn) if data_type == "float8e4m3fn" else view

    def take(self, name, x):
        kinds = {torch.float32: "float32", torch.int32: "int32", torch.float8_e4m3fn: "float8e4m3fn"}
        self.empty(name, list(x.shape), kinds[x.dtype])
        self.views[name].view(torch.uint8).copy_(x.contiguous().view(torch.uint8))

    def __getitem__(self, name):
        return self.tensors.get(name)

    def __del__(self):
        try:
            torch.cuda.synchronize()
            for t in self.tensors.values():
                t.dispose()
        except Exception:  # (the interpreter may be on its way out)
            pass


# ---- a pass --------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    return _own_pass(c, s["device"]) if own else {"rope": _rope, "append": _append, "tree": _attend, "verify": _verify, "keep": _keep}[c["kind"]](c, s)


def _own_pass(c, d):
    H, ctx, v = d.H, d.ctx, d.views
    if c["kind"] == "rope":
        H.rotary_embedding(ctx, d["x"], d["cos"], d["sin"], d["positions"], c["heads"], c["d"], k_heads=c["kv_heads"], q_scale=d["q_gamma"],
                           k_scale=d["k_gamma"], interleaved=c["interleaved"], epsilon=EPS, out=d["y"])
        return v["y"]
    if c["kind"] == "append":
        H.cache_append_rotary(ctx, d.cache, d["kv"], d["kv"], d["table"], d["lens"], d["starts"], d["cos"], d["sin"], d["positions"],
                              k_scale=d["k_gamma"], interleaved=c["interleaved"], epsilon=EPS, v_column=c["kv_heads"] * c["d"])
        return [v["k_pages"], v["k_scales"], v["v_pages"], v["v_scales"]]
    if c["kind"] == "tree":
        H.cache_attention_tree(ctx, d.cache, d["q"], c["heads"], c["d"] ** -0.5, d["table"], d["lens"], d["starts"], d["mask"], out=d["y"])
        return v["y"]
    if c["kind"] == "verify":
        H.verify_drafts(ctx, d["p"], d["tokens"], d["parents"], d["uniform"], d["starts"], draft=d["draft"], out=(d["next"], d["count"], d["path"]))
        return [v["next"], v["count"], v["path"]]
    H.cache_keep(ctx, d.cache, d["table"], d["lens"], d["starts"], d["path"], d["count"])
    return [v["k_pages"], v["k_scales"], v["v_pages"], v["v_scales"]]


def _rotated(c, x, gamma, cos, sin):
    """x [tokens, heads, d], normed for each head if gamma is there, its first `rotary` elements turned by angles [tokens, rotary / 2]."""
    if gamma is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma
    turned, rest = x[..., :c["rotary"]], x[..., c["rotary"]:]
    cos, sin = cos[:, None], sin[:, None]
    if c["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    a, b = turned.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _rope(c, s):
    heads, kv, d, at = c["heads"], c["kv_heads"], c["d"], s["positions"].long()
    x = s["x"].view(c["tokens"], heads + 2 * kv, d)
    cos, sin = s["cos"][at], s["sin"][at]
    parts = [_rotated(c, x[:, :heads], s.get("q_gamma"), cos, sin), _rotated(c, x[:, heads:heads + kv], s.get("k_gamma"), cos, sin)]
    return torch.cat(parts, 1).reshape(c["tokens"], (heads + kv) * d)


def _rows(s, tokens):
    """For each row of the call: its sequence and its position there."""
    row = torch.arange(tokens, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"], row, right=True) - 1
    return seq, (s["lens"] - s["starts"][1:])[seq] + row


def _append(c, s):
    tokens, kv, d = s["kv"].shape[0], c["kv_heads"], c["d"]
    pages = s["k_pages"].shape[0]
    angle = s["positions"].long()
    keys = _rotated(c, s["kv"][:, :kv * d].reshape(tokens, kv, d), s.get("k_gamma"), s["cos"][angle], s["sin"][angle])
    values = s["kv"][:, kv * d:].reshape(tokens, kv, d)
    seq, at = _rows(s, tokens)
    page, slot = s["table"][seq, at // PAGE].long(), (at % PAGE).long()
    first = torch.full((pages,), PAGE, dtype=torch.int64, device="cuda").scatter_reduce(0, page, slot, "amin")
    touched, behind = (first < PAGE)[:, None], (first > 0)[:, None]
    # which pages, in a list with repeats: a page of a sequence's first, second, ... touched one
    most = (c["new"] + c["spread"] + PAGE - 2) // PAGE + 1
    new = s["starts"][1:] - s["starts"][:-1]
    begin, end = (s["lens"] - new) // PAGE, (s["lens"] - 1) // PAGE
    which = torch.minimum(begin[:, None] + torch.arange(most, device="cuda", dtype=torch.int32), end[:, None])
    listed_pages = torch.gather(s["table"].long(), 1, which.long()).reshape(-1)
    kept = (torch.arange(PAGE, device="cuda") < first[listed_pages, None])

    def into(name, x, transposed):
        need = torch.zeros((pages, kv), device="cuda").scatter_reduce(0, page[:, None].expand(tokens, kv), _finite_amax(x, 2), "amax")
        need = _power_of_two_scale(need)
        old = s[name + "_scales"]
        scale = torch.where(touched, torch.where(behind, torch.maximum(old, need), need), old)
        store, before = s[name + "_pages"], s[name + "_pages"][listed_pages]
        again = _to_e4m3(before.float() * (old / scale)[listed_pages][:, :, None, None])
        keep = kept[:, None, None, :] if transposed else kept[:, None, :, None]
        # (bytes: torch scatters no e4m3)
        store.view(torch.uint8)[listed_pages] = torch.where(keep, again.view(torch.uint8), before.view(torch.uint8))
        q = _to_e4m3(x / scale[page][:, :, None]).view(torch.uint8)
        head = torch.arange(kv, device="cuda")[None, :]
        if transposed:
            store.view(torch.uint8)[page[:, None], head, :, slot[:, None]] = q
        else:
            store.view(torch.uint8)[page[:, None], head, slot[:, None], :] = q
        old.copy_(scale)
        return [store, old]

    return into("k", keys, False) + into("v", values, True)


def _attend(c, s):
    tokens, heads, kv, d = s["q"].shape[0], c["heads"], c["kv_heads"], c["d"]
    seqs, width = s["table"].shape
    group, keys = heads // kv, width * PAGE
    seq, at = _rows(s, tokens)
    most = c["new"] + c["spread"]
    place = torch.arange(tokens, device="cuda") - s["starts"][seq]
    table = s["table"].long()
    k = s["k_pages"][table].float() * s["k_scales"][table][..., None, None]
    v = s["v_pages"][table].float() * s["v_scales"][table][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(seqs, kv, keys, d)
    v = v.permute(0, 2, 1, 4, 3).reshape(seqs, kv, keys, d)
    v = torch.where((torch.arange(keys, device="cuda") < s["lens"][:, None])[:, None, :, None], v, 0.0)
    q = torch.zeros((seqs, most, kv, group, d), device="cuda")
    q[seq, place] = s["q"].view(tokens, kv, group, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, d)
    # a row sees what lies before the call's rows, and those of its sequence that its mask names
    past = (s["lens"] - s["starts"][1:] + s["starts"][:-1])[:, None]
    own_rows = torch.zeros((seqs, most, 32 * s["mask"].shape[1]), dtype=torch.bool, device="cuda")
    own_rows[seq, place] = ((s["mask"][:, :, None] >> torch.arange(32, device="cuda")) & 1).bool().flatten(1)
    column = torch.arange(keys, device="cuda") - past
    bit = column.clamp(min=0, max=own_rows.shape[2] - 1)[:, None].expand(seqs, most, keys)
    seen = torch.where((column < 0)[:, None], True, torch.gather(own_rows, 2, bit) & (column < own_rows.shape[2])[:, None])
    seen = seen & (torch.arange(keys, device="cuda") < s["lens"][:, None])[:, None]
    scores = (q @ k.transpose(2, 3)).view(seqs, kv, group, most, keys) * (d ** -0.5)
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    y = (p.view(seqs, kv, group * most, keys) @ v).view(seqs, kv, group, most, d)
    y = torch.where(total > 0, y / total, 0.0).permute(0, 3, 1, 2, 4)
    return y[seq, place].reshape(tokens, heads * d)


def _verify(c, s):
    """All drafts' tests at once (a test goes by its parent's row and by how many siblings come before it), then the paths that passed ones make."""
    p, parents, starts, u = s["p"], s["parents"].long(), s["starts"].long(), s["uniform"].double()
    tokens, vocab = p.shape
    row = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    root = parents < 0
    above = torch.where(root, row, starts[seq] + parents)
    token = s["tokens"].long()
    sibling = (above[:, None] == above) & ~root[:, None] & ~root
    earlier = sibling & (row < row[:, None])
    rank = earlier.sum(1)
    px = p[above, token].double()
    if c["drawn"]:
        draft = s["draft"]
        t, mass = torch.zeros(tokens, dtype=torch.float64, device="cuda"), torch.ones(tokens, dtype=torch.float64, device="cuda")
        ts, masses = [t], [mass]
        for _ in range(c["width"]):
            t = t + mass
            mass = (p.double() - t[:, None] * draft.double()).clamp(min=0).sum(1)
            ts.append(t)
            masses.append(mass)
        ts, masses = torch.stack(ts), torch.stack(masses)
        qx = draft[above, token].double()
        passed = u * masses[rank, above] * qx < (px - ts[rank, above] * qx).clamp(min=0)
    else:
        px = torch.where((earlier & (token[:, None] == token)).any(1), 0.0, px)
        passed = u * (1 - earlier.double() @ px) < px
    passed = passed & ~root
    best = torch.full((tokens,), tokens, device="cuda").scatter_reduce(0, above, torch.where(passed, row, tokens), "amin")
    lost = ~root & (best[above] != row)
    jump = above
    for _ in range((c["new"] + c["spread"]).bit_length()):
        lost, jump = lost | lost[jump], jump[jump]
    place = torch.cumsum(~lost, 0) - 1
    place = place - place[starts[:-1]][seq]
    path = torch.full((tokens + 1,), -1, dtype=torch.int64, device="cuda")
    path[torch.where(lost, tokens, starts[seq] + place)] = row - starts[seq]
    last = torch.zeros(c["seqs"], dtype=torch.int64, device="cuda").scatter_reduce(0, seq, torch.where(lost, 0, row), "amax")
    count = torch.zeros(c["seqs"], dtype=torch.int64, device="cuda").scatter_add(0, seq, (~lost).long()) - 1
    pl = p[last].double()
    if c["drawn"]:
        children = torch.zeros(tokens, dtype=torch.int64, device="cuda").scatter_add(0, above, (~root).long())[last]
        left = (pl - ts[children, last][:, None] * s["draft"][last].double()).clamp(min=0)
    else:
        mine = (last[seq] == above) & ~root
        out = torch.zeros((c["seqs"], vocab + 1), dtype=torch.bool, device="cuda")
        out[seq, torch.where(mine, token, vocab)] = True
        left = torch.where(out[:, :vocab], 0.0, pl)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, pl)
    upto = torch.cumsum(left, 1)
    token = torch.searchsorted(upto, u[starts[:-1], None] * upto[:, -1:], right=True)[:, 0]
    return [token.int(), count.int(), path[:tokens].int()]


def _keep(c, s):
    """A path's tokens go behind each other, from the first row's slot on; a page that they outgrow takes a larger scale."""
    tokens, kv, d = s["path"].shape[0], c["kv_heads"], c["d"]
    pages = s["k_pages"].shape[0]
    starts, path = s["starts"], s["path"]
    row = torch.arange(tokens, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(starts, row, right=True) - 1
    new = starts[1:] - starts[:-1]
    past = s["lens"] - new
    kept = row - starts[seq] <= s["count"][seq]
    to = past[seq] + row - starts[seq]
    at = past[seq] + torch.where(kept, path, row - starts[seq])
    page, slot = s["table"][seq, to // PAGE].long(), (to % PAGE).long()
    page_from, slot_from = s["table"][seq, at // PAGE].long(), (at % PAGE).long()
    # the pages that kept tokens go to, and which of their slots hold earlier tokens
    most = (c["new"] + c["spread"] + PAGE - 2) // PAGE + 1
    which = torch.minimum((past // PAGE)[:, None] + torch.arange(most, device="cuda", dtype=torch.int32), ((past + s["count"]) // PAGE)[:, None])
    listed_pages = torch.gather(s["table"].long(), 1, which.long()).reshape(-1)
    earlier = torch.arange(PAGE, device="cuda") < (past[:, None] - which * PAGE).reshape(-1, 1)
    head = torch.arange(kv, device="cuda")[None, :]

    def move(name, transposed):
        store, old = s[name + "_pages"], s[name + "_scales"]
        if transposed:
            x = store[page_from[:, None], head, :, slot_from[:, None]].float()
        else:
            x = store[page_from[:, None], head, slot_from[:, None], :].float()
        x = x * old[page_from][:, :, None]
        need = _power_of_two_scale(torch.where(kept[:, None], _finite_amax(x, 2), 0.0))
        scale = old.scatter_reduce(0, torch.where(kept, page, listed_pages[0])[:, None].expand(tokens, kv), need, "amax")
        before = store[listed_pages]
        again = _to_e4m3(before.float() * (old / scale)[listed_pages][:, :, None, None])
        mask = earlier[:, None, None, :] if transposed else earlier[:, None, :, None]
        store.view(torch.uint8)[listed_pages] = torch.where(mask, again.view(torch.uint8), before.view(torch.uint8))
        # (rows that are not kept write what is there)
        q = _to_e4m3(x / scale[page][:, :, None]).view(torch.uint8)
        if transposed:
            there = store.view(torch.uint8)[page[:, None], head, :, slot[:, None]]
            store.view(torch.uint8)[page[:, None], head, :, slot[:, None]] = torch.where(kept[:, None, None], q, there)
        else:
            there = store.view(torch.uint8)[page[:, None], head, slot[:, None], :]
            store.view(torch.uint8)[page[:, None], head, slot[:, None], :] = torch.where(kept[:, None, None], q, there)
        old.copy_(scale)
        return [store, old]

    return move("k", False) + move("v", True)


# ---- what a pass cannot do without -----------------------------------------------------------
def _sequences(c):
    """(tokens of the call, tokens that lie before them) of each sequence, as prepare() has them."""
    new, past = _counts(c)
    return list(zip(new.tolist(), past.tolist()))


def work(case):
    c, k = case, case["kind"]
    if k == "rope":
        n = c["tokens"] * (c["heads"] + c["kv_heads"]) * c["d"]
        return {"bytes": 8 * n + 4 * min(c["tokens"], 9000) * c["rotary"] + 4 * c["tokens"], "flops": (3 * n if c["norm"] else 0) + 3 * n * c["rotary"] // c["d"]}
    rows = _sequences(c)
    tokens = sum(n for n, _ in rows)
    if k == "verify":
        # single elements decide which drafts stay; then a row of each sequence, and where drafts were drawn the row they were drawn from
        return {"bytes": c["seqs"] * c["vocab"] * (8 if c["drawn"] else 4) + 20 * tokens + 12 * c["seqs"], "flops": c["seqs"] * c["vocab"] * 2}
    width = c["kv_heads"] * c["d"]
    if k == "append":
        # the new keys and values in 32 bits, and in 8; a scale for each page and head; angles
        return {"bytes": 10 * tokens * width + 16 * sum(-(-n // PAGE) for n, _ in rows) * c["kv_heads"] + 4 * tokens * c["rotary"],
                "flops": 10 * tokens * width}
    if k == "keep":
        # the path's tokens (about log(n) of them), read and written in 8 bits
        moved = sum(int(math.log(n * (c["width"] - 1) + 1, c["width"])) if c["width"] > 1 else n for n, _ in rows)
        return {"bytes": 4 * moved * width + 16 * len(rows) * c["kv_heads"] + 4 * tokens, "flops": 2 * moved * width}
    pairs = sum(n * p + n * (1 + int(math.log(n, max(2, c["width"])))) for n, p in rows)
    return {"bytes": 2 * sum(n + p for n, p in rows) * width + 8 * tokens * c["heads"] * c["d"], "flops": 4 * pairs * c["heads"] * c["d"]}


# ---- the operators' definitions in 64 bits ---------------------------------------------------
def _nearest_e4m3(x):
    """x in 64 bits to the nearest e4m3 value, ties to even: steps of 2^(e-3) from 2^e on, of 2^-9 below 2^-6."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -60))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _turned_64(c, x, gamma, angles):
    """Element by element: pair j of a head is (x[j], x[j + rotary / 2]), or (x[2j], x[2j + 1])."""
    y = x.double()
    if gamma is not None:
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / c["d"] + EPS) * gamma.double()
    out, half = y.clone(), c["rotary"] // 2
    for j in range(half):
        a, b = (2 * j, 2 * j + 1) if c["interleaved"] else (j, j + half)
        cos, sin = (t[:, None, j].double() for t in angles)
        out[..., a], out[..., b] = y[..., a] * cos - y[..., b] * sin, y[..., b] * cos + y[..., a] * sin
    return out


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    d = c.get("d")
    if c["kind"] == "rope":
        x, heads, kv = s["x"].view(c["tokens"], -1, d), c["heads"], c["kv_heads"]
        angles = [s[n][s["positions"].long()] for n in ("cos", "sin")]
        y = [_turned_64(c, x[:, :heads], s.get("q_gamma"), angles), _turned_64(c, x[:, heads:heads + kv], s.get("k_gamma"), angles)]
        return torch.cat(y, 1).view(c["tokens"], (heads + kv) * d)
    starts = s["starts"].tolist()
    if c["kind"] == "verify":
        return _walk(c, s, starts)
    table, lens = (s[n].tolist() for n in ("table", "lens"))
    kv = c["kv_heads"]

    def scale_of(x):
        return torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)).clamp(min=2.0 ** -140) / E4M3_MAX)).clamp(min=-100))

    if c["kind"] == "append":
        out = []
        keys = _turned_64(c, s["kv"][:, :kv * d].reshape(-1, kv, d), s.get("k_gamma"), [s[n][s["positions"].long()] for n in ("cos", "sin")])
        for name, x, turned in (("k", keys, False), ("v", s["kv"][:, kv * d:].reshape(-1, kv, d).double(), True)):
            pages, scales = s[name + "_pages"].double(), s[name + "_scales"].double()
            for i, length in enumerate(lens):
                row, position = starts[i], length - (starts[i + 1] - starts[i])
                while position < length:
                    p, slot = table[i][position // PAGE], position % PAGE
                    n = min(PAGE - slot, length - position)
                    new = x[row:row + n].permute(1, 0, 2)
                    scale = torch.maximum(scales[p], scale_of(new)) if slot else scale_of(new)
                    page = pages[p].transpose(1, 2) if turned else pages[p]  # [heads, tokens, d], written through
                    if slot:
                        page[:, :slot] = _nearest_e4m3(page[:, :slot] * (scales[p] / scale)[:, None, None])
                    page[:, slot:slot + n] = _nearest_e4m3(new / scale[:, None, None])
                    scales[p] = scale
                    row, position = row + n, position + n
            out += [pages, scales]
        return out
    if c["kind"] == "keep":
        out = []
        path, count = s["path"].tolist(), s["count"].tolist()
        for name, turned in (("k", False), ("v", True)):
            pages, scales = s[name + "_pages"].double(), s[name + "_scales"].double()
            view = pages.transpose(2, 3) if turned else pages  # [pages, heads, tokens, d], written through
            for i, length in enumerate(lens):
                past = length - (starts[i + 1] - starts[i])
                order = [past + path[starts[i] + j] for j in range(count[i] + 1)]
                held = [view[table[i][a // PAGE], :, a % PAGE] * scales[table[i][a // PAGE]][:, None] for a in order]
                for b in range(past // PAGE, (past + count[i]) // PAGE + 1):
                    p, lo, hi = table[i][b], max(past, b * PAGE), min(past + count[i] + 1, (b + 1) * PAGE)
                    moved = torch.stack(held[lo - past:hi - past], 1)
                    scale = torch.maximum(scales[p], scale_of(moved))
                    if lo % PAGE:
                        view[p, :, :lo % PAGE] = _nearest_e4m3(view[p, :, :lo % PAGE] * (scales[p] / scale)[:, None, None])
                    view[p, :, lo % PAGE:lo % PAGE + hi - lo] = _nearest_e4m3(moved / scale[:, None, None])
                    scales[p] = scale
            out += [pages, scales]
        return out
    group = c["heads"] // kv
    y = torch.zeros((s["q"].shape[0], kv, group, d), dtype=torch.float64, device="cuda")
    q = s["q"].double().view(-1, kv, group, d)
    sees = ((s["mask"].long()[:, :, None] >> torch.arange(32, device="cuda")) & 1).flatten(1) == 0
    for i, length in enumerate(lens):
        n = starts[i + 1] - starts[i]
        p = torch.tensor(table[i][:-(-length // PAGE)], device="cuda")
        k = (s["k_pages"][p].double() * s["k_scales"][p].double()[..., None, None]).permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :length]
        v = (s["v_pages"][p].double() * s["v_scales"][p].double()[..., None, None]).permute(1, 0, 3, 2).reshape(kv, -1, d)[:, :length]
        hidden = torch.cat([torch.zeros((n, length - n), dtype=torch.bool, device="cuda"), sees[starts[i]:starts[i + 1], :n]], 1)
        for h in range(kv):
            for e in range(group):
                t = (q[starts[i]:starts[i + 1], h, e] @ k[h].t()) / math.sqrt(d)
                y[starts[i]:starts[i + 1], h, e] = torch.softmax(t.masked_fill(hidden, -math.inf), 1) @ v[h]
    return y.view(-1, c["heads"] * d)


def _walk(c, s, starts):
    """One sequence after the other, one draft after the other."""
    parents, tokens, u = s["parents"].tolist(), s["tokens"].tolist(), s["uniform"].tolist()
    drawn_tokens, counts, path = [], [], [-1] * starts[-1]
    for i in range(c["seqs"]):
        lo, n = starts[i], starts[i + 1] - starts[i]
        node, taken = 0, [0]
        while True:
            left, mass = s["p"][lo + node].double(), 1.0
            follow = None
            for child in [j for j in range(n) if parents[lo + j] == node]:
                x = tokens[lo + child]
                likely = float(s["draft"][lo + node, x]) if c["drawn"] else 1.0
                if u[lo + child] * mass * likely < float(left[x]):
                    follow = child
                    break
                if c["drawn"]:
                    left = (left - mass * s["draft"][lo + node].double()).clamp(min=0)
                    mass = float(left.sum())
                else:
                    mass -= float(left[x])
                    left = left.index_fill(0, torch.tensor([x], device="cuda"), 0.0)
            if follow is None:
                break
            node = follow
            taken.append(node)
        if float(left.sum()) <= 0:
            left = s["p"][lo + node].double()
        upto = torch.cumsum(left, 0)
        drawn_tokens.append(int((upto > u[lo] * float(upto[-1])).nonzero()[0]))
        counts.append(len(taken) - 1)
        path[lo:lo + len(taken)] = taken
    return [torch.tensor(t, dtype=torch.int32, device="cuda") for t in (drawn_tokens, counts, path)]
