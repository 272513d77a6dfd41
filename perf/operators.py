"""The 8-bit serving operators as cases that can be timed: root-mean-square norm with an 8-bit output, quantisation to
e4m3 in blocks, the e4m3 product with a scale for each block of 128, appending to a cache held in e4m3, and attention over it.

A pass is one call as a program in a serving loop makes it: operands lie on the device, results go to buffers that the
program keeps.  `own = False` computes the same from elementary torch operations in 32 bits.

Layouts (row-major): activations [rows, cols]; their scales [rows, ceil(cols/128)]; weights [n, k], scales
[ceil(n/128), ceil(k/128)]; cache pages of 64 tokens, keys [pages, heads, 64, d], values [pages, heads, d, 64], scales
[pages, heads]; table [sequences, most pages] of page numbers, lens [sequences] with the tokens of this call counted, and
starts [sequences + 1]: which rows of the call's tokens belong to which sequence (they are the last of its lens tokens).
"""
import math

import torch

own = False

BLOCK, PAGE, E4M3_MAX, LEAST_SCALE = 128, 64, 448.0, 2.0 ** -100


def listed():
    return [
        # a decoder's norm between two products, a few sequences of one token each: latency is all there is
        dict(name="norm_4x4096", kind="norm", rows=4, cols=4096, skip=True, to8=True),
        # the same for a batch of prompts
        dict(name="norm_8192x4096", kind="norm", rows=8192, cols=4096, skip=True, to8=True),
        # what attention or an activation leaves is quantised for the next product
        dict(name="quantize_rows_5000x8192", kind="quantize", rows=5000, cols=8192, block_rows=1),
        # weights at load time, an odd size (vocabulary of the text encoder's size)
        dict(name="quantize_weight_30000x1030", kind="quantize", rows=30000, cols=1030, block_rows=128),
        # one token through a linear layer: the weights are read for a single row
        dict(name="product_1x8192x4096", kind="product", m=1, n=8192, k=4096, bias=False, residual=True),
        # a ragged batch with sizes that are multiples of nothing
        dict(name="product_333x1000x2050", kind="product", m=333, n=1000, k=2050, bias=True, residual=False),
        # a batch of prompts through a wide layer
        dict(name="product_8192x8192x8192", kind="product", m=8192, n=8192, k=8192, bias=False, residual=False),
        # one new token for each of 48 sequences
        dict(name="append_48_tokens", kind="append", seqs=48, new=1, spread=0, past=1000, kv_heads=8, d=128),
        # a batch of prompts of different lengths goes into an empty cache
        dict(name="append_6_prompts", kind="append", seqs=6, new=1500, spread=1400, past=0, kv_heads=8, d=128),
        # one new token for each of 32 sequences of different lengths
        dict(name="attend_32_tokens", kind="attend", seqs=32, new=1, spread=0, past=4500, past_spread=4000, heads=32, kv_heads=8, d=128),
        # one token of a single long conversation: the cache of one sequence has to fill the chip
        dict(name="attend_one_of_100000", kind="attend", seqs=1, new=1, spread=0, past=100000, past_spread=0, heads=16, kv_heads=2, d=128),
        # prompts of different lengths, none of them behind earlier tokens but the second part of one
        dict(name="attend_3_prompts", kind="attend", seqs=3, new=2500, spread=1500, past=500, past_spread=500, heads=16, kv_heads=4, d=128),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "product", "product", "append", "attend", "attend", "attend"])
    if kind == "norm":
        cols = _log_int(rng, 64, 10000)
        return dict(kind=kind, rows=_log_int(rng, 1, 8192 * 4096 // cols), cols=cols, skip=rng.random() < 0.7, to8=rng.random() < 0.7)
    if kind == "quantize":
        cols = _log_int(rng, 64, 16384)
        return dict(kind=kind, rows=_log_int(rng, 1, 5000 * 8192 // cols), cols=cols, block_rows=rng.choice([1, 1, 128]))
    if kind == "product":
        m = 1 if rng.random() < 0.2 else _log_int(rng, 2, 8192)
        return dict(kind=kind, m=m, n=_log_int(rng, 128, 8192), k=_log_int(rng, 128, 8192), bias=rng.random() < 0.5,
                    residual=rng.random() < 0.5)
    d, kv = rng.choice([32, 64, 128, 128]), rng.choice([1, 2, 4, 8])
    if kind == "append":
        if rng.random() < 0.5:
            return dict(kind=kind, seqs=_log_int(rng, 1, 200), new=rng.choice([1, 1, 4]), spread=0, past=_log_int(rng, 1, 2000), kv_heads=kv, d=d)
        seqs = _log_int(rng, 1, 16)
        new = _log_int(rng, 16, 9000 // seqs)
        return dict(kind=kind, seqs=seqs, new=new, spread=new // 2, past=rng.choice([0, 0, 100, 700]), kv_heads=kv, d=d)
    heads = kv * rng.choice([1, 2, 4, 8])
    if rng.random() < 0.6:
        seqs = _log_int(rng, 1, 64)
        past = _log_int(rng, 1, min(100000, 150000 // seqs))
        return dict(kind=kind, seqs=seqs, new=rng.choice([1, 1, 1, 3]), spread=0, past=past, past_spread=past // 2, heads=heads, kv_heads=kv, d=d)
    seqs = _log_int(rng, 1, 8)
    new = _log_int(rng, 20, 2800 if seqs < 4 else 1000)
    past = rng.choice([0, 0, 300, 1500])
    return dict(kind=kind, seqs=seqs, new=new, spread=new // 2, past=past, past_spread=past // 2, heads=min(heads, 16), kv_heads=min(kv, 4) if heads >= 4 else kv, d=d)


# ---- the 8-bit forms, in plain torch -------------------------------------------------------
def _blocks(n):
    return -(-n // BLOCK)


def _finite_amax(x, dims):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dims)


def _to_e4m3(x):
    """Nearest e4m3 value; what is not finite becomes NaN."""
    return torch.where(torch.isfinite(x), x.clamp(-E4M3_MAX, E4M3_MAX), torch.full_like(x, math.nan)).to(torch.float8_e4m3fn)


def _quantize(x, block_rows):
    """[rows, cols] -> e4m3 of the same shape and a scale for each block of block_rows x 128."""
    rows, cols = x.shape
    nr, nc = -(-rows // block_rows), _blocks(cols)
    padded = torch.nn.functional.pad(x, (0, nc * BLOCK - cols, 0, nr * block_rows - rows)).view(nr, block_rows, nc, BLOCK)
    scale = (_finite_amax(padded, (1, 3)) / E4M3_MAX).clamp(min=LEAST_SCALE)
    q = _to_e4m3(padded / scale[:, None, :, None]).view(nr * block_rows, nc * BLOCK)[:rows, :cols]
    return q.contiguous(), scale


def _power_of_two_scale(amax):
    """The least 2^e with amax <= 448 * 2^e, and e >= -100 (448 is 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), torch.clamp(torch.where(m <= 0.875, e - 9, e - 8), min=-100))


# ---- inputs --------------------------------------------------------------------------------
def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    uniform = lambda lo, hi, *shape: torch.rand(shape, generator=g, device="cuda") * (hi - lo) + lo
    if c["kind"] == "norm":
        # a residual stream: a few channels are much larger than the others
        channel = torch.exp(normal(c["cols"]) * 0.5)
        s = dict(x=normal(c["rows"], c["cols"]) * channel, gamma=uniform(0.5, 1.5, c["cols"]))
        if c["skip"]:
            s["skip"] = normal(c["rows"], c["cols"])
        return s
    if c["kind"] == "quantize":
        return dict(x=normal(c["rows"], c["cols"]) * torch.exp(normal(c["cols"]) * 0.5) * 0.02)
    if c["kind"] == "product":
        a, sa = _quantize(normal(c["m"], c["k"]), 1)
        w, sw = _quantize(normal(c["n"], c["k"]) * c["k"] ** -0.5, BLOCK)
        s = dict(a=a, sa=sa, w=w, sw=sw)
        if c["bias"]:
            s["bias"] = normal(c["n"])
        if c["residual"]:
            s["residual"] = normal(c["m"], c["n"])
        return s
    # sequences: how long they are, how many of their tokens are this call's, and on which pages they lie
    cpu = torch.Generator().manual_seed(seed)
    # (which rows and lengths come first is a matter of the case's sizes: passes of other seeds do the same work)
    steps = torch.linspace(-1, 1, c["seqs"]) if c["seqs"] > 1 else torch.zeros(1)
    new = (c["new"] + (steps * c["spread"]).round()).int().clamp(min=1)
    past = (c["past"] + (steps.flip(0) * c.get("past_spread", 0)).round()).int()
    lens = past + new
    count = (lens + PAGE - 1) // PAGE
    pages, most = int(count.sum()) + 3, int(count.max())
    order = torch.randperm(pages, generator=cpu).int()
    first = torch.cumsum(count, 0) - count
    column = torch.arange(most)
    table = torch.where(column < count[:, None], order[(first[:, None] + column).clamp(max=pages - 1)], torch.zeros((), dtype=torch.int32))
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(new, 0)]).int()
    tokens, kv, d = int(starts[-1]), c["kv_heads"], c["d"]
    s = dict(table=table.cuda(), lens=lens.cuda(), starts=starts.cuda())
    keys, values = normal(pages, kv, PAGE, d), normal(pages, kv, d, PAGE)
    for name, x in (("k", keys), ("v", values)):
        scale = _power_of_two_scale(x.abs().amax((2, 3)))
        s[name + "_pages"], s[name + "_scales"] = _to_e4m3(x / scale[:, :, None, None]), scale
    del keys, values, x
    if c["kind"] == "append":
        # now and then a token outgrows what its page held so far
        grown = lambda: normal(tokens, kv * d) * torch.where(uniform(0, 1, tokens, 1) < 0.1, 3.0, 1.0)
        s.update(k=grown(), v=grown())
    else:
        s.update(q=normal(tokens, c["heads"] * d))
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
        if c["kind"] in ("append", "attend"):
            self.cache = hostops.KvCache(self.ctx, self["k_pages"], self["k_scales"], self["v_pages"], self["v_scales"])
        if c["kind"] == "norm":
            shape = [c["rows"], c["cols"]]
            if c["skip"]:
                self.empty("sum", shape)
            if c["to8"]:
                self.empty("q8", shape, "float8e4m3fn")
                self.empty("scales", [c["rows"], _blocks(c["cols"])])
            else:
                self.empty("y", shape)
        elif c["kind"] == "quantize":
            self.empty("q8", [c["rows"], c["cols"]], "float8e4m3fn")
            self.empty("scales", [-(-c["rows"] // c["block_rows"]), _blocks(c["cols"])])
        elif c["kind"] == "product":
            self.empty("y", [c["m"], c["n"]])
        elif c["kind"] == "attend":
            self.empty("y", list(s["q"].shape))
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
    return _own_pass(c, s["device"]) if own else {"norm": _norm, "quantize": _quantize_pass, "product": _product, "append": _append,
                                                  "attend": _attend}[c["kind"]](c, s)


def _own_pass(c, d):
    H, ctx, v = d.H, d.ctx, d.views
    if c["kind"] == "norm":
        if c["to8"]:
            H.rms_normalization_fp8(ctx, d["x"], d["gamma"], d["skip"], 1e-5, out=(d["sum"], d["q8"], d["scales"]))
            return [v["sum"], v["q8"], v["scales"]] if c["skip"] else [v["q8"], v["scales"]]
        H.rms_normalization(ctx, d["x"], d["gamma"], d["skip"], 1e-5, out=(d["sum"], d["y"]))
        return [v["sum"], v["y"]] if c["skip"] else [v["y"]]
    if c["kind"] == "quantize":
        H.quantize_fp8(ctx, d["x"], c["block_rows"], out=(d["q8"], d["scales"]))
        return [v["q8"], v["scales"]]
    if c["kind"] == "product":
        H.matmul_fp8(ctx, d["a"], d["sa"], d["w"], d["sw"], bias=d["bias"], residual=d["residual"], out=d["y"])
        return v["y"]
    if c["kind"] == "append":
        H.cache_append(ctx, d.cache, d["k"], d["v"], d["table"], d["lens"], d["starts"])
        return [v["k_pages"], v["k_scales"], v["v_pages"], v["v_scales"]]
    H.cache_attention(ctx, d.cache, d["q"], c["heads"], c["d"] ** -0.5, d["table"], d["lens"], d["starts"], out=d["y"])
    return v["y"]


def _norm(c, s):
    x = s["x"] + s["skip"] if c["skip"] else s["x"]
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * s["gamma"]
    return ([x] if c["skip"] else []) + (list(_quantize(y, 1)) if c["to8"] else [y])


def _quantize_pass(c, s):
    return list(_quantize(s["x"], c["block_rows"]))


def _product(c, s):
    a = s["a"].float() * s["sa"].repeat_interleave(BLOCK, 1)[:, :c["k"]]
    w = s["w"].float() * s["sw"].repeat_interleave(BLOCK, 0)[:c["n"]].repeat_interleave(BLOCK, 1)[:, :c["k"]]
    y = a @ w.t()
    if c["bias"]:
        y = y + s["bias"]
    return y + s["residual"] if c["residual"] else y


def _rows(s, tokens):
    """For each row of the call: its sequence and its position there."""
    row = torch.arange(tokens, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"], row, right=True) - 1
    return seq, (s["lens"] - s["starts"][1:])[seq] + row


def _append(c, s):
    tokens, kv, d = s["k"].shape[0], c["kv_heads"], c["d"]
    pages = s["k_pages"].shape[0]
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
        x = x.view(tokens, kv, d)
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

    return into("k", s["k"], False) + into("v", s["v"], True)


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
    last = torch.full((seqs, most), -1, dtype=torch.int32, device="cuda")
    last[seq, place] = at.int()
    scores = (q @ k.transpose(2, 3)).view(seqs, kv, group, most, keys) * (d ** -0.5)
    scores = torch.where((torch.arange(keys, device="cuda") <= last[..., None])[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    y = (p.view(seqs, kv, group * most, keys) @ v).view(seqs, kv, group, most, d)
    y = torch.where(total > 0, y / total, 0.0).permute(0, 3, 1, 2, 4)
    return y[seq, place].reshape(tokens, heads * d)


# ---- what a pass cannot do without -----------------------------------------------------------
def _sequences(c):
    """(tokens of the call, tokens that lie before them) of each sequence, as prepare() has them."""
    steps = [2 * i / (c["seqs"] - 1) - 1 for i in range(c["seqs"])] if c["seqs"] > 1 else [0.0]
    return [(max(1, c["new"] + round(x * c["spread"])), c["past"] + round(-x * c.get("past_spread", 0))) for x in steps]


def work(case):
    c, k = case, case["kind"]
    if k == "norm":
        n = c["rows"] * c["cols"]
        return {"bytes": 4 * n + 4 * c["cols"] + (8 * n if c["skip"] else 0) + (n + 4 * c["rows"] * _blocks(c["cols"]) if c["to8"] else 4 * n),
                "flops": 4 * n}
    if k == "quantize":
        n = c["rows"] * c["cols"]
        return {"bytes": 5 * n + 4 * -(-c["rows"] // c["block_rows"]) * _blocks(c["cols"]), "flops": 2 * n}
    if k == "product":
        m, n, kk = c["m"], c["n"], c["k"]
        return {"bytes": m * kk + n * kk + 4 * (m + _blocks(n)) * _blocks(kk) + 4 * m * n * (2 if c["residual"] else 1) + (4 * n if c["bias"] else 0),
                "flops": 2 * m * n * kk}
    rows = _sequences(c)
    width = c["kv_heads"] * c["d"]
    tokens = sum(n for n, _ in rows)
    if k == "append":
        # the new keys and values in 32 bits, and in 8; a scale for each page and head
        return {"bytes": 10 * tokens * width + 16 * sum(-(-n // PAGE) for n, _ in rows) * c["kv_heads"], "flops": 4 * tokens * width}
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in rows)
    return {"bytes": 2 * sum(n + p for n, p in rows) * width + 8 * tokens * c["heads"] * c["d"], "flops": 4 * pairs * c["heads"] * c["d"]}


# ---- the operators' definitions in 64 bits ---------------------------------------------------
def _nearest_e4m3(x):
    """x in 64 bits to the nearest e4m3 value, ties to even: steps of 2^(e-3) from 2^e on, of 2^-9 below 2^-6."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -60))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact(case, seed):
    c, s = case, _inputs(case, seed)

    def blocks(y, block_rows):
        """The quotients that are rounded to e4m3 (each 8-bit value stands for one of them), and the scales."""
        rows, cols = y.shape
        scales = torch.zeros((-(-rows // block_rows), _blocks(cols)), dtype=torch.float64, device="cuda")
        q = torch.empty_like(y)
        for b in range(_blocks(cols)):
            piece = y[:, b * BLOCK:(b + 1) * BLOCK]
            top = piece.abs().amax(1)
            top = torch.nn.functional.pad(top, (0, scales.shape[0] * block_rows - rows)).view(-1, block_rows).amax(1)
            scales[:, b] = (top / E4M3_MAX).clamp(min=LEAST_SCALE)
            q[:, b * BLOCK:(b + 1) * BLOCK] = piece / scales[:, b].repeat_interleave(block_rows)[:rows, None]
        return [q, scales]

    if c["kind"] == "norm":
        x = s["x"].double() + (s["skip"].double() if c["skip"] else 0.0)
        y = x / torch.sqrt((x * x).sum(1, keepdim=True) / c["cols"] + 1e-5) * s["gamma"].double()
        return ([x] if c["skip"] else []) + (blocks(y, 1) if c["to8"] else [y])
    if c["kind"] == "quantize":
        return blocks(s["x"].double(), c["block_rows"])
    if c["kind"] == "product":
        y = torch.zeros((c["m"], c["n"]), dtype=torch.float64, device="cuda")
        for b in range(_blocks(c["k"])):
            cut = slice(b * BLOCK, (b + 1) * BLOCK)
            weight = s["w"][:, cut].double() * s["sw"][:, b].double().repeat_interleave(BLOCK)[:c["n"], None]
            y += (s["a"][:, cut].double() * s["sa"][:, b:b + 1].double()) @ weight.t()
        return y + (s["bias"].double() if c["bias"] else 0.0) + (s["residual"].double() if c["residual"] else 0.0)
    kv, d = c["kv_heads"], c["d"]
    table, lens, starts = (s[n].tolist() for n in ("table", "lens", "starts"))
    if c["kind"] == "append":
        out = []
        for name, turned in (("k", False), ("v", True)):
            pages, scales = s[name + "_pages"].double(), s[name + "_scales"].double()
            x = s[name].double().view(-1, kv, d)
            for i, length in enumerate(lens):
                row, position = starts[i], length - (starts[i + 1] - starts[i])
                while position < length:
                    p, slot = table[i][position // PAGE], position % PAGE
                    n = min(PAGE - slot, length - position)
                    new = x[row:row + n].permute(1, 0, 2)
                    need = torch.exp2(torch.ceil(torch.log2(new.abs().amax((1, 2)).clamp(min=2.0 ** -140) / E4M3_MAX)).clamp(min=-100))
                    scale = torch.maximum(scales[p], need) if slot else need
                    page = pages[p].transpose(1, 2) if turned else pages[p]  # [heads, tokens, d], written through
                    if slot:
                        page[:, :slot] = _nearest_e4m3(page[:, :slot] * (scales[p] / scale)[:, None, None])
                    page[:, slot:slot + n] = _nearest_e4m3(new / scale[:, None, None])
                    scales[p] = scale
                    row, position = row + n, position + n
            out += [pages, scales]
        return out
    group = c["heads"] // kv
    y = torch.zeros((s["q"].shape[0], kv, group, d), dtype=torch.float64, device="cuda")
    q = s["q"].double().view(-1, kv, group, d)
    for i, length in enumerate(lens):
        n = starts[i + 1] - starts[i]
        p = torch.tensor(table[i][:-(-length // PAGE)], device="cuda")
        k = (s["k_pages"][p].double() * s["k_scales"][p].double()[..., None, None]).permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :length]
        v = (s["v_pages"][p].double() * s["v_scales"][p].double()[..., None, None]).permute(1, 0, 3, 2).reshape(kv, -1, d)[:, :length]
        hidden = torch.arange(length, device="cuda") > (length - n + torch.arange(n, device="cuda"))[:, None]
        for h in range(kv):
            for e in range(group):
                t = (q[starts[i]:starts[i + 1], h, e] @ k[h].t()) / math.sqrt(d)
                y[starts[i]:starts[i + 1], h, e] = torch.softmax(t.masked_fill(hidden, -math.inf), 1) @ v[h]
    return y.view(-1, c["heads"] * d)
