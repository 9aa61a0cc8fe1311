"""Measured cases of the operators of a sampling step over the paged cache.

Four operators, each as a user calls it through kestrel_b200.cuda.Context:

  rope     rotary positions on the heads of rows: interleaved pairs or halves,
           the whole head or its first part, frequencies scaled for long contexts
  append   new keys and values written into the pages of their sequences, the
           keys (and the queries beside them) rotated by their positions
  shared   attention of one new token per sequence where groups of sequences
           begin with the same pages (branches of one prompt)
  sample   one token per row of logits by temperature, top-k, top-p and min-p,
           from given uniform numbers

`own` False computes them in plain torch operations in 32 bits (angles and the
sums of probabilities in 64); True calls the library. The cache: k and v
[n_layer, n_pages, n_kv, page, hd], table [n_seq, max_pages] int32 page ids (-1:
none), length [n_seq] int32, refs [n_pages] int32 holders of each page (0: free).

Rotation of pair i of dim / 2 at position p: the angle p * w_i turns (a, b) into
m * (a cos - b sin, a sin + b cos), with w_i = base^(-2 i / dim) / f_i, and then
  linear  w_i / s
  yarn    w_i (r_i / s + 1 - r_i); r_i rises from 0 to 1 between the pairs that
          turn `high` times and `low` times in the original context L:
          c(x) = dim ln(L / (2 pi x)) / (2 ln base), from floor(c(high)) >= 0 to
          ceil(c(low)) <= dim - 1; m = 1 + 0.1 ln s
  bands   wavelengths below L / high stay, above L / low are w_i / s, between
          them z w_i + (1 - z) w_i / s with z = (L w_i / 2 pi - low) / (high - low)

Sampling: w_j = exp((l_j - max l) / T). Of equal logits the lower index comes
first. Top-k keeps the k first; top-p the shortest run of the first of these
whose sum reaches p of all of theirs; min-p those of w_j >= min_p. The token is
the first in the order of the indices at which the running sum of what is kept
exceeds u times all of it. T = 0: the first maximum.
"""
import itertools
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# (query heads, key-value heads, head size) of this package's model
# configurations, then generic ones: no sharing, a group of seven, head sizes
# that are no power of two.
HEADS = [(8, 2, 64), (32, 4, 128), (32, 8, 128), (16, 16, 64), (28, 4, 128), (16, 4, 80), (24, 8, 96)]
TYPES = [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]  # (rows, cache)
VOCABS = [4096, 32000, 50257, 100277, 151936, 201088]


def listed():
    return [
        # The queries and keys of one token of the smallest configuration.
        _rope("rope one row", 1, 10, 64, 64, "f32", "interleaved", "none", 4096),
        # Queries and keys of a long prompt's rows, far positions of a stretched
        # context.
        _rope("rope prompt rows", 8192, 36, 128, 128, "bf16", "half", "yarn", 131072),
        # One chat's next token, where latency counts.
        _append("append one row", 1, 97, 97, 1, (8, 2, 64), 16, 0, 64, "interleaved", "none"),
        # A serving batch's decode step.
        _append("append decode 96", 96, 700, 4096, 1, (32, 8, 128), 32, 2, 128, "half", "bands"),
        # The runtime's 256-token chunks of several prompts in one call, at odd
        # lengths; half of each head turns.
        _append("append chunks of 256", 24, 200, 4000, 256, (32, 4, 128), 64, 0, 64, "half", "linear"),
        # Four samples of one short prompt of the smallest configuration.
        _shared("shared four short", 1, 4, 300, 1, 40, (8, 2, 64), 16, 0),
        # Parallel samples of one prompt, well on their way.
        _shared("shared samples of one prompt", 1, 32, 4001, 1, 600, (32, 4, 128), 64, 0),
        # Four system prompts, a batch of chats under each.
        _shared("shared four prompts", 4, 32, 6000, 100, 2000, (32, 8, 128), 32, 2),
        # Many questions about one long document.
        _shared("shared long document", 1, 64, 32768, 1, 800, (32, 4, 128), 64, 1),
        # One token of the smallest configuration.
        _sample("sample one row", 1, 4096, "f32", "usual"),
        # A serving batch, every request with its own settings.
        _sample("sample batch 32", 32, 151936, "f32", "mixed"),
        # A large batch of parallel samples.
        _sample("sample batch 256", 256, 151936, "f32", "top_p"),
    ]


def _rope(name, rows, heads, hd, dim, t, layout, scaling, reach):
    return {"name": name, "op": "rope", "rows": rows, "heads": heads, "hd": hd, "dim": dim, "t": t, "layout": layout,
            "scaling": scaling, "reach": reach}


def _append(name, n, lo, hi, rows, heads, page, types, dim, layout, scaling):
    return {"name": name, "op": "append", "n": n, "len_lo": lo, "len_hi": hi, "rows": rows, "n_head": heads[0],
            "n_kv": heads[1], "hd": heads[2], "page": page, "t_q": TYPES[types][0], "t_kv": TYPES[types][1],
            "dim": dim, "layout": layout, "scaling": scaling}


def _shared(name, groups, each, prefix, lo, hi, heads, page, types):
    return {"name": name, "op": "shared", "groups": groups, "each": each, "prefix": prefix, "own_lo": lo, "own_hi": hi,
            "n_head": heads[0], "n_kv": heads[1], "hd": heads[2], "page": page, "t_q": TYPES[types][0],
            "t_kv": TYPES[types][1]}


def _sample(name, n, vocab, t, mode):
    return {"name": name, "op": "sample", "n": n, "vocab": vocab, "t": t, "mode": mode}


def _between(rng, lo, hi):
    """A whole number of lo .. hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["rope", "append", "shared", "shared", "sample", "sample"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        heads, page, types = rng.choice(HEADS), rng.choice([16, 32, 64, 128]), rng.randrange(3)
        hd = heads[2]
        dim = rng.choice([hd, hd, hd // 2, hd // 4 * 2 + 4])
        turn = rng.choice(["interleaved", "half"]), rng.choice(["none", "linear", "yarn", "bands", "factors"])
        fits = True
        if op == "rope":
            c = _rope("", _between(rng, 1, 16384), rng.choice([heads[0], sum(heads[:2])]), hd, dim,
                      rng.choice(["f32", "f16", "bf16"]), *turn, _between(rng, 100, 1 << 20))
        elif op == "append":
            hi, n = _between(rng, 1, 16384), _between(rng, 1, 256)
            c = _append("", n, max(1, int(hi * rng.uniform(0.1, 1.0))), hi, _between(rng, 1, min(hi, 512)), heads,
                        page, types, dim, *turn)
            fits = n * hi * heads[1] * hd <= 4e8
        elif op == "shared":
            prefix, hi = _between(rng, 1, 65536), _between(rng, 1, 4000)
            groups, each = _between(rng, 1, 24), _between(rng, 1, 200)
            c = _shared("", groups, each, prefix, max(1, int(hi * rng.uniform(0.0, 1.0))), hi, heads, page, types)
            fits = groups * each * (prefix + hi) * heads[1] * hd <= 1.2e9
        else:
            c = _sample("", _between(rng, 1, 256), rng.choice(VOCABS + [_between(rng, 2, 201088)]),
                        rng.choice(["f32", "f32", "f16", "bf16"]), rng.choice(["usual", "mixed", "top_p", "all"]))
        if fits and _cost(c) <= most:
            del c["name"]
            return c


def _cost(c):
    w = work(c)
    return w["bytes"] + w["flops"] / 200


def _lengths(c):
    """Positions held by each sequence: the case's, whatever the seed."""
    if c["op"] == "append":
        r = random.Random("%d %d %d" % (c["n"], c["len_lo"], c["len_hi"]))
        ls = [r.randint(c["len_lo"], c["len_hi"]) for _ in range(c["n"])]
        ls[0] = c["len_hi"]
        return ls
    r = random.Random("%d %d %d" % (c["groups"], c["each"], c["prefix"]))
    return [c["prefix"] + r.randint(c["own_lo"], c["own_hi"]) for _ in range(c["groups"] * c["each"])]


def _rows(c):
    """New rows of each sequence of an append (its last positions)."""
    return [min(n, c["rows"]) for n in _lengths(c)]


def work(c):
    if c["op"] == "rope":
        n = c["rows"] * c["heads"]
        return {"bytes": 2 * n * c["hd"] * DTYPES[c["t"]].itemsize + 4 * c["rows"], "flops": 3 * n * c["dim"]}
    if c["op"] == "append":
        rows, el = sum(_rows(c)), DTYPES[c["t_q"]].itemsize
        per = c["hd"] * (2 * c["n_head"] * el + 2 * c["n_kv"] * (el + 2))
        return {"bytes": rows * per + 12 * c["n"], "flops": 3 * rows * (c["n_head"] + c["n_kv"]) * c["dim"]}
    if c["op"] == "shared":
        ls, page = _lengths(c), c["page"]
        both = c["prefix"] // page * page  # the positions whose pages a group has in common
        keys = c["groups"] * both + sum(n - both for n in ls)
        io = len(ls) * c["n_head"] * c["hd"] * DTYPES[c["t_q"]].itemsize * 2
        return {"bytes": keys * c["n_kv"] * c["hd"] * 4 + io + sum(-(-n // page) for n in ls) * 4,
                "flops": 4 * sum(ls) * c["n_head"] * c["hd"]}
    return {"bytes": c["n"] * c["vocab"] * DTYPES[c["t"]].itemsize + 24 * c["n"], "flops": 4 * c["n"] * c["vocab"]}


# ---- rotation --------------------------------------------------------------------
BASE, ORIGINAL, FACTOR = 1e6, 8192, 8.0
LOW_HIGH = {"yarn": (1.0, 32.0), "bands": (1.0, 4.0)}


def _factors(dim):
    """Per-pair divisors, as files of stretched models carry them."""
    return [1.0 + 7.0 * (i / max(1, dim // 2 - 1)) ** 2 for i in range(dim // 2)]


def _frequencies(c):
    """(w, m) of a case, w [dim / 2] in 64 bits."""
    dim, scaling = c["dim"], c["scaling"]
    w = BASE ** (-2.0 * torch.arange(dim // 2, device="cuda", dtype=torch.float64) / dim)
    if scaling == "factors":
        return w / torch.tensor(_factors(dim), device="cuda").double(), 1.0
    if scaling == "linear":
        return w / FACTOR, 1.0
    if scaling == "yarn":
        low, high = LOW_HIGH["yarn"]
        at = lambda x: dim * math.log(ORIGINAL / (2 * math.pi * x)) / (2 * math.log(BASE))
        a, b = max(0, math.floor(at(high))), min(dim - 1, math.ceil(at(low)))
        r = ((torch.arange(dim // 2, device="cuda", dtype=torch.float64) - a) / max(0.001, b - a)).clamp(0, 1)
        return w * (r / FACTOR + 1 - r), 1 + 0.1 * math.log(FACTOR)
    if scaling == "bands":
        low, high = LOW_HIGH["bands"]
        z = ((ORIGINAL * w / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return z * w + (1 - z) * w / FACTOR, 1.0
    return w, 1.0


def _turn(c, x, positions):
    """x [rows, heads, hd] in 32 bits, turned; cos and sin come from 64 bits."""
    w, m = _frequencies(c)
    angle = positions.double()[:, None] * w
    cos, sin = ((m * f(angle)).float()[:, None] for f in (torch.cos, torch.sin))
    dim, out = c["dim"], x.clone()
    if c["layout"] == "half":
        first, second = slice(0, dim // 2), slice(dim // 2, dim)
    else:
        first, second = slice(0, dim, 2), slice(1, dim, 2)
    a, b = x[..., first], x[..., second]
    out[..., first] = a * cos - b * sin
    out[..., second] = a * sin + b * cos
    return out


# ---- states ----------------------------------------------------------------------
_context = None
_ids = itertools.count()


def _handle(s):
    """The library's handles of a state, as a user's program keeps them."""
    global _context
    from kestrel_b200.cuda import Context
    if _context is None:
        _context = Context(torch.cuda.current_device())
        _context.set_stream(torch.cuda.current_stream().cuda_stream)
    c = s["case"]
    s["ctx"], s["id"] = _context, next(_ids)
    if "k" in s:
        _context.kv_cache(s["id"], s["k"], s["v"], s["table"], s["length"], s["refs"])
    if "dim" in c:
        scaling = c["scaling"]
        low, high = LOW_HIGH.get(scaling, (0.0, 0.0))
        _context.rope(s["id"], c["dim"], layout=c["layout"], base=BASE,
                      scaling="none" if scaling == "factors" else scaling, factor=FACTOR, original=ORIGINAL, low=low,
                      high=high, freq_factors=_factors(c["dim"]) if scaling == "factors" else None)


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    s = {"case": c}
    if c["op"] == "rope":
        # Queries and keys lie side by side in a row, as a fused projection
        # leaves them, the values behind them.
        t = DTYPES[c["t"]]
        s["x"] = torch.randn((c["rows"], c["heads"] + 2, c["hd"]), generator=g, device="cuda").to(t)[:, :c["heads"]]
        s["positions"] = torch.randint(c["reach"], (c["rows"],), generator=cpu, dtype=torch.int32).cuda()
        s["out"] = torch.empty((c["rows"], c["heads"], c["hd"]), device="cuda", dtype=t)
    elif c["op"] == "append":
        _prepare_cache(c, s, _lengths(c), None, g, cpu)
        rows = _rows(c)
        start = torch.tensor([0] + list(itertools.accumulate(rows)), dtype=torch.int32)
        s["row_start"] = start.cuda() if c["rows"] > 1 else None
        s["seq_of"] = torch.arange(c["n"]).repeat_interleave(torch.tensor(rows)).cuda()
        s["positions"] = torch.cat([torch.arange(n - r, n) for n, r in zip(_lengths(c), rows)]).cuda()
        nq, nkv = c["n_head"], c["n_kv"]
        fused = torch.randn((int(start[-1]), nq + 2 * nkv, c["hd"]), generator=g, device="cuda").to(DTYPES[c["t_q"]])
        s["q"], s["k_new"], s["v_new"] = fused.split([nq, nkv, nkv], 1)
        s["q_out"] = torch.empty(s["q"].shape, device="cuda", dtype=fused.dtype)
    elif c["op"] == "shared":
        _prepare_cache(c, s, _lengths(c), c["each"], g, cpu)
        n = c["groups"] * c["each"]
        s["group_start"] = torch.arange(0, n + 1, c["each"], dtype=torch.int32, device="cuda")
        # Queries as a normalised projection gives them: scores of a few units,
        # so that some keys stand out.
        q = 1.5 * torch.randn((n, c["n_head"], c["hd"]), generator=g, device="cuda")
        s["q"] = q.to(DTYPES[c["t_q"]])
        s["out"] = torch.empty_like(s["q"])
    else:
        _prepare_logits(c, s, g, cpu)
    if own:
        _handle(s)
    return s


def _prepare_cache(c, s, lens, each, g, cpu):
    """Pools and tables. With `each`, that many sequences in turn have the full
    pages of their first c["prefix"] positions in common."""
    page, n = c["page"], len(lens)
    held = [-(-x // page) for x in lens]
    both = c["prefix"] // page if each else 0
    groups = n // each if each else 0
    n_pages = groups * both + sum(h - both for h in held) + 3
    order = torch.randperm(n_pages, generator=cpu, dtype=torch.int32)
    table = torch.full((n, max(held)), -1, dtype=torch.int32)
    refs = torch.zeros(n_pages, dtype=torch.int32)
    at = 0
    for i in range(n):
        if both and i % each == 0:
            shared, at = order[at:at + both], at + both
        if both:
            table[i, :both] = shared
        table[i, both:held[i]] = order[at:at + held[i] - both]
        at += held[i] - both
        refs[table[i, :held[i]].long()] += 1
    t = DTYPES[c["t_kv"]]
    shape = (1, n_pages, c["n_kv"], page, c["hd"])
    s.update(table=table.cuda(), length=torch.tensor(lens, dtype=torch.int32, device="cuda"), refs=refs.cuda(),
             k=torch.randn(shape, generator=g, device="cuda", dtype=t),
             v=torch.randn(shape, generator=g, device="cuda", dtype=t))


def _prepare_logits(c, s, g, cpu):
    """Logits of a language model's size and shape: most tokens within a few
    units, some tens that stand out by more, row by row to another degree."""
    n, v = c["n"], c["vocab"]
    x = 2.2 * torch.randn((n, v), generator=g, device="cuda")
    lead = min(v, 40)
    who = torch.randint(v, (n, lead), generator=g, device="cuda")
    by = 4 + 8 * torch.rand((n, 1), generator=g, device="cuda")
    lift = by * torch.rand((n, lead), generator=g, device="cuda")
    s["logits"] = x.scatter_add_(1, who, lift).to(DTYPES[c["t"]])
    s["u"] = torch.rand(n, generator=g, device="cuda")
    pick = lambda values: torch.tensor(values)[torch.randint(len(values), (n,), generator=cpu)]
    mode = c["mode"]
    if mode == "usual":
        kind = (pick([0.8]), pick([40]), pick([0.95]), pick([0.05]))
    elif mode == "top_p":
        kind = (pick([0.7, 1.0]), pick([0]), pick([0.9, 0.95]), pick([0.0]))
    elif mode == "all":
        kind = (pick([0.6, 1.0, 1.3]), pick([0]), pick([1.0]), pick([0.0]))
    else:
        kind = (pick([0.0, 0.5, 0.8, 1.0, 1.2]), pick([0, 1, 20, 50, 200, 1000]), pick([0.5, 0.9, 0.95, 0.99, 1.0]),
                pick([0.0, 0.0, 0.02, 0.1]))
    for name, x, t in zip(("temperature", "top_k", "top_p", "min_p"), kind,
                          (torch.float32, torch.int32, torch.float32, torch.float32)):
        s[name] = x.to(t).cuda()
    s["tokens"] = torch.empty(n, dtype=torch.int32, device="cuda")
    s["probs"] = torch.empty(n, device="cuda")


# ---- one pass ----------------------------------------------------------------------
def run(s):
    return {"rope": _run_rope, "append": _run_append, "shared": _run_shared, "sample": _run_sample}[s["case"]["op"]](s)


def _run_rope(s):
    if own:
        s["ctx"].rope_dev(s["id"], s["x"], s["positions"], s["out"])
        return s["out"]
    return _turn(s["case"], s["x"].float(), s["positions"]).to(s["x"].dtype)


def _run_append(s):
    if own:
        s["ctx"].kv_append_dev(s["id"], 0, s["id"], s["k_new"], s["v_new"], q=s["q"], q_out=s["q_out"],
                               row_start=s["row_start"])
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    c, pos = s["case"], s["positions"]
    page = c["page"]
    to = s["table"][s["seq_of"], pos // page].long()
    s["k"][0][to, :, pos % page] = _turn(c, s["k_new"].float(), pos).to(s["k"].dtype)
    s["v"][0][to, :, pos % page] = s["v_new"].to(s["v"].dtype)
    return {"q": _turn(c, s["q"].float(), pos).to(s["q"].dtype), "k": s["k"], "v": s["v"]}


def _run_shared(s):
    c = s["case"]
    scale = c["hd"] ** -0.5
    if own:
        s["ctx"].attn_shared_dev(s["id"], 0, s["q"], s["group_start"], s["out"], scale=scale)
        return s["out"]
    nkv, hd, group = c["n_kv"], c["hd"], c["n_head"] // c["n_kv"]
    n = s["q"].shape[0]
    ids = s["table"].clamp(min=0).long()
    k, v = (x[0][ids].transpose(1, 2).reshape(n, nkv, -1, hd).float() for x in (s["k"], s["v"]))
    score = (s["q"].float().view(n, nkv, group, hd) @ k.transpose(2, 3)).mul_(scale)
    hidden = torch.arange(k.shape[2], device="cuda") >= s["length"][:, None]
    score = score.masked_fill_(hidden[:, None, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    return ((p @ v) / p.sum(-1, keepdim=True)).reshape(n, c["n_head"], hd).to(s["q"].dtype)


def _run_sample(s):
    if own:
        s["ctx"].sample_dev(s["logits"], s["u"], s["tokens"], probs=s["probs"], temperature=s["temperature"],
                            top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return {"tokens": s["tokens"], "probs": s["probs"]}
    logits = s["logits"].double()
    vocab = logits.shape[1]
    t = s["temperature"].double()[:, None]
    # In the order of the logits, equal ones in the order of their indices.
    ranked, order = torch.sort(logits, dim=1, descending=True, stable=True)
    w = torch.where(t > 0, ((ranked - ranked[:, :1]) / torch.where(t > 0, t, 1.0)).exp(), 0.0)
    w[:, 0] = 1.0
    rank = torch.arange(vocab, device="cuda")
    k = s["top_k"][:, None]
    keep = (k <= 0) | (rank < k)
    w = w * keep
    run_to = w.cumsum(1)
    p = s["top_p"].double()[:, None]
    keep &= (p >= 1) | (run_to - w < p * run_to[:, -1:])
    keep &= w >= s["min_p"].double()[:, None]
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, order, w * keep)
    run_to = w.cumsum(1)
    total = run_to[:, -1:]
    token = (run_to > s["u"].double()[:, None] * total).int().argmax(1)
    prob = w.gather(1, token[:, None]) / total
    return {"tokens": token.int(), "probs": prob[:, 0].float()}


# ---- 64 bits, from the definitions ---------------------------------------------------
def exact(c, seed):
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    return {"rope": _exact_rope, "append": _exact_append, "shared": _exact_shared, "sample": _exact_sample}[c["op"]](c, s)


def _exact_turn(c, x, positions):
    """The pairs as complex numbers, multiplied by m e^(i angle)."""
    w, m = _frequencies(c)
    z = torch.polar(torch.full((len(positions), len(w)), m, device="cuda", dtype=torch.float64),
                    torch.outer(positions.double(), w))[:, None]
    x, dim = x.double(), c["dim"]
    body = x[..., :dim]
    if c["layout"] == "half":
        body = torch.complex(body[..., :dim // 2].contiguous(), body[..., dim // 2:].contiguous()) * z
        body = torch.cat([body.real, body.imag], -1)
    else:
        body = torch.view_as_real(torch.view_as_complex(body.unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
    return torch.cat([body, x[..., dim:]], -1)


def _exact_rope(c, s):
    return _exact_turn(c, s["x"], s["positions"])


def _exact_append(c, s):
    k, v, page = s["k"].double(), s["v"].double(), c["page"]
    table, row = s["table"].tolist(), 0
    turned = _exact_turn(c, s["k_new"], s["positions"])
    for i, (n, r) in enumerate(zip(_lengths(c), _rows(c))):
        pos = range(n - r, n)
        ids = torch.tensor([table[i][p // page] for p in pos], device="cuda")
        at = torch.tensor([p % page for p in pos], device="cuda")
        k[0, ids, :, at] = turned[row:row + r]
        v[0, ids, :, at] = s["v_new"][row:row + r].double()
        row += r
    return {"q": _exact_turn(c, s["q"], s["positions"]), "k": k, "v": v}


def _exact_shared(c, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = c["n_head"] // c["n_kv"]
    if c["groups"] * c["each"] * c["n_kv"] > 20000:
        return None
    for i, n in enumerate(_lengths(c)):
        ids = s["table"][i, :-(-n // c["page"])].long()
        for h in range(c["n_kv"]):
            k, v = (x[0, ids, h].reshape(-1, c["hd"])[:n].double() for x in (s["k"], s["v"]))
            q = s["q"][i, h * group:(h + 1) * group].double()
            out[i, h * group:(h + 1) * group] = torch.softmax(q @ k.T / math.sqrt(c["hd"]), -1) @ v
    return out


def _exact_sample(c, s):
    tokens, probs = [], []
    for i in range(c["n"]):
        l = s["logits"][i].double()
        t, k, p, least, u = (float(s[x][i]) for x in ("temperature", "top_k", "top_p", "min_p", "u"))
        if t <= 0:
            tokens.append(int((l == l.max()).nonzero()[0]))
            probs.append(1.0)
            continue
        w = torch.softmax(l / t, 0)
        first = torch.argsort(-l, stable=True)
        if k > 0:
            first = first[:int(k)]
        if p < 1:
            reach = torch.cumsum(w[first], 0)
            first = first[:1 + int((reach[:-1] < p * reach[-1]).sum())]
        first = first[w[first] >= least * w.max()]
        first = first.sort().values
        reach = torch.cumsum(w[first], 0)
        j = int((reach <= u * reach[-1]).sum())
        tokens.append(int(first[j]))
        probs.append(float(w[first[j]] / reach[-1]))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "probs": torch.tensor(probs, dtype=torch.float64)}
