"""Measured cases of the paged key-value cache and the attention over it.

Four operators, each as a user calls it through kestrel_b200.cuda.Context:

  decode   attention of one new token per sequence over the pages of a cache
  prompt   attention of the prompt rows of several sequences over the same
           pages, causal, with an optional sliding window and first tokens
           (sinks) that stay visible
  branch   sequences freed, forked, extended (pages allocated; a shared last
           page copied before it is written) and their new rows written
  compact  live pages moved to the front of the pool, the tables following

`own` False computes them in plain torch operations in 32 bits; True calls
the library. The cache: k and v [n_layer, n_pages, n_kv, page, hd], table
[n_seq, max_pages] int32 page ids (-1: none), length [n_seq] int32, refs
[n_pages] int32 holders of each page (0: free).

Key position j is visible to the query at position i when j <= i and
(j > i - window or j < sinks); window 0 is no window. A row that sees nothing
gives zeros.
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
TYPES = [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]  # (query and output, cache)


def listed():
    return [
        # One short sequence of the smallest configuration: a chat's first
        # tokens, where latency counts.
        _attn("decode one short", "decode", 1, 97, 97, 1, (8, 2, 64), 16, 0),
        # A serving batch, sequences at every stage up to a 4096 context.
        _attn("decode batch 32", "decode", 32, 200, 4096, 1, (32, 4, 128), 64, 0),
        # One long document: few rows, so the cache's length is the only axis.
        _attn("decode long", "decode", 1, 131071, 131071, 1, (32, 4, 128), 64, 1),
        # A large ragged batch with a window and sinks over longer caches.
        _attn("decode window 96", "decode", 96, 1500, 8192, 1, (32, 8, 128), 32, 2, window=4096, sinks=4),
        # A short chunk after a short context (a follow-up question).
        _attn("prompt short chunk", "prompt", 1, 545, 545, 33, (8, 2, 64), 16, 0),
        # The runtime's 256-token chunks of several sequences in one call.
        _attn("prompt chunks of 256", "prompt", 6, 300, 4000, 256, (32, 4, 128), 64, 0),
        # One long prompt from its first token, fully causal.
        _attn("prompt 8192", "prompt", 1, 8192, 8192, 8192, (32, 4, 128), 64, 1),
        # Two long prompts of odd lengths under a window with sinks.
        _attn("prompt window 2048", "prompt", 2, 6001, 7400, 7400, (32, 8, 128), 32, 2, window=2048, sinks=16),
        # Parallel samples of one prompt.
        _branch("branch small", 1, 4, 100, 101, 1, 2, (2, 64), 16, 0, 64),
        # A serving batch in which every sequence branches four ways; the
        # pages hold all layers of the model's cache.
        _branch("branch large", 32, 4, 500, 2100, 3, 16, (4, 128), 64, 0, 1600),
        # A small pool with half its pages free.
        _compact("compact small", 8, 40, 300, 2, (2, 64), 16, 0, 256, 0.5),
        # A large pool after many sequences ended: a third of it is free.
        _compact("compact large", 64, 400, 1900, 16, (4, 128), 64, 2, 1800, 0.65),
    ]


def _attn(name, op, n, lo, hi, rows, heads, page, types, window=0, sinks=0):
    return {"name": name, "op": op, "n": n, "len_lo": lo, "len_hi": hi, "rows": rows, "n_head": heads[0],
            "n_kv": heads[1], "hd": heads[2], "page": page, "t_q": TYPES[types][0], "t_kv": TYPES[types][1],
            "window": window, "sinks": sinks}


def _branch(name, parents, children, lo, hi, rows, layers, heads, page, types, pages):
    return {"name": name, "op": "branch", "n": parents, "children": children, "len_lo": lo, "len_hi": hi,
            "rows": rows, "layers": layers, "n_kv": heads[0], "hd": heads[1], "page": page,
            "t_q": TYPES[types][0], "t_kv": TYPES[types][1], "pages": pages}


def _compact(name, n, lo, hi, layers, heads, page, types, pages, full):
    return {"name": name, "op": "compact", "n": n, "len_lo": lo, "len_hi": hi, "layers": layers,
            "n_kv": heads[0], "hd": heads[1], "page": page, "t_kv": TYPES[types][1], "pages": pages, "full": full}


def _between(rng, lo, hi):
    """A whole number of lo .. hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "branch", "compact"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        heads, page, types = rng.choice(HEADS), rng.choice([16, 32, 64, 128]), rng.randrange(3)
        if op in ("decode", "prompt"):
            hi = _between(rng, 40, 131072 if op == "decode" else 8192)
            lo = max(1, int(hi * rng.uniform(0.1, 1.0)))
            n = _between(rng, 1, 128 if op == "decode" else 12)
            rows = 1 if op == "decode" else _between(rng, 2, hi)
            window = rng.choice([0, _between(rng, 16, 8192)])
            c = _attn("", op, n, lo, hi, rows, heads, page, types, window, rng.choice([0, 1, 4, 64]) if window else 0)
            fits = n * hi * heads[1] * heads[2] <= 1.1e9 and (op == "decode" or n * heads[0] * rows * hi <= 2.3e9)
        elif op == "branch":
            hi = _between(rng, 30, 4000)
            n, children = _between(rng, 1, 48), rng.randint(1, 6)
            lo, rows = max(1, hi // rng.randint(1, 8)), rng.randint(1, 40)
            pages = n * (hi // page + 1) + n * children * (rows // page + 2)
            pages += rng.randint(0, pages)
            c = _branch("", n, children, lo, hi, rows, rng.randint(1, 24), heads[1:], page, types, pages)
            fits = True
        else:
            hi, n = _between(rng, 30, 4000), _between(rng, 1, 100)
            full = rng.uniform(0.1, 0.95)
            pages = max(8, int(n * (hi // page + 1) / full))
            c = _compact("", n, max(1, hi // rng.randint(1, 8)), hi, rng.randint(1, 24), heads[1:], page, types,
                         pages, round(full, 3))
            fits = True
        if op in ("branch", "compact"):
            fits = c["pages"] * c["layers"] * c["n_kv"] * c["page"] * c["hd"] <= 9.5e8
        if fits and _cost(c) <= most:
            del c["name"]
            return c


def _cost(c):
    w = work(c)
    return w["bytes"] + w["flops"] / 200


def _lengths(c):
    """Positions held by each sequence: the case's, whatever the seed."""
    r = random.Random("%d %d %d" % (c["n"], c["len_lo"], c["len_hi"]))
    ls = [r.randint(c["len_lo"], c["len_hi"]) for _ in range(c["n"])]
    ls[0] = c["len_hi"]
    return ls


def _rows(c):
    """Query rows of each sequence of a prompt call (its last positions)."""
    return [min(n, c["rows"]) for n in _lengths(c)]


def _seen(c, pos):
    """Key positions visible to the query at `pos` (a tensor)."""
    if not c["window"]:
        return pos + 1
    lo = (pos - c["window"] + 1).clamp(min=0)
    return pos + 1 - lo + torch.minimum(lo, torch.tensor(c["sinks"]))


def work(c):
    if c["op"] in ("decode", "prompt"):
        seen = keys = rows = 0
        for n, r in zip(_lengths(c), [1] * c["n"] if c["op"] == "decode" else _rows(c)):
            seen += int(_seen(c, torch.arange(n - r, n)).sum())
            rows += r
            # key positions that any of the sequence's rows sees
            lo = max(0, n - r - c["window"] + 1) if c["window"] else 0
            keys += n - lo + min(lo, c["sinks"])
        io = rows * c["n_head"] * c["hd"] * DTYPES[c["t_q"]].itemsize * 2
        return {"bytes": keys * c["n_kv"] * c["hd"] * 4 + io + keys // c["page"] * 4,
                "flops": 4 * seen * c["n_head"] * c["hd"]}
    tok = c["n_kv"] * c["hd"] * 4  # bytes of one position of one layer, k and v
    if c["op"] == "branch":
        part = sum(n % c["page"] for n in _lengths(c)) * c["children"]
        new = c["n"] * c["children"] * c["rows"]
        table = sum(-(-n // c["page"]) for n in _lengths(c)) * c["children"] * 4
        return {"bytes": 2 * part * tok * c["layers"] + new * (tok + c["n_kv"] * c["hd"] * 2 * DTYPES[c["t_q"]].itemsize)
                + 2 * table + c["pages"] * 4, "flops": 0}
    used = _compact_used(c)
    moved = round(used * (1 - used / c["pages"]))  # what a random order of the pages leaves above the live ones
    return {"bytes": 2 * moved * c["page"] * tok * c["layers"] + c["pages"] * 8 + used * 8, "flops": 0}


def _compact_used(c):
    return sum(-(-n // c["page"]) for n in _lengths(c))


_context = None
_ids = itertools.count()


def _handle(s):
    """The library's handle of a state's cache, as a user's program keeps it."""
    global _context
    from kestrel_b200.cuda import Context
    if _context is None:
        _context = Context(torch.cuda.current_device())
        _context.set_stream(torch.cuda.current_stream().cuda_stream)
    s["ctx"], s["id"] = _context, next(_ids)
    _context.kv_cache(s["id"], s["k"], s["v"], s["table"], s["length"], s["refs"])


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    t_kv, page, lens = DTYPES[c["t_kv"]], c["page"], _lengths(c)
    extra = c["rows"] if c["op"] == "branch" else 0
    used = [-(-n // page) for n in lens]
    n_seq = c["n"] * (1 + c.get("children", 0))
    n_pages = c.get("pages") or sum(used) + 3
    layers = c.get("layers", 1)
    width = max(-(-(n + extra) // page) for n in lens)
    table = torch.full((n_seq, width), -1, dtype=torch.int32)
    order = torch.randperm(n_pages, generator=cpu, dtype=torch.int32)[:sum(used)].split(used)
    for i, ids in enumerate(order):
        table[i, :len(ids)] = ids
    length = torch.tensor(lens + [0] * (n_seq - c["n"]), dtype=torch.int32)
    refs = torch.zeros(n_pages, dtype=torch.int32)
    refs[torch.cat(order).long()] = 1
    shape = (layers, n_pages, c["n_kv"], page, c["hd"])
    s = {"case": c, "table": table.cuda(), "length": length.cuda(), "refs": refs.cuda(),
         "k": torch.randn(shape, generator=g, device="cuda", dtype=t_kv),
         "v": torch.randn(shape, generator=g, device="cuda", dtype=t_kv)}
    if c["op"] in ("decode", "prompt"):
        t_q, rows = DTYPES[c["t_q"]], [1] * c["n"] if c["op"] == "decode" else _rows(c)
        start = torch.tensor([0] + list(itertools.accumulate(rows)), dtype=torch.int32)
        s["row_start"], s["n_rows"], s["max_rows"] = start.cuda(), int(start[-1]), max(rows)
        # Queries as a normalised projection gives them: scores of a few units,
        # so that some keys stand out.
        s["q"] = (1.5 * torch.randn((s["n_rows"], c["n_head"], c["hd"]), generator=g, device="cuda")).to(t_q)
        s["out"] = torch.empty_like(s["q"])
    elif c["op"] == "branch":
        kids, m = c["n"] * c["children"], c["rows"]
        s["src"] = torch.arange(c["n"], dtype=torch.int32, device="cuda").repeat_interleave(c["children"])
        s["dst"] = torch.arange(c["n"], n_seq, dtype=torch.int32, device="cuda")
        s["n_new"] = torch.full((kids,), m, dtype=torch.int32, device="cuda")
        s["row_start"] = torch.arange(0, kids * m + 1, m, dtype=torch.int32, device="cuda")
        s["layer"] = layers - 1
        for x in ("k_new", "v_new"):
            s[x] = torch.randn((kids * m, c["n_kv"], c["hd"]), generator=g, device="cuda").to(DTYPES[c["t_q"]])
    else:
        for x in ("table", "refs"):
            s[x + "_0"] = s[x].clone()
    if own:
        _handle(s)
    return s


def run(s):
    op = s["case"]["op"]
    if op in ("decode", "prompt"):
        return _run_attention(s)
    if op == "branch":
        return _run_branch(s)
    return _run_compact(s)


def _cache(s):
    return {x: s[x] for x in ("k", "v", "table", "length", "refs")}


def _run_attention(s):
    c = s["case"]
    scale = c["hd"] ** -0.5
    if own:
        if c["op"] == "decode":
            s["ctx"].attn_decode_dev(s["id"], 0, s["q"], s["out"], scale=scale, window=c["window"], sinks=c["sinks"])
        else:
            s["ctx"].attn_prompt_dev(s["id"], 0, s["q"], s["row_start"], s["out"], scale=scale, window=c["window"],
                                     sinks=c["sinks"])
        return s["out"]
    n, nkv, hd, group = c["n"], c["n_kv"], c["hd"], c["n_head"] // c["n_kv"]
    ids = s["table"].clamp(min=0).long()
    k, v = (x[0][ids].transpose(1, 2).reshape(n, nkv, -1, hd).float() for x in (s["k"], s["v"]))
    # Rows of every sequence side by side, padded to the longest.
    start, length = s["row_start"].long(), s["length"].long()
    count = start[1:] - start[:-1]
    step = torch.arange(s["max_rows"], device="cuda")
    real = step[None] < count[:, None]
    row = (start[:-1, None] + step[None]).clamp(max=s["n_rows"] - 1)
    q = s["q"][row].float().view(n, -1, nkv, group, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, hd)
    at = (length - count)[:, None] + step[None]
    key = torch.arange(k.shape[2], device="cuda")
    see = (key <= at[..., None]) & (key < length[:, None, None])
    if c["window"]:
        see &= (key > at[..., None] - c["window"]) | (key < c["sinks"])
    see = see[:, None, None]
    score = (q @ k.transpose(2, 3)).mul_(scale).view(n, nkv, group, -1, key.numel())
    score = score.masked_fill_(~see, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(n, nkv, -1, key.numel()) @ v).view(n, nkv, group, -1, hd) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(n, -1, c["n_head"], hd)[real].to(s["q"].dtype)


def _run_branch(s):
    if own:
        ctx, cache = s["ctx"], s["id"]
        ctx.kv_free_dev(cache, s["dst"])
        ctx.kv_fork_dev(cache, s["src"], s["dst"])
        ctx.kv_extend_dev(cache, s["dst"], s["n_new"])
        ctx.kv_write_dev(cache, s["layer"], s["k_new"], s["v_new"], seqs=s["dst"], row_start=s["row_start"])
        return _cache(s)
    page, table, length, refs = s["case"]["page"], s["table"], s["length"], s["refs"]
    src, dst, n_new = s["src"].long(), s["dst"].long(), s["n_new"].long()
    # Free what the branches of the last pass held.
    old = table[dst]
    held = old >= 0
    refs.index_add_(0, old[held].long(), -torch.ones_like(old[held]))
    # Fork: the branch shares its parent's pages.
    table[dst] = table[src]
    length[dst] = length[src]
    got = table[dst]
    refs.index_add_(0, got[got >= 0].long(), torch.ones_like(got[got >= 0]))
    # Extend. A shared last page that is partly full is copied first, by its
    # holders in their order until one is left; new pages are the lowest free.
    ln = length[dst].long()
    have, want = (ln + page - 1) // page, (ln + n_new + page - 1) // page
    last = table[dst, (have - 1).clamp(min=0)].long()
    part = (ln % page != 0) & (n_new > 0)
    before = ((last[:, None] == last[None]) & part[:, None] & part[None]).tril(-1).sum(1)
    copy = part & (refs[last.clamp(min=0)] - before > 1)
    need = want - have + copy
    first = need.cumsum(0) - need
    free = torch.argsort((refs > 0).int(), stable=True)
    slot = torch.arange(table.shape[1] + 1, device="cuda")
    take = slot[None] < need[:, None]
    ids = free[(first[:, None] + slot[None]).clamp(max=free.numel() - 1)]
    col = (have - copy.long())[:, None] + slot[None]
    seq = dst[:, None].expand_as(col)
    table[seq[take], col[take]] = ids[take].int()
    refs[ids[take]] = 1
    refs.index_add_(0, last[copy], -torch.ones_like(last[copy], dtype=torch.int32))
    keep = (torch.arange(page, device="cuda")[None] < (ln % page)[copy][:, None])[None, :, None, :, None]
    for x in (s["k"], s["v"]):
        x[:, ids[copy, 0]] = torch.where(keep, x[:, last[copy]], x[:, ids[copy, 0]])
    length[dst] += s["n_new"]
    # Write the new rows.
    count = (s["row_start"][1:] - s["row_start"][:-1]).long()
    seq = dst.repeat_interleave(count)
    row = torch.arange(seq.numel(), device="cuda")
    pos = length[seq].long() - (s["row_start"][1:].long().repeat_interleave(count) - row)
    to = table[seq, pos // page].long()
    for x, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
        x[s["layer"]][to, :, pos % page] = new.to(x.dtype)
    return _cache(s)


def _run_compact(s):
    # The fragmented state comes back first: the pages that compaction moved
    # still hold their rows.
    for x in ("table", "refs"):
        s[x].copy_(s[x + "_0"])
    if own:
        s["ctx"].kv_compact_dev(s["id"])
        return _cache(s)
    refs, table = s["refs"], s["table"]
    live = refs > 0
    below = torch.arange(refs.numel(), device="cuda") < live.sum()
    hole, move = (~live & below).nonzero()[:, 0], (live & ~below).nonzero()[:, 0]
    for x in (s["k"], s["v"]):
        x[:, hole] = x[:, move]
    to = torch.arange(refs.numel(), device="cuda", dtype=torch.int32)
    to[move] = hole.int()
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    refs[hole] = refs[move]
    refs[move] = 0
    return _cache(s)


def exact(c, seed):
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    if c["op"] in ("decode", "prompt"):
        return _exact_attention(c, s)
    k, v = s["k"].double(), s["v"].double()
    table, length, refs = s["table"].tolist(), s["length"].tolist(), s["refs"].tolist()
    page = c["page"]
    if c["op"] == "branch":
        moves, src, dst = [], s["src"].tolist(), s["dst"].tolist()
        for a, b in zip(src, dst):
            table[b], length[b] = list(table[a]), length[a]
            for p in table[b]:
                if p >= 0:
                    refs[p] += 1
        free = [p for p in range(len(refs)) if refs[p] == 0][::-1]
        for b in dst:
            n, m = length[b], length[b] + c["rows"]
            if n % page and refs[table[b][n // page]] > 1:
                p, new = table[b][n // page], free.pop()
                refs[p], refs[new], table[b][n // page] = refs[p] - 1, 1, new
                moves.append((p, new, n % page))
            for j in range(-(-n // page), -(-m // page)):
                table[b][j] = free.pop()
                refs[table[b][j]] = 1
            length[b] = m
        for p, new, rows in moves:
            k[:, new, :, :rows], v[:, new, :, :rows] = k[:, p, :, :rows], v[:, p, :, :rows]
        for i, b in enumerate(dst):
            for r in range(c["rows"]):
                pos = length[b] - c["rows"] + r
                for x, new in ((k, s["k_new"]), (v, s["v_new"])):
                    x[s["layer"], table[b][pos // page], :, pos % page] = new[i * c["rows"] + r].to(s["k"].dtype).double()
    else:
        n_live = sum(r > 0 for r in refs)
        holes = [p for p in range(n_live) if refs[p] == 0]
        moving = [p for p in range(n_live, len(refs)) if refs[p] > 0]
        to = dict(zip(moving, holes))
        if moving:
            k[:, holes], v[:, holes] = k[:, moving], v[:, moving]
        for a, b in to.items():
            refs[b], refs[a] = refs[a], 0
        table = [[to.get(p, p) for p in row] for row in table]
    return {"k": k, "v": v, "table": torch.tensor(table, dtype=torch.int32),
            "length": torch.tensor(length, dtype=torch.int32), "refs": torch.tensor(refs, dtype=torch.int32)}


def _exact_attention(c, s):
    out = torch.zeros((s["n_rows"], c["n_head"], c["hd"]), dtype=torch.float64, device="cuda")
    group, start = c["n_head"] // c["n_kv"], s["row_start"].tolist()
    for i, n in enumerate(_lengths(c)):
        ids = s["table"][i, :-(-n // c["page"])].long()
        rows = slice(start[i], start[i + 1])
        at = torch.arange(n - (rows.stop - rows.start), n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        hidden = j > at
        if c["window"]:
            hidden |= (j <= at - c["window"]) & (j >= c["sinks"])
        for h in range(c["n_kv"]):
            k, v = (x[0, ids, h].reshape(-1, c["hd"])[:n].double() for x in (s["k"], s["v"]))
            for g in range(h * group, (h + 1) * group):
                score = s["q"][rows, g].double() @ k.T / math.sqrt(c["hd"])
                out[rows, g] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
    return out
