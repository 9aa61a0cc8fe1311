"""Every path of the paged attention against 64 bits, row by row (run with -m gpu).

The bounds, fixed before the first run, are on the 2-norm of a row's error (one
query, one head) relative to the row's, for values that are random and so as
large, by themselves, as what a lost or doubled position would change: of n
equal weights, 16 lost ones change a row by sqrt(16 / n), over 1% up to 160000
positions.

* 16-bit results: with u the type's unit roundoff (f16 2^-11, bf16 2^-8), the
  result's rounding is at most u of the row, and so, in the 2-norm of random
  values, is that of the weights where they are rounded to the type; together
  below sqrt(2 / 3) u on the average, 2 u for any row of 40 columns or more.
* f32 results: queries and weights are good to 2^-22, f32 sums to a few 2^-24,
  and the tensor cores cut about 2^-27 of a sum off per 16 positions and operand,
  3.8e-6 over 4096 positions: below 5e-6 together, 1e-5 allowed for a call and
  2e-5 for a row. One 16-bit operand in place of two is off by more than 3e-5.
"""
import numpy as np
import pytest

from test_gpu_paged import BF16, F16, F32, PAIRS, ctx, ints, queries, torch  # noqa: F401

pytestmark = pytest.mark.gpu
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def pair_id(p):
    return f"{p[0]}-{p[1]}".replace("torch.", "")


class Pool:
    """A cache on the GPU: pages of random rows in random order, NaN and
    infinities wherever no sequence's position is."""

    def __init__(self, ctx, lens, page, n_kv, hd, t, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.page, self.ctx, self.id = lens, page, ctx, 5000
        held = [-(-n // page) for n in lens]
        n_pages = sum(held) + 2
        shape = (1, n_pages, n_kv, page, hd)
        self.k, self.v = (torch.randn(shape, generator=g, device="cuda").to(t) for _ in range(2))
        order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).int()
        table = torch.full((len(lens), max(held + [1]) + 1), -1, dtype=torch.int32)
        stale = torch.ones((n_pages, page), dtype=torch.bool)
        at = 0
        for s, n in enumerate(lens):
            table[s, :held[s]] = order[at:at + held[s]]
            own = torch.arange(held[s] * page).view(-1, page) >= n
            stale[order[at:at + held[s]].long()] = own
            at += held[s]
        stale = stale.cuda()[None, :, None, :, None]
        self.k.masked_fill_(stale, float("nan"))
        self.v.masked_fill_(stale, float("inf"))
        self.table, self.length = table.cuda(), ints(lens)
        refs = (torch.zeros(n_pages, dtype=torch.int32)).scatter_(0, order[:at].long(), 1).cuda()
        ctx.kv_cache(self.id, self.k, self.v, self.table, self.length, refs)

    def rows(self, s):
        ids = self.table[s, :-(-self.lens[s] // self.page)].long()
        return (x[0, ids].transpose(1, 2).reshape(-1, x.shape[2], x.shape[4])[:self.lens[s]] for x in (self.k, self.v))

    def expected(self, q, seqs, counts, scale, window, sinks):
        """In 64 bits, position masks from the definition."""
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        group, r = q.shape[1] // self.k.shape[2], 0
        for s, c in zip(seqs, counts):
            k, v = self.rows(s)
            n = self.lens[s]
            j = torch.arange(n, device="cuda")
            for r0 in range(0, c, 512):
                at = torch.arange(n - c + r0, min(n, n - c + r0 + 512), device="cuda")[:, None]
                see = j <= at
                if window:
                    see &= (j > at - window) | (j < sinks)
                rows = slice(r + r0, r + r0 + len(at))
                if not bool(see.any()):
                    continue
                for h in range(self.k.shape[2]):
                    heads = slice(h * group, (h + 1) * group)
                    score = torch.einsum("rgd,jd->rgj", q[rows, heads].double(), k[:, h].double()) * scale
                    top = score.masked_fill_(~see[:, None], float("-inf")).amax(-1, keepdim=True)
                    p = score.sub_(torch.where(top.isneginf(), 0.0, top)).exp_()
                    total = p.sum(-1, keepdim=True)
                    seen_v = v[:, h].double().masked_fill(~see.any(0)[:, None], 0.0)  # (hidden from all: not touched)
                    out[rows, heads] = p @ seen_v / torch.where(total == 0, 1.0, total)
            r += c
        return out


def near(got, want, t, extra=0.0):
    err = torch.linalg.vector_norm(got.double() - want, dim=-1)
    size = torch.linalg.vector_norm(want, dim=-1)
    assert torch.isfinite(got).all()
    assert bool((err[size == 0] == 0).all())
    rel = (err / size)[size > 0]
    bound = (2 * U[t] if t in U else 2e-5) + extra
    assert float(rel.max()) <= bound, (float(rel.max()), int(rel.argmax()))
    if t == F32:
        assert float(err.norm() / size.norm()) <= 1e-5 + extra


def prompt(ctx, c, q, counts, window=0, sinks=0, seqs=None, scale=None, extra=0.0):
    seqs = list(range(len(counts))) if seqs is None else seqs
    out, again = (torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") for _ in range(2))
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for o in (out, again):
        ctx.attn_prompt_dev(c.id, 0, q, ints([0] + list(np.cumsum(counts))), o, seqs=ints(seqs), window=window,
                            sinks=sinks, scale=scale)
    ctx.sync()
    near(out, c.expected(q, seqs, counts, scale, window, sinks), q.dtype, extra)
    assert torch.equal(out, again)


def decode(ctx, c, q, window=0, sinks=0, seqs=None, scale=None, extra=0.0):
    seqs = list(range(q.shape[0])) if seqs is None else seqs
    out, again = (torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") for _ in range(2))
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for o in (out, again):
        ctx.attn_decode_dev(c.id, 0, q, o, seqs=ints(seqs), window=window, sinks=sinks, scale=scale)
    ctx.sync()
    near(out, c.expected(q, seqs, [1] * len(seqs), scale, window, sinks), q.dtype, extra)
    assert torch.equal(out, again)


# Two row tiles an item (16-bit, 148 pairs of tiles and more), and several items
# a block: rows * group / 256 * key-value heads is 190 to 630.
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 5), (129, 200)])
@pytest.mark.parametrize("heads,counts,lens", [
    ((32, 4, 128), [700, 513, 300], [1000, 513, 2000]),
    ((32, 4, 128), [2600, 1, 2400], [2600, 700, 2900]),
    ((16, 2, 64), [1500, 0, 1700], [1501, 40, 2300]),
    ((20, 5, 80), [999, 1200, 500], [1300, 1200, 3000]),
    ((7, 7, 128), [2000, 1777, 2300], [2000, 2100, 2300]),
    ((5, 1, 40), [4100, 3700], [4100, 3999])], ids=str)
@pytest.mark.parametrize("t", [F16, BF16], ids=str)
def test_two_row_tiles(ctx, t, heads, counts, lens, window, sinks):
    nh, nkv, hd = heads
    c = Pool(ctx, lens, 64 if nh > 16 else 16, nkv, hd, t, seed=sum(lens))
    q = queries(sum(counts), nh, hd, t, 7, pad=3 if nkv == 5 else 0)  # (rows that TMA cannot address)
    prompt(ctx, c, q, counts, window, sinks)


# One row tile an item, more items than blocks, and head sizes past 128.
@pytest.mark.parametrize("window,sinks", [(0, 0), (257, 5)])
@pytest.mark.parametrize("heads,counts,lens", [
    ((32, 4, 128), [700, 513, 300], [1000, 513, 2000]),
    ((8, 2, 64), [3000, 2600], [3000, 4096]),
    ((12, 6, 96), [1100, 900, 30], [1500, 900, 4000]),
    ((8, 2, 200), [2500, 300], [2600, 1300]),
    ((6, 6, 256), [1500, 1300], [1500, 1999])], ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids=pair_id)
def test_more_items_than_blocks(ctx, pair, heads, counts, lens, window, sinks):
    nh, nkv, hd = heads
    c = Pool(ctx, lens, 32, nkv, hd, pair[1], seed=nh)
    prompt(ctx, c, queries(sum(counts), nh, hd, pair[0], 8), counts, window, sinks)


@pytest.mark.parametrize("heads,most", [((8, 2, 64), 60), ((8, 1, 128), 400), ((4, 2, 256), 60)], ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids=pair_id)
def test_prompts_of_many_sequences(ctx, pair, heads, most):
    """More than 32 entries, which are looked for in the list: ragged, some
    without rows, some with more rows than positions, in any order."""
    rng = np.random.default_rng(most)
    nh, nkv, hd = heads
    lens = [int(n) for n in rng.integers(0, 900, 75)]
    lens[3] = lens[40] = 0
    c = Pool(ctx, lens, 16, nkv, hd, pair[1], seed=most)
    seqs = [int(s) for s in rng.permutation(75)]
    counts = [0 if i % 9 == 4 else int(rng.integers(0, most)) for i in range(75)]
    q = queries(sum(counts), nh, hd, pair[0], 9)
    prompt(ctx, c, q, counts, 0, 0, seqs)
    prompt(ctx, c, q, counts, 100, 3, seqs)


@pytest.mark.parametrize("heads,n,most", [((8, 2, 64), 300, 700), ((8, 1, 128), 1000, 90), ((32, 2, 128), 261, 300),
                                          ((4, 2, 256), 140, 500), ((16, 1, 200), 300, 200)], ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids=pair_id)
def test_decode_of_many_sequences(ctx, pair, heads, n, most):
    """More sequences than one round of a block's threads holds."""
    rng = np.random.default_rng(n)
    nh, nkv, hd = heads
    lens = [int(x) for x in rng.integers(0, most, n)]
    lens[5], lens[-1], lens[n // 2] = 4000, 0, 1
    c = Pool(ctx, lens, 16, nkv, hd, pair[1], seed=n)
    q = queries(n, nh, hd, pair[0], 10)
    decode(ctx, c, q)
    decode(ctx, c, q, 64, 17, [int(s) for s in rng.permutation(n)])


@pytest.mark.parametrize("heads", [(8, 1, 128), (4, 2, 64), (32, 2, 80), (20, 1, 96), (7, 1, 40), (2, 2, 256)], ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids=pair_id)
def test_long_rows(ctx, pair, heads):
    """Parts of very unequal sequences, joined; nothing lost between them."""
    nh, nkv, hd = heads
    lens = [4096, 3, 0, 3500, 777, 129]
    c = Pool(ctx, lens, 64, nkv, hd, pair[1], seed=nh)
    q = queries(len(lens), nh, hd, pair[0], 11)
    decode(ctx, c, q)
    decode(ctx, c, q, 1500, 70)
    counts = [33, 3, 0, 1, 70, 129]
    q = queries(sum(counts), nh, hd, pair[0], 12)
    prompt(ctx, c, q, counts)
    prompt(ctx, c, q, counts, 1500, 70)


@pytest.mark.parametrize("rise", [13.0, 40.0, -13.0])
@pytest.mark.parametrize("heads,counts", [((8, 2, 64), [130, 400]), ((8, 1, 128), [64, 37]), ((32, 4, 128), [600, 650]),
                                          ((16, 4, 64), [1500, 1400]), ((4, 2, 200), [130, 20])], ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids=pair_id)
def test_scores_that_rise_and_fall(ctx, pair, heads, counts, rise):
    """Scores that grow by `rise` every 200 positions: each tile outgrows the
    maximum of those before it, past what 16-bit weights hold, so that the sums
    so far are rescaled again and again. Falling: what follows weighs nothing.
    A score of up to 7 rises is a sum of head_dim / 16 steps on the tensor cores,
    each off by up to 2^-23 of it, and so is its weight: added to the bounds."""
    nh, nkv, hd = heads
    lens, extra = [1500, 1430], hd / 16 * 2.0 ** -23 * abs(7 * rise)
    c = Pool(ctx, lens, 32, nkv, hd, pair[1], seed=3)
    for s, n in enumerate(lens):
        j = torch.arange(-(-n // 32) * 32, device="cuda").view(-1, 32)
        ids = c.table[s, :j.shape[0]].long()
        own = (j < n)[:, None].expand(-1, nkv, -1)
        steps = (j // 200 * rise)[:, None].expand(-1, nkv, -1).to(pair[1])
        c.k[0, ids, :, :, 7] = torch.where(own, steps, c.k[0, ids, :, :, 7])
    q = 0.3 * queries(sum(counts), nh, hd, F32, 13)
    q[..., 7] = 1
    q[:, ::3, 7] = 0.5
    prompt(ctx, c, q.to(pair[0]), counts, scale=1.0, extra=extra)
    prompt(ctx, c, q.to(pair[0]), counts, 700, 10, scale=1.0, extra=extra)
    decode(ctx, c, q[:2].to(pair[0]), scale=1.0, extra=extra)


@pytest.mark.parametrize("pair", PAIRS, ids=pair_id)
def test_hidden_values_that_are_not_finite(ctx, pair):
    """Infinities and NaN that lie in tiles a row sees in part, past its own
    position or before its window: of many items, in one and in two row tiles."""
    for heads, n, count in (((32, 4, 128), 1500, 1300), ((4, 1, 64), 900, 130)):
        nh, nkv, hd = heads
        c = Pool(ctx, [n], 16, nkv, hd, pair[1], seed=5)
        at = lambda j: (0, int(c.table[0, j // 16]), slice(None), j % 16)
        c.k[at(n - 1)], c.v[at(n - 1)] = float("nan"), float("inf")  # only the last row sees it
        c.v[at(n - count - 41)][:, 3] = float("nan")                   # no row's window holds it
        q = queries(count, nh, hd, pair[0], 6)
        out = torch.full_like(q, 7.0)
        ctx.attn_prompt_dev(c.id, 0, q, ints([0, count]), out, window=41, sinks=2)
        ctx.sync()
        assert torch.isnan(out[-1]).all()
        c.lens = [n - 1]
        near(out[:-1], c.expected(q[:-1], [0], [count - 1], hd ** -0.5, 41, 2), pair[0])
