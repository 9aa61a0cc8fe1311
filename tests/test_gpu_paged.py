"""The paged cache and its attention against plain models (run with -m gpu).

Tolerances, fixed before the first run. With u the unit roundoff of the query /
output type (f16 2^-11, bf16 2^-8), an output is a weighted mean of values of
at most max|v|: the weights' rounding to that type and the result's own each
move it by at most u * max|v|, so 2 u max|v| bounds a 16-bit result (scores and
sums are f32). For f32 results the queries and weights carry at least 21 bits;
a score is a sum of at most 256 products whose magnitudes add up to about
sqrt(head_dim) <= 16 here, so it is off by at most 16 * 2^-21 * 2, its weight by
that share, and the mean by twice it: 2^-15 max|v|.
Page contents, tables, lengths and counts are equal, bit for bit.
"""
import numpy as np
import pytest

from paged_model import PageModel, Refused, attention

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TOL = {F32: 2.0 ** -15, F16: 2.0 ** -10, BF16: 2.0 ** -7}
PAIRS = [(F32, F16), (F16, F16), (BF16, BF16)]


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from kestrel_b200.cuda import Context
    c = Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def wide(t):
    return t.float().cpu().numpy()


class Cache:
    """A cache of random rows on the GPU, its model beside it."""
    ids = iter(range(1 << 30))

    def __init__(self, ctx, lens, page, n_kv, hd, t, n_layer=2, spare=3, seed=0, poison=True, max_pages=None):
        rng = np.random.default_rng(seed)
        held = [-(-n // page) for n in lens]
        n_pages, max_pages = sum(held) + spare, max_pages or max(held + [1]) + 1
        g = torch.Generator(device="cuda").manual_seed(seed)
        shape = (n_layer, n_pages, n_kv, page, hd)
        self.k, self.v = (torch.randn(shape, generator=g, device="cuda").to(t) for _ in range(2))
        self.m = PageModel(n_layer, n_pages, page, n_kv, hd, len(lens), max_pages, wide(self.k), wide(self.v))
        order = list(rng.permutation(n_pages))
        for s, n in enumerate(lens):
            for j in range(held[s]):
                p = int(order.pop())
                self.m.table[s][j], self.m.refs[p] = p, 1
            self.m.length[s] = n
        if poison:  # what no sequence holds is NaN and infinities, on the GPU and in the model
            used = torch.zeros((n_pages, page), dtype=torch.bool)
            for s, n in enumerate(lens):
                for j in range(n):
                    used[self.m.table[s][j // page], j % page] = True
            for x, bad in ((self.k, float("nan")), (self.v, float("inf"))):
                x.masked_fill_(~used.cuda()[None, :, None, :, None], bad)
            self.m.k, self.m.v = wide(self.k), wide(self.v)
        self.table, self.length, self.refs = ints(self.m.table), ints(self.m.length), ints(self.m.refs)
        self.ctx, self.id = ctx, next(Cache.ids)
        ctx.kv_cache(self.id, self.k, self.v, self.table, self.length, self.refs)

    def same(self):
        self.ctx.sync()
        self.m.check()
        assert self.length.tolist() == self.m.length
        assert self.refs.tolist() == self.m.refs
        assert self.table.tolist() == self.m.table
        assert np.array_equal(wide(self.k), self.m.k, equal_nan=True)
        assert np.array_equal(wide(self.v), self.m.v, equal_nan=True)

    def expected(self, layer, q, seqs, counts, scale, window, sinks):
        out, r = [], 0
        for s, c in zip(seqs, counts):
            k, v = self.m.rows(layer, s)
            out.append(attention(q[r:r + c], k, v, len(k) - c, scale, window, sinks))
            r += c
        return np.concatenate(out)


def close(got, want, t):
    """Within the tolerance of values of unit normal size (max|v| <= 6 here)."""
    assert got.shape == want.shape
    assert np.isfinite(got).all() == np.isfinite(want).all()
    err = np.abs(got.astype(np.float64) - want).max(initial=0.0)
    assert err <= TOL[t] * 6, err


def queries(rows, nh, hd, t, seed, pad=0):
    """q as a slice of wider rows (`pad` values before and after)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.randn((rows, nh * hd + 2 * pad), generator=g, device="cuda").to(t)
    return buf[:, pad:pad + nh * hd].unflatten(1, (nh, hd))


# (query heads, kv heads, head size): this package's configurations, one head
# per group, groups that are no power of two, more than sixteen and a hundred
# heads to one, head sizes that are no multiple of 64 or 16, and the extremes.
HEADS = [(8, 2, 64), (32, 4, 128), (4, 4, 64), (7, 1, 128), (6, 2, 80), (20, 1, 96), (128, 1, 64), (3, 1, 8),
         (10, 2, 256), (4, 2, 40), (5, 1, 200)]
LENS = [1, 0, 15, 16, 17, 64, 129, 300]


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: f"{p[0]}-{p[1]}".replace("torch.", ""))
def test_decode(ctx, heads, pair):
    nh, nkv, hd = heads
    for page, window, sinks in ((16, 0, 0), (32, 20, 3), (128, 1, 0), (256, 100, 64)):
        c = Cache(ctx, LENS, page, nkv, hd, pair[1], seed=nh + page)
        q = queries(len(LENS), nh, hd, pair[0], 5)
        out = torch.full_like(q.contiguous(), 7.0)
        c.ctx.attn_decode_dev(c.id, 1, q, out, window=window, sinks=sinks)
        ctx.sync()
        close(wide(out), c.expected(1, wide(q), range(len(LENS)), [1] * len(LENS), hd ** -0.5, window, sinks), pair[0])


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: f"{p[0]}-{p[1]}".replace("torch.", ""))
def test_prompt(ctx, heads, pair):
    nh, nkv, hd = heads
    lens, counts = [40, 0, 129, 200, 1, 33, 70], [40, 0, 1, 37, 1, 32, 17]
    for page, window, sinks in ((16, 0, 0), (64, 20, 3), (32, 1, 0), (128, 130, 40)):
        c = Cache(ctx, lens, page, nkv, hd, pair[1], seed=nh + page)
        q = queries(sum(counts), nh, hd, pair[0], 6)
        out = torch.full_like(q.contiguous(), 7.0)
        start = ints([0] + list(np.cumsum(counts)))
        c.ctx.attn_prompt_dev(c.id, 1, q, start, out, window=window, sinks=sinks)
        ctx.sync()
        close(wide(out), c.expected(1, wide(q), range(len(lens)), counts, hd ** -0.5, window, sinks), pair[0])


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: f"{p[0]}-{p[1]}".replace("torch.", ""))
def test_prompt_long_rows(ctx, pair):
    """Several tiles of rows and of positions; window edges inside tiles."""
    for (nh, nkv, hd), n, count, window, sinks in (((4, 2, 64), 700, 700, 0, 0), ((4, 1, 128), 900, 401, 0, 0),
                                                   ((2, 2, 96), 1000, 500, 260, 5), ((3, 1, 128), 611, 611, 128, 130),
                                                   ((2, 1, 256), 515, 300, 0, 0), ((2, 1, 200), 515, 300, 257, 1)):
        c = Cache(ctx, [n, 50], 32, nkv, hd, pair[1], seed=n)
        q = queries(count + 50, nh, hd, pair[0], 7)
        out = torch.empty_like(q.contiguous())
        ctx.attn_prompt_dev(c.id, 0, q, ints([0, count, count + 50]), out, window=window, sinks=sinks)
        ctx.sync()
        close(wide(out), c.expected(0, wide(q), [0, 1], [count, 50], hd ** -0.5, window, sinks), pair[0])


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: f"{p[0]}-{p[1]}".replace("torch.", ""))
def test_decode_long(ctx, pair):
    """Long and very unequal lengths: many parts to join, and none."""
    lens = [9001, 3, 0, 5000, 777]
    for (nh, nkv, hd), window, sinks in (((8, 1, 128), 0, 0), ((4, 2, 64), 0, 0), ((32, 2, 80), 4100, 70)):
        c = Cache(ctx, lens, 64, nkv, hd, pair[1], seed=nh)
        q = queries(len(lens), nh, hd, pair[0], 8)
        out = torch.empty_like(q.contiguous())
        ctx.attn_decode_dev(c.id, 0, q, out, window=window, sinks=sinks)
        ctx.sync()
        close(wide(out), c.expected(0, wide(q), range(5), [1] * 5, hd ** -0.5, window, sinks), pair[0])


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: f"{p[0]}-{p[1]}".replace("torch.", ""))
def test_sequence_order_strides_and_scale(ctx, pair):
    """seqs in any order, rows that are slices of wider ones at odd offsets,
    output rows in no sequence's range left alone, scales of either sign."""
    c = Cache(ctx, [30, 100, 5, 64], 16, 2, 64, pair[1])
    for pad, scale in ((8, 0.3), (1, -0.2), (3, 0.0)):
        q = queries(3, 4, 64, pair[0], 9, pad)
        buf = torch.full((3, 4 * 64 + 2 * pad), 7.0, device="cuda", dtype=pair[0])
        out = buf[:, pad:pad + 256].unflatten(1, (4, 64))
        ctx.attn_decode_dev(c.id, 1, q, out, seqs=ints([3, 0, 2]), scale=scale)
        ctx.sync()
        close(wide(out), c.expected(1, wide(q), [3, 0, 2], [1, 1, 1], scale, 0, 0), pair[0])
        assert (buf[:, :pad] == 7).all() and (buf[:, pad + 256:] == 7).all()
        q = queries(40, 4, 64, pair[0], 10, pad)
        buf = torch.full((40, 4 * 64 + 2 * pad), 7.0, device="cuda", dtype=pair[0])
        out = buf[:, pad:pad + 256].unflatten(1, (4, 64))
        ctx.attn_prompt_dev(c.id, 1, q, ints([2, 27, 30]), out, seqs=ints([1, 2]), scale=scale)
        ctx.sync()
        close(wide(out)[2:30], c.expected(1, wide(q)[2:30], [1, 2], [25, 3], scale, 0, 0), pair[0])
        assert (buf[:2] == 7).all() and (buf[30:] == 7).all()
        assert (buf[:, :pad] == 7).all() and (buf[:, pad + 256:] == 7).all()


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: f"{p[0]}-{p[1]}".replace("torch.", ""))
def test_values_at_the_ends_of_the_range(ctx, pair):
    """Scores far apart, equal scores, one that outweighs all others, and rows
    that hold more than the first ones see."""
    c = Cache(ctx, [200, 200, 200], 16, 1, 64, pair[1], poison=False)
    k, v = c.k, c.v
    ids = c.table[1, :13].long()
    k[0, ids] = 0  # every score equal
    top = int(c.table[2, 3])
    k[0, top, :, 5] = 60  # position 53 outweighs the rest
    k[0, int(c.table[0, 11]), :, 9] = float("nan")  # position 185
    v[0, int(c.table[0, 11]), :, 10] = float("inf")  # position 186
    c.m.k, c.m.v = wide(k), wide(v)
    q = queries(3 * 60, 2, 64, pair[0], 11)
    q[60:] = q[60:].abs()
    out = torch.empty_like(q.contiguous())
    ctx.attn_prompt_dev(c.id, 0, q, ints([0, 60, 120, 180]), out)
    ctx.sync()
    want = c.expected(0, wide(q), [0, 1, 2], [60] * 3, 0.125, 0, 0)
    got = wide(out)
    # Sequence 0: rows 0 .. 44 do not see position 185; later ones see NaN.
    assert np.isnan(want[45:60]).all() and np.isnan(got[45:60]).all()
    close(got[:45], want[:45], pair[0])
    close(got[60:], want[60:], pair[0])
    # Single tokens, the NaN outside the window and inside it.
    q = queries(3, 2, 64, pair[0], 12)
    out = torch.empty_like(q.contiguous())
    ctx.attn_decode_dev(c.id, 0, q, out, window=13, sinks=100)
    ctx.sync()
    close(wide(out), c.expected(0, wide(q), [0, 1, 2], [1] * 3, 0.125, 13, 100), pair[0])
    ctx.attn_decode_dev(c.id, 0, q, out)
    ctx.sync()
    assert np.isnan(wide(out)[0]).all()


def test_large_f32_queries(ctx):
    """f32 queries beyond f16's range, against keys small enough to leave
    ordinary scores."""
    c = Cache(ctx, [90, 300], 16, 2, 64, F16, poison=False)
    c.k.mul_(2.0 ** -12)
    c.m.k = wide(c.k)
    q = queries(2, 8, 64, F32, 3) * 2.0 ** 18
    out = torch.empty_like(q)
    # The scores are sums of products of about 64 * 2^6 * scale.
    ctx.attn_decode_dev(c.id, 0, q, out, scale=2.0 ** -9)
    ctx.sync()
    close(wide(out), c.expected(0, wide(q), [0, 1], [1, 1], 2.0 ** -9, 0, 0), F32)
    q = queries(100, 8, 64, F32, 3) * 2.0 ** 18
    out = torch.empty_like(q)
    ctx.attn_prompt_dev(c.id, 0, q, ints([0, 30, 100]), out, scale=2.0 ** -9)
    ctx.sync()
    close(wide(out), c.expected(0, wide(q), [0, 1], [30, 70], 2.0 ** -9, 0, 0), F32)


def test_results_repeat(ctx):
    """The same call twice gives the same bits (parts are joined in order)."""
    c = Cache(ctx, [5000, 41, 900], 32, 2, 128, F16)
    q = queries(3, 16, 128, F32, 4)
    outs = [torch.empty_like(q.contiguous()) for _ in range(6)]
    for o in outs:
        ctx.attn_decode_dev(c.id, 0, q, o)
    qp = queries(130, 16, 128, F32, 5)
    more = [torch.empty_like(qp.contiguous()) for _ in range(6)]
    for o in more:
        ctx.attn_prompt_dev(c.id, 0, qp, ints([0, 100, 130, 130]), o)
    ctx.sync()
    for o in outs[1:]:
        assert torch.equal(o, outs[0])
    for o in more[1:]:
        assert torch.equal(o, more[0])


@pytest.mark.parametrize("page,t", [(16, F16), (64, BF16), (256, F16)], ids=str)
def test_page_operations(ctx, page, t):
    """Two hundred random calls, the model beside them; everything equal after
    each, and attention over what they leave."""
    rng = np.random.default_rng(page)
    n_seq, n_layer, n_kv, hd = 7, 3, 2, 24
    c = Cache(ctx, [0] * n_seq, page, n_kv, hd, t, n_layer=n_layer, spare=24, seed=page, poison=False, max_pages=9)
    refused = 0
    for step in range(200):
        op = rng.choice(["extend", "extend", "extend", "fork", "free", "compact"])
        seqs = [int(s) for s in rng.permutation(n_seq)[:rng.integers(1, n_seq + 1)]]
        if op == "extend":
            add = [int(rng.choice([0, 1, 2, page - 1, page, int(rng.integers(1, 3 * page))])) for _ in seqs]
            ctx.kv_extend_dev(c.id, ints(seqs), ints(add))
            try:
                c.m.extend(seqs, add)
            except Refused:
                refused += 1
                with pytest.raises(Exception, match="free pages|more positions"):
                    ctx.sync()
                continue
            layer, src = int(rng.integers(n_layer)), rng.choice([0, 1])
            rows = sum(add)
            if rows:
                x = torch.randn((rows, (n_kv + 3) * hd), device="cuda").to(F32 if src else t)
                k, v = x[:, :n_kv * hd].unflatten(1, (n_kv, hd)), x[:, 3 * hd:].unflatten(1, (n_kv, hd))
                ctx.kv_write_dev(c.id, layer, k, v, seqs=ints(seqs), row_start=ints([0] + list(np.cumsum(add))))
                c.m.write(layer, seqs, add, wide(k.to(t)), wide(v.to(t)))
        elif op == "fork":
            empty = [s for s in range(n_seq) if not c.m.length[s]]
            full = [s for s in range(n_seq) if c.m.length[s]]
            if not empty or not full:
                continue
            dst = empty[:rng.integers(1, len(empty) + 1)]
            src = [int(rng.choice(full)) for _ in dst]
            ctx.kv_fork_dev(c.id, ints(src), ints(dst))
            c.m.fork(src, dst)
        elif op == "free":
            seqs = seqs[:3]
            keep = None if rng.random() < 0.5 else [int(rng.integers(0, 4 * page)) for _ in seqs]
            ctx.kv_free_dev(c.id, ints(seqs), None if keep is None else ints(keep))
            c.m.free(seqs, keep)
        else:
            live = ints([-1])
            ctx.kv_compact_dev(c.id, live)
            assert live.item() == c.m.compact()
        if step % 10 == 0:
            c.same()
    c.same()
    assert refused  # the pool is small enough to run out
    q = queries(n_seq, 4, hd, t, 1)
    out = torch.empty_like(q.contiguous())
    ctx.attn_decode_dev(c.id, 1, q, out)
    ctx.sync()
    close(wide(out), c.expected(1, wide(q), range(n_seq), [1] * n_seq, hd ** -0.5, 0, 0), t)


def test_copy_pages(ctx):
    c = Cache(ctx, [100], 16, 3, 40, F16, n_layer=3, spare=8, poison=False)
    free = [p for p in range(c.m.n_pages) if not c.m.refs[p]]
    src, dst = [c.m.table[0][2], c.m.table[0][2], c.m.table[0][6]], free[:3]
    ctx.kv_copy_pages_dev(c.id, ints(src), ints(dst))
    for a, b in zip(src, dst):
        c.m.k[:, b], c.m.v[:, b] = c.m.k[:, a], c.m.v[:, a]
    c.same()
    for src, dst in (([0, 1], [free[0], free[0]]), ([0, free[0]], [free[0], free[1]]), ([0], [c.m.n_pages]),
                     ([-1], [0])):
        ctx.kv_copy_pages_dev(c.id, ints(src), ints(dst))
        with pytest.raises(Exception, match="page to copy"):
            ctx.sync()
        c.same()


def test_large_tables_and_pools(ctx):
    """More pages and sequences than one pass of the bookkeeping kernels."""
    rng = np.random.default_rng(3)
    n_pages, n_seq = 30000, 1500
    k = torch.zeros((1, n_pages, 1, 16, 8), dtype=F16, device="cuda")
    v = torch.zeros_like(k)
    c = Cache(ctx, [0] * 2, 16, 1, 8, F16)  # its methods, on other tensors
    c.k, c.v = k, v
    c.m = PageModel(1, n_pages, 16, 1, 8, n_seq, 40, wide(k), wide(v))
    c.table, c.length, c.refs = ints(c.m.table), ints(c.m.length), ints(c.m.refs)
    ctx.kv_cache(c.id, k, v, c.table, c.length, c.refs)
    add = [int(x) for x in rng.integers(0, 300, n_seq)]
    ctx.kv_extend_dev(c.id, None, ints(add))
    c.m.extend(list(range(n_seq)), add)
    c.same()
    gone = [int(s) for s in rng.permutation(n_seq)[:700]]
    ctx.kv_free_dev(c.id, ints(gone))
    c.m.free(gone)
    k.copy_(torch.randn_like(k))
    c.m.k = wide(k)
    ctx.kv_compact_dev(c.id)
    c.m.compact()
    c.same()
    full = [s for s in range(n_seq) if c.m.length[s]][:300]
    ctx.kv_fork_dev(c.id, ints(full * 2), ints(gone[:600]))
    c.m.fork(full * 2, gone[:600])
    seqs = gone[:600] + full
    ctx.kv_extend_dev(c.id, ints(seqs), ints([1] * 900))
    c.m.extend(seqs, [1] * 900)
    c.same()


def test_errors_the_device_reports(ctx):
    from kestrel_b200.cuda import KestrelCudaError

    def reported(code, text):
        with pytest.raises(KestrelCudaError, match=text) as e:
            ctx.sync()
        assert e.value.code == code
        ctx.sync()  # told once

    c = Cache(ctx, [20, 0, 33, 0], 16, 1, 16, F16, poison=False)
    for src, dst in (([0], [2]), ([0, 0], [1, 0]), ([0], [0]), ([9], [1]), ([0], [-1])):
        ctx.kv_fork_dev(c.id, ints(src), ints(dst))
        reported(1, "paged cache")
    ctx.kv_fork_dev(c.id, ints([0, 2]), ints([1, 1]))  # the first pair is good
    reported(1, "given twice")
    c.m.fork([0], [1])
    c.same()
    ctx.kv_extend_dev(c.id, ints([0, 0]), ints([1, 1]))
    reported(1, "given twice")
    ctx.kv_extend_dev(c.id, ints([0, 7]), ints([1, 1]))
    reported(1, "out of range")
    ctx.kv_extend_dev(c.id, ints([0, 2]), ints([1, -1]))
    reported(1, "negative count")
    ctx.kv_extend_dev(c.id, ints([0, 2]), ints([1, 60]))
    reported(2, "more positions")
    ctx.kv_extend_dev(c.id, ints([0, 2, 3]), ints([28, 28, 64]))
    reported(8, "free pages")
    c.same()
    ctx.kv_free_dev(c.id, ints([2, 2]))
    reported(1, "given twice")
    c.m.free([2])
    c.same()
    x = torch.zeros((2, 1, 16), dtype=F16, device="cuda")
    ctx.kv_write_dev(c.id, 0, x, x, seqs=ints([2]), row_start=ints([0, 2]))  # an empty sequence
    reported(1, "more rows than positions")
    ctx.kv_write_dev(c.id, 0, x, x, seqs=ints([0, 8]))
    reported(1, "out of range")
    c.m.k[0, c.m.table[0][1], :, 3] = 0
    c.m.v[0, c.m.table[0][1], :, 3] = 0
    c.same()
    q = torch.ones((2, 2, 16), dtype=F16, device="cuda")
    out = torch.zeros_like(q)
    ctx.attn_decode_dev(c.id, 0, q, out, seqs=ints([0, 8]))
    reported(1, "out of range")
    ctx.attn_prompt_dev(c.id, 0, q, ints([0, 2, 1]), out)
    reported(1, "rows that do not ascend")
    ctx.attn_prompt_dev(c.id, 0, q, ints([0, 3]), out)
    reported(1, "rows that do not ascend")
    c.table[0, 0] = c.m.n_pages  # a table entry outside the pool
    ctx.attn_decode_dev(c.id, 0, q[:1], out[:1])
    reported(1, "table entry")
    ctx.attn_prompt_dev(c.id, 0, q, ints([0, 2]), out)
    reported(1, "table entry")


def test_refusals(ctx):
    from kestrel_b200.cuda import KestrelCudaError
    from kestrel_b200 import cuda
    lib = cuda.lib()
    c = Cache(ctx, [20], 16, 2, 16, F16)

    def refused(code, rc):
        assert rc == code, (rc, lib.kc_last_error(ctx.h))
        assert lib.kc_last_error(ctx.h)

    p = c.k.data_ptr()
    i = c.table.data_ptr()
    reg = lambda t=1, layers=1, pages=2, page=16, nkv=1, hd=16, n_seq=1, width=2, k=p, table=i, id=999: \
        lib.kc_kv_cache(ctx.h, id, t, layers, pages, page, nkv, hd, n_seq, width, k, p, table, i, i)
    refused(3, reg(t=0))
    refused(3, reg(t=8))
    for page in (0, 8, 24, 512):
        refused(2, reg(page=page))
    for hd in (0, 12, 264):
        refused(2, reg(hd=hd))
    refused(2, reg(layers=0))
    refused(2, reg(width=1 << 28))
    refused(2, reg(n_seq=1 << 20, width=1 << 12))
    refused(1, reg(k=None))
    refused(1, reg(k=p + 2))
    refused(1, reg(id=-1))
    refused(7, lib.kc_kv_drop(ctx.h, 999))
    refused(7, lib.kc_kv_compact_dev(ctx.h, 999, None))
    q = torch.zeros((1, 4, 16), dtype=F16, device="cuda")
    dec = lambda layer=0, n=1, nh=4, t=1, qp=q.data_ptr(), stride=64, window=0, sinks=0, scale=1.0: \
        lib.kc_attn_decode_dev(ctx.h, c.id, layer, None, n, nh, t, qp, stride, scale, window, sinks, q.data_ptr(), 64)
    refused(1, dec(layer=2))
    refused(1, dec(n=2))
    refused(2, dec(nh=3))
    refused(2, dec(nh=258))
    refused(3, dec(t=30))
    refused(2, dec(stride=63))
    refused(1, dec(window=-1))
    refused(1, dec(sinks=-1))
    refused(1, dec(scale=float("nan")))
    refused(1, dec(qp=None))
    refused(1, dec(qp=q.data_ptr() + 1))
    refused(1, lib.kc_attn_prompt_dev(ctx.h, c.id, 0, None, None, 1, 1, 4, 1, q.data_ptr(), 64, 1.0, 0, 0,
                                      q.data_ptr(), 64))
    refused(1, lib.kc_kv_extend_dev(ctx.h, c.id, None, i, 2))
    refused(1, lib.kc_kv_write_dev(ctx.h, c.id, 0, None, None, 1, 2, 1, p, p, 32, 32))
    refused(3, lib.kc_kv_write_dev(ctx.h, c.id, 0, None, None, 1, 1, 30, p, p, 32, 32))
    refused(2, lib.kc_kv_write_dev(ctx.h, c.id, 0, None, None, 1, 1, 1, p, p, 31, 32))
    assert lib.kc_attn_decode_dev(ctx.h, c.id, 0, None, 0, 4, 1, None, 64, 1.0, 0, 0, None, 64) == 0
    with pytest.raises(ValueError, match="contiguous"):
        ctx.attn_decode_dev(c.id, 0, q.expand(1, 4, 16).transpose(1, 2).contiguous().transpose(1, 2), q)
    with pytest.raises(ValueError, match="shape and type"):
        ctx.attn_decode_dev(c.id, 0, q, q.float())
    ctx.kv_drop(c.id)
    with pytest.raises(KestrelCudaError):
        ctx.kv_compact_dev(c.id)


def test_graph_of_decode_steps(ctx):
    """Extend, write and attend captured once and replayed: the lengths the
    kernels read are those of the replay."""
    from kestrel_b200.cuda import Context
    c2 = Context(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c2.set_stream(s.cuda_stream)
        c = Cache(c2, [30, 15], 16, 2, 64, F16, spare=12, poison=False, max_pages=8)
        g = torch.Generator(device="cuda").manual_seed(2)
        k, v = (torch.randn((2, 2, 64), generator=g, device="cuda") for _ in range(2))
        q = torch.randn((2, 4, 64), generator=g, device="cuda")
        out, one = torch.empty_like(q), ints([1, 1])

        def step():
            c2.kv_extend_dev(c.id, None, one)
            c2.kv_write_dev(c.id, 0, k, v)
            c2.attn_decode_dev(c.id, 0, q, out)

        step()
        c2.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
        for _ in range(20):
            graph.replay()
        c2.sync()
        for _ in range(21):
            c.m.extend([0, 1], [1, 1])
            c.m.write(0, [0, 1], [1, 1], wide(k.half()), wide(v.half()))
        c.same()
        close(wide(out), c.expected(0, wide(q), [0, 1], [1, 1], 0.125, 0, 0), F32)
        del graph
    torch.cuda.current_stream().wait_stream(s)
    c2.close()


def test_weights_of_many_positions(ctx):
    """A long cache whose weights are all small against one: none is lost."""
    n = 6000
    c = Cache(ctx, [n], 64, 1, 64, F16, poison=False)
    c.k.zero_()
    c.k[0, int(c.table[0, 0]), 0, 0, 0] = 8  # position 0 outweighs each other one by exp(8)
    c.m.k = wide(c.k)
    q = torch.zeros((1, 2, 64), device="cuda")
    q[..., 0] = 1
    out = torch.empty_like(q)
    ctx.attn_decode_dev(c.id, 0, q, out, scale=1.0)
    ctx.sync()
    close(wide(out), c.expected(0, wide(q), [0], [1], 1.0, 0, 0), F32)
    q, out = q.repeat(40, 1, 1), out.repeat(40, 1, 1)
    ctx.attn_prompt_dev(c.id, 0, q, ints([0, 40]), out, scale=1.0)
    ctx.sync()
    close(wide(out), c.expected(0, wide(q), [0], [40], 1.0, 0, 0), F32)


def test_offsets_past_32_bits(ctx):
    """Pools of more than 2^31 elements, with the sequence's pages at their end:
    every call addresses them."""
    page, n_kv, hd = 256, 8, 128
    n_pages = (1 << 31) // (page * n_kv * hd) + 40
    k, v = (torch.empty((1, n_pages, n_kv, page, hd), dtype=F16, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(1)
    n = 900
    ids = [n_pages - 1, n_pages - 30, n_pages - 2, n_pages - 29]
    table = torch.full((2, 5), -1, dtype=torch.int32, device="cuda")
    table[0, :4] = ints(ids)
    length, refs = ints([n - 1, 0]), torch.ones(n_pages, dtype=torch.int32, device="cuda")
    refs[n_pages - 5:n_pages - 2] = 0
    ctx.kv_cache(9999, k, v, table, length, refs)
    rows_k, rows_v = (torch.randn((n, n_kv, hd), generator=g, device="cuda", dtype=F16) for _ in range(2))
    ctx.kv_write_dev(9999, 0, rows_k[:n - 1], rows_v[:n - 1], row_start=ints([0, n - 1]))
    ctx.kv_fork_dev(9999, ints([0]), ints([1]))
    ctx.kv_extend_dev(9999, ints([1]), ints([1]))  # copies the last page into the pool's last free ones
    ctx.kv_write_dev(9999, 0, rows_k[n - 1:], rows_v[n - 1:], seqs=ints([1]))
    ctx.sync()
    assert table[1].tolist() == ids[:3] + [n_pages - 5, -1] and length.tolist() == [n - 1, n]
    for heads, t in (((16, 8), F32), ((8, 8), F16)):
        q = queries(40, heads[0], hd, t, 2)
        want = attention(wide(q), wide(rows_k), wide(rows_v), n - 40, hd ** -0.5)
        out = torch.empty_like(q.contiguous())
        ctx.attn_prompt_dev(9999, 0, q, ints([0, 40]), out, seqs=ints([1]))
        one = torch.empty_like(out[:1])
        ctx.attn_decode_dev(9999, 0, q[39:], one, seqs=ints([1]))
        ctx.sync()
        close(wide(out), want, t)
        close(wide(one), want[39:], t)
    ctx.kv_drop(9999)


@pytest.mark.parametrize("args", [dict(), dict(window=100, sinks=4, page=16, prompt=500, chunk=130),
                                  dict(sequences=1, branches=5, prompt=40, steps=6)], ids=str)
def test_example(args):
    """kestrel_b200.paged_example: the operators as a server calls them. The two
    kernels' f32 results differ by at most twice an f32 result's tolerance."""
    from kestrel_b200 import paged_example
    got = paged_example.run(**args)
    assert got["finite"] and got["same_after_compaction"]
    assert got["kernels_differ"] <= 2 * TOL[F32]
    assert got["pages_live"] < got["pages_without_sharing"]
    assert got["pages_after_compaction"] < got["pages_live"]
