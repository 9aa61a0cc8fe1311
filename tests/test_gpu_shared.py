"""Attention over shared prefixes against plain models (run with -m gpu).

Tolerances are those of the two kernels that it joins (test_gpu_paged.py): with u
the unit roundoff of a 16-bit type, 2 u max|v| for its results; 2^-15 max|v| for
f32 ones. The join is a mean of the parts' results with f32 weights, which adds a
few 2^-24 of the same.
"""
import numpy as np
import pytest

from test_gpu_paged import BF16, F16, F32, HEADS, PAIRS, Cache, close, ints, queries, wide

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from kestrel_b200.cuda import OPT_SHARE_ALWAYS, Context
    c = Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    c.set_option(OPT_SHARE_ALWAYS, 1)  # these sizes would not be shared for their time
    yield c
    c.close()


def branches(ctx, groups, page, nkv, hd, t, seed=0, poison=True):
    """groups: (common pages, lengths) each; sequences in that order. The first
    `common` table entries of a group are its first sequence's."""
    lens = [n for _, ls in groups for n in ls]
    c = Cache(ctx, lens, page, nkv, hd, t, seed=seed, poison=poison)
    start, at = [0], 0
    for common, ls in groups:
        for s in range(at + 1, at + len(ls)):
            for j in range(min(common, -(-ls[s - at] // page))):
                c.m.table[s][j] = c.m.table[at][j]
        at += len(ls)
        start.append(at)
    c.table.copy_(ints(c.m.table))
    return c, start


def run(ctx, c, q, start, seqs=None, scale=None, layer=1):
    out = torch.full_like(q.contiguous(), 7.0)
    ctx.attn_shared_dev(c.id, layer, q, ints(start), out, seqs=None if seqs is None else ints(seqs), scale=scale)
    ctx.sync()
    return out


def check(ctx, c, q, start, t, seqs=None, scale=None, layer=1):
    hd = q.shape[2]
    out = run(ctx, c, q, start, seqs, scale, layer)
    order = range(q.shape[0]) if seqs is None else seqs
    close(wide(out), c.expected(layer, wide(q), order, [1] * q.shape[0], hd ** -0.5 if scale is None else scale, 0, 0), t)
    return out


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: f"{p[0]}-{p[1]}".replace("torch.", ""))
def test_groups(ctx, heads, pair):
    """Prefixes of a part of a tile to several, groups of one and of more rows than
    a tile holds, sequences that end just behind the prefix, empty ones among them."""
    nh, nkv, hd = heads
    for page, groups in ((16, [(5, [90, 81, 85]), (0, [40]), (9, [300, 145, 0, 160, 200]), (3, [100, 33])]),
                         (64, [(2, [129, 130, 300, 200, 128]), (4, [257, 257])]),
                         (32, [(8, [256 + 1 + i for i in range(20)]), (20, [700, 650])])):
        c, start = branches(ctx, groups, page, nkv, hd, pair[1], seed=nh + page)
        q = queries(start[-1], nh, hd, pair[0], 5)
        check(ctx, c, q, start, pair[0])


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: f"{p[0]}-{p[1]}".replace("torch.", ""))
def test_long_prefixes(ctx, pair):
    """Prefixes split over many blocks, own parts from one position to thousands."""
    for (nh, nkv, hd), groups in (((8, 1, 128), [(128, [8200, 8193, 9000, 12000])]), ((4, 2, 64), [(70, [4500] * 3), (64, [4097] * 2)]),
                                  ((32, 2, 80), [(40, [2561 + 40 * i for i in range(9)])]), ((2, 1, 256), [(60, [3900, 4000])])):
        c, start = branches(ctx, groups, 64, nkv, hd, pair[1], seed=nh)
        q = queries(start[-1], nh, hd, pair[0], 8)
        out = check(ctx, c, q, start, pair[0], layer=0)
        again = run(ctx, c, q, start, layer=0)
        assert torch.equal(out, again)  # the same bits
        alone = torch.empty_like(out)
        ctx.attn_decode_dev(c.id, 0, q, alone)
        ctx.sync()
        off = (alone.double() - out.double()).norm() / alone.double().norm()
        assert off < {F32: 1e-5, F16: 2.0 ** -10, BF16: 2.0 ** -7}[pair[0]]


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: f"{p[0]}-{p[1]}".replace("torch.", ""))
def test_many_entries(ctx, pair):
    """More groups than the finder sorts, and more rows than the workspace takes at
    a time: several launches."""
    groups = [(5, [81 + (i * 7 + j) % 20 for j in range(1 + i % 5)]) for i in range(60)]
    c, start = branches(ctx, groups, 16, 2, 64, pair[1], seed=3)
    q = queries(start[-1], 8, 64, pair[0], 4)
    check(ctx, c, q, start, pair[0])
    c, start = branches(ctx, [(6, [97 + i % 3 for i in range(300)]), (4, [70] * 50)], 16, 1, 256, pair[1], seed=4)
    q = queries(start[-1], 64, 256, pair[0], 4)  # 350 entries of 66 KB
    check(ctx, c, q, start, pair[0])


def test_what_is_common_is_looked_up(ctx):
    """Groups whose tables part early, in the middle or never; what is claimed does
    not matter: another order, overlapping requests, the same sequence twice."""
    c, start = branches(ctx, [(20, [400, 390, 380, 321])], 16, 2, 64, F16, seed=9, poison=False)
    c.m.table[2][7] = c.m.table[0][30 - 7]  # parts at page 7 (any other page of the pool)
    c.m.table[3][0] = c.m.table[1][24]
    c.table.copy_(ints(c.m.table))
    q = queries(4, 4, 64, F32, 1)
    for seqs, groups in ((None, [0, 4]), (None, [0, 2, 4]), ([3, 2, 1, 0], [0, 1, 4]), ([1, 1, 0, 0], [0, 4]), (None, [0, 0, 3, 3]),
                         (None, [1, 3]), (None, [0, 1, 2, 3, 4])):
        check(ctx, c, q, groups, F32, seqs=seqs)
    check(ctx, c, q, [0, 4], F32, scale=-0.2)
    check(ctx, c, q, [0, 4], F32, scale=0.0)
    one, start = branches(ctx, [(8, [129, 129])], 16, 2, 64, F16)
    one.m.length[1] = 128  # ends with the prefix: a page less is common
    one.length[1] = 128
    check(ctx, one, queries(2, 4, 64, F32, 2), [0, 2], F32)


def test_after_fork_and_extend(ctx):
    """The pages as the cache's own calls leave them."""
    c = Cache(ctx, [200, 0, 0, 0], 16, 2, 64, F16, spare=12, max_pages=20)
    kids = [1, 2, 3]
    ctx.kv_fork_dev(c.id, ints([0] * 3), ints(kids))
    c.m.fork([0] * 3, kids)
    for step in range(3):
        ctx.kv_extend_dev(c.id, ints(kids), ints([7, 1, 20]))
        c.m.extend(kids, [7, 1, 20])
        n = 28
        g = torch.Generator(device="cuda").manual_seed(step)
        k, v = (torch.randn((n, 2, 64), generator=g, device="cuda").half() for _ in range(2))
        ctx.kv_write_dev(c.id, 1, k, v, seqs=ints(kids), row_start=ints([0, 7, 8, 28]))
        c.m.write(1, kids, [7, 1, 20], wide(k), wide(v))
        check(ctx, c, queries(3, 8, 64, F16, step), [0, 3], F16, seqs=kids)
        check(ctx, c, queries(4, 8, 64, F16, step), [0, 4], F16, seqs=[0] + kids)


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: f"{p[0]}-{p[1]}".replace("torch.", ""))
def test_values_at_the_ends(ctx, pair):
    """Scores that leave one position, in the prefix or behind it; infinite and NaN
    values that a row sees give what the formula gives, and only there."""
    for spot in (10, 700, 1100):  # first and second part of the prefix, own part
        c, start = branches(ctx, [(64, [1150, 1030])], 16, 1, 64, pair[1], poison=False)
        page, row = c.m.table[0][spot // 16], spot % 16
        c.k[1, page, 0, row] = 20.0
        c.m.k = wide(c.k)
        q = queries(2, 4, 64, pair[0], 3).abs().contiguous()
        check(ctx, c, q, start, pair[0])
        for bad in (float("inf"), -float("inf"), float("nan")):
            c, start = branches(ctx, [(64, [1150, 1030])], 16, 1, 64, pair[1], poison=False)
            c.v[1, page, 0, row, 5] = bad
            out = wide(run(ctx, c, q, start))
            sees = [True, spot < 1024]
            for i in range(2):
                assert (np.isnan(out[i, :, 5]).all() if bad != bad else (out[i, :, 5] == bad).all()) == sees[i]
                assert np.isfinite(np.delete(out[i], 5, 1)).all()
            c.v[1, page, 0, row, 5] = 0.0
            c.k[1, page, 0, row, 5] = float("nan")
            out = wide(run(ctx, c, q, start))
            assert [bool(np.isnan(out[i]).all()) for i in range(2)] == sees


def test_strides_rows_and_graphs(ctx):
    c, start = branches(ctx, [(9, [150, 170, 149]), (4, [70, 66])], 16, 2, 64, BF16, seed=2)
    for pad in (8, 1, 3):
        q = queries(5, 4, 64, BF16, 9, pad)
        buf = torch.full((5, 4 * 64 + 2 * pad), 7.0, device="cuda", dtype=BF16)
        out = buf[:, pad:pad + 256].unflatten(1, (4, 64))
        ctx.attn_shared_dev(c.id, 1, q, ints(start), out)
        ctx.sync()
        close(wide(out), c.expected(1, wide(q), range(5), [1] * 5, 0.125, 0, 0), BF16)
        assert (buf[:, :pad] == 7).all() and (buf[:, pad + 256:] == 7).all()
    q = queries(5, 4, 64, BF16, 11).contiguous()
    want = run(ctx, c, q, start)
    out, groups = torch.zeros_like(q), ints(start)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx.set_stream(stream.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ctx.attn_shared_dev(c.id, 1, q, groups, out)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        out.zero_()
        graph.replay()
        ctx.sync()
        assert torch.equal(out, want)
    # Longer sequences and another table: the graph looks them up again.
    c.m.length[0] = c.m.length[1] = 149
    c.length[:2] = 149
    graph.replay()
    ctx.sync()
    close(wide(out), c.expected(1, wide(q), range(5), [1] * 5, 0.125, 0, 0), BF16)


def test_by_expected_time(ctx):
    """Without the option: what is not worth it is not shared (the decode call's bits),
    what is (64 x 24000 positions, 790 MB unshared) gives the same within tolerance."""
    from kestrel_b200.cuda import OPT_SHARE_ALWAYS
    ctx.set_option(OPT_SHARE_ALWAYS, 0)
    try:
        for pages, lens, same in ((5, [90, 81, 85], True), (375, [24001 + 61 * i for i in range(64)], False)):
            c, start = branches(ctx, [(pages, lens)], 16 if same else 64, 2, 64, F16, poison=False)
            q = queries(len(lens), 8, 64, F16, 5).contiguous()
            out, alone = run(ctx, c, q, start), torch.empty_like(q)
            ctx.attn_decode_dev(c.id, 1, q, alone)
            ctx.sync()
            assert torch.equal(out, alone) == same
            assert (alone.double() - out.double()).norm() <= 2.0 ** -10 * alone.double().norm()
    finally:
        ctx.set_option(OPT_SHARE_ALWAYS, 1)


def test_reports_and_refusals(ctx):
    from kestrel_b200.cuda import KestrelCudaError
    c, start = branches(ctx, [(9, [150, 170, 149])], 16, 2, 64, F16, seed=2)
    q = queries(3, 4, 64, F16, 1)
    want = run(ctx, c, q, start)

    def reported(start, seqs=None):
        out = torch.full_like(q.contiguous(), 7.0)
        ctx.attn_shared_dev(c.id, 1, q, ints(start), out, seqs=None if seqs is None else ints(seqs))
        with pytest.raises(KestrelCudaError) as e:
            ctx.sync()
        assert e.value.code == 1
        return out

    for bad in ([0, 4], [2, 1, 3], [-1, 3], [0, 3, 2]):
        out = reported(bad)
        close(wide(out), wide(want).astype(np.float64), F16)  # nothing is shared, the results are the same
    out = reported([0, 3], [0, 9, 2])
    assert (out[1] == 7).all()
    close(wide(out)[[0, 2]], wide(want)[[0, 2]].astype(np.float64), F16)
    assert torch.equal(run(ctx, c, q, start), want)
    for bad, code in ((lambda: ctx.attn_shared_dev(c.id, 2, q, ints(start), torch.empty_like(q)), 1),
                      (lambda: ctx.attn_shared_dev(c.id, 0, q, ints([0] * 9), torch.empty_like(q)), 1),
                      (lambda: ctx.attn_shared_dev(c.id, 0, q.float(), ints(start), q.float(), scale=float("inf")), 1),
                      (lambda: ctx.attn_shared_dev(c.id, 0, q.bfloat16(), ints(start), q.bfloat16()), 3)):
        with pytest.raises(KestrelCudaError) as e:
            bad()
        assert e.value.code == code
    ctx.attn_shared_dev(c.id, 0, q[:0], ints([0]), torch.empty_like(q)[:0])
    ctx.sync()
