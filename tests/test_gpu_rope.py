"""Rotary positions, alone and on the way into the pages, against the formulas
(run with -m gpu).

Tolerance, fixed before the first run. With u = 2^-24, a value gain (a cos - b
sin) is off by: the angle's rest within an eighth of a turn rounded to f32, u of
at most pi / 4; sincospif, a unit in the last place or two, 4 u; the gain rounded,
and the product with it, 2 u; then a rounded product and a fused sum, 2 u of at
most |a| + |b| times the gain. That is below 10 u |gain| (|a| + |b|). A result of a
16-bit type is rounded once more: eps / 2 of it, and of a subnormal f16 half of
2^-24. Values that do not turn are converted, at most.
"""
import numpy as np
import pytest

from rope_model import turn
from test_gpu_paged import Cache, F32, F16, BF16, PAIRS, ints, wide

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
HALF_STEP = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}
PLAIN = dict(base=10000.0)
HOWS = [PLAIN, dict(base=1e6, scaling="linear", factor=4.0),
        dict(base=1e6, scaling="yarn", factor=8.0, original=4096, low=1.0, high=32.0),
        dict(base=5e5, scaling="bands", factor=8.0, original=8192, low=1.0, high=4.0),
        dict(base=1e4, scaling="yarn", factor=2.5, original=2048, low=2.0, high=16.0, gain=-0.7)]
IDS = iter(range(1000, 1 << 30))


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from kestrel_b200.cuda import Context
    c = Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def register(ctx, dim, layout, how):
    rope = next(IDS)
    ctx.rope(rope, dim, layout=layout, **how)
    return rope


def near(got, want, size, t):
    want, size = want.astype(np.float64), size.astype(np.float64)
    room = 10 * U * size + HALF_STEP[t] * (np.abs(want) + 10 * U * size) + (2.0 ** -25 if t == F16 else 0.0)
    over = np.abs(got.astype(np.float64) - want) - room
    assert got.shape == want.shape and (over <= 0).all(), over.max()


def rows_of(rows, heads, hd, t, pad, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.randn((rows, heads * hd + 2 * pad), generator=g, device="cuda").to(t)
    return buf, buf[:, pad:pad + heads * hd].unflatten(1, (heads, hd))


def places(rows, seed, reach=1 << 17):
    p = np.random.default_rng(seed).integers(-reach, reach, rows).astype(np.int32)
    p[:8] = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, reach, 4095, 12345678][:min(8, rows)]
    return p


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope(ctx, layout, t):
    """Head sizes and parts of them that are no multiple of 8, 4 or 16; rows from
    slices of wider ones, at offsets of one value."""
    for n, (rows, heads, hd, dim, pad) in enumerate(((1, 1, 64, 64, 0), (37, 10, 64, 64, 8), (5, 3, 128, 64, 0),
                                                     (9, 7, 128, 68, 1), (130, 2, 80, 44, 2), (4, 5, 6, 6, 0),
                                                     (3, 4, 10, 2, 3), (64, 36, 128, 128, 128), (2, 1, 256, 256, 4),
                                                     (11, 3, 96, 48, 1), (6, 2, 200, 104, 0))):
        how = HOWS[n % len(HOWS)]
        buf, x = rows_of(rows, heads, hd, t, pad, n)
        keep, at = buf.clone(), places(rows, n)
        want, size = turn(wide(x), at, dim, layout, **how)
        rope = register(ctx, dim, layout, how)
        out_buf, out = rows_of(rows, heads, hd, t, (3 * pad) % 7, 99)
        edge = out_buf.clone()
        ctx.rope_dev(rope, x, ints(at.tolist()), out)
        ctx.sync()
        near(wide(out), want, size, t)
        assert torch.equal(buf, keep)  # the input, and what lies around the output
        o = (3 * pad) % 7
        assert torch.equal(out_buf[:, :o], edge[:, :o])
        assert torch.equal(out_buf[:, o + heads * hd:], edge[:, o + heads * hd:])
        ctx.rope_dev(rope, x, ints(at.tolist()))  # in place: the same bits, nothing around them
        ctx.sync()
        assert torch.equal(x, out)
        assert torch.equal(buf[:, :pad], keep[:, :pad])
        assert torch.equal(buf[:, pad + heads * hd:], keep[:, pad + heads * hd:])


@pytest.mark.parametrize("how", HOWS, ids=lambda h: h.get("scaling", "none") + ("-gain" if "gain" in h else ""))
def test_rope_many_rows_and_far_positions(ctx, how):
    """Rows enough for several heads a thread; positions to the ends of int32."""
    at = np.random.default_rng(3).integers(-2 ** 31, 2 ** 31, 3000).astype(np.int32)
    for layout, dim in (("half", 128), ("interleaved", 96)):
        _, x = rows_of(3000, 19, 128, F32, 0, 5)
        out = torch.empty((3000, 19, 128), device="cuda")
        ctx.rope_dev(register(ctx, dim, layout, how), x, ints(at.tolist()), out)
        ctx.sync()
        some = np.arange(0, 3000, 53)
        want, size = turn(wide(x)[some], at[some], dim, layout, **how)
        near(wide(out)[some], want, size, F32)


def test_rope_factors_and_nothing_to_do(ctx):
    ff = np.linspace(0.5, 9.0, 32).astype(np.float32)
    rope = next(IDS)
    ctx.rope(rope, 64, freq_factors=ff, base=1e4)
    _, x = rows_of(20, 2, 64, F32, 0, 1)
    at = places(20, 2)
    want, size = turn(wide(x), at, 64, "half", base=1e4, freq_factors=ff)
    ctx.rope_dev(rope, x, ints(at.tolist()))
    ctx.sync()
    near(wide(x), want, size, F32)
    ctx.rope_dev(rope, x[:0], ints([]))
    ctx.sync()
    x = torch.full((1, 1, 64), float("inf"), device="cuda")
    x[..., 5] = float("nan")
    ctx.rope_dev(rope, x, ints([3]))
    ctx.sync()
    ok = torch.ones(64, dtype=torch.bool)
    assert not torch.isfinite(x[0, 0].cpu()[ok]).any()


def test_refusals(ctx):
    from kestrel_b200.cuda import KestrelCudaError
    for bad, code in ((dict(dim=63), 2), (dict(dim=0), 2), (dict(dim=258), 2), (dict(dim=64, base=0.0), 1),
                      (dict(dim=64, base=float("nan")), 1), (dict(dim=64, scaling="linear", factor=0.0), 1),
                      (dict(dim=64, scaling="yarn", factor=2.0), 1), (dict(dim=64, gain=float("inf")), 1),
                      (dict(dim=64, scaling="bands", factor=2.0, original=99, low=4.0, high=4.0), 1),
                      (dict(dim=64, scaling="yarn", factor=2.0, original=99, low=1.0, high=9.0, base=1.0), 1),
                      (dict(dim=4, freq_factors=[1.0, -1.0]), 1), (dict(dim=4, freq_factors=[0.2, 1.0]), 1),
                      (dict(dim=64, base=1e-3), 1)):
        with pytest.raises(KestrelCudaError) as e:
            ctx.rope(7, **bad)
        assert e.value.code == code
    with pytest.raises(KestrelCudaError):
        ctx.rope(-1, 64)
    _, x = rows_of(4, 2, 64, F32, 0, 0)
    at = ints([0, 1, 2, 3])
    with pytest.raises(KestrelCudaError) as e:
        ctx.rope_dev(7, x, at)
    assert e.value.code == 7
    ctx.rope(7, 80)
    with pytest.raises(KestrelCudaError) as e:  # more than the head
        ctx.rope_dev(7, x, at)
    assert e.value.code == 2
    ctx.rope(7, 64)
    wide_rows = torch.zeros((4, 5, 64), device="cuda")
    with pytest.raises(KestrelCudaError, match="overlaps"):
        ctx.rope_dev(7, wide_rows[:, :3], at, wide_rows[:, 2:])
    ctx.rope_dev(7, wide_rows[:, :2], at, wide_rows[:, 2:4])  # side by side
    with pytest.raises(ValueError):
        ctx.rope_dev(7, x, at[:3])
    with pytest.raises(ValueError):
        ctx.rope_dev(7, x, at, x.half())
    ctx.sync()


def fused(rows, nq, nkv, hd, t, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, nq + 2 * nkv, hd), generator=g, device="cuda").to(t)
    return x.split([nq, nkv, nkv], 1)


APPEND = [((8, 2, 64), 64, "interleaved"), ((32, 4, 128), 128, "half"), ((6, 3, 80), 44, "half"),
          ((4, 4, 8), 8, "half"), ((5, 1, 256), 130, "interleaved"), ((3, 1, 200), 198, "half")]


@pytest.mark.parametrize("pair", PAIRS + [(F32, BF16)], ids=lambda p: f"{p[0]}-{p[1]}".replace("torch.", ""))
@pytest.mark.parametrize("heads,dim,layout", APPEND, ids=str)
def test_append(ctx, heads, dim, layout, pair):
    """Ragged rows of several sequences, and one row each; every value of the
    pools that no row goes to stays, bit for bit."""
    nq, nkv, hd = heads
    t, tc = pair
    how = HOWS[nq % len(HOWS)]
    rope = register(ctx, dim, layout, how)
    lens, counts, seqs = [40, 7, 129, 16, 300], [40, 1, 0, 16, 33], [0, 1, 2, 3, 4]
    for rows, order, start in ((counts, seqs, True), ([1, 1, 1], [4, 0, 2], False)):
        c = Cache(ctx, lens, 16, nkv, hd, tc, seed=nq, poison=False)
        n = sum(rows)
        q, k, v = fused(n, nq, nkv, hd, t, 3)
        at = np.concatenate([np.arange(lens[s] - r, lens[s]) for s, r in zip(order, rows)])
        q_out = torch.full((n, nq, hd), 9.0, device="cuda", dtype=t)
        ctx.kv_append_dev(c.id, 1, rope, k, v, q=q, q_out=q_out, seqs=ints(order),
                          row_start=ints([0] + list(np.cumsum(rows))) if start else None)
        ctx.sync()
        want, size = turn(wide(q), at, dim, layout, **how)
        near(wide(q_out), want, size, t)
        want, size = turn(wide(k), at, dim, layout, **how)
        row = 0
        mine = torch.zeros(c.k.shape[1:4:2], dtype=torch.bool)
        before = c.m.k
        got = np.empty((n, nkv, hd), np.float32)
        for s, r in zip(order, rows):
            for p in range(lens[s] - r, lens[s]):
                page = c.m.table[s][p // 16]
                got[row] = wide(c.k[1, page, :, p % 16])
                assert torch.equal(c.v[1, page, :, p % 16], v[row].to(tc))
                mine[page, p % 16] = True
                row += 1
        near(got, want, size, tc)
        left = ~mine.numpy()[:, None, :, None] & np.ones(before.shape[1:], bool)
        assert (wide(c.k)[1][left] == before[1][left]).all() and (wide(c.k)[0] == before[0]).all()
        assert (wide(c.v)[1][left] == c.m.v[1][left]).all() and (wide(c.v)[0] == c.m.v[0]).all()


def test_append_is_rope_then_write(ctx):
    """The same bits as the rotation alone, then the write; queries in place, and
    none; captured and replayed."""
    how = HOWS[2]
    rope = register(ctx, 128, "half", how)
    lens = [257, 1000, 31]
    a, b = (Cache(ctx, lens, 32, 4, 128, BF16, seed=8, poison=False) for _ in range(2))
    counts = [257, 400, 5]
    start = ints([0] + list(np.cumsum(counts)))
    q, k, v = fused(sum(counts), 12, 4, 128, BF16, 4)
    at = ints(np.concatenate([np.arange(n - r, n) for n, r in zip(lens, counts)]).tolist())
    k2, q2 = torch.empty(k.shape, dtype=BF16, device="cuda"), torch.empty(q.shape, dtype=BF16, device="cuda")
    ctx.rope_dev(rope, k, at, k2)
    ctx.rope_dev(rope, q, at, q2)
    ctx.kv_write_dev(a.id, 0, k2, v, row_start=start)
    ctx.kv_append_dev(b.id, 0, rope, k, v, row_start=start)
    ctx.sync()
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    b.k.zero_()
    b.v.zero_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx.set_stream(stream.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ctx.kv_append_dev(b.id, 0, rope, k, v, q=q, row_start=start)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    graph.replay()
    ctx.sync()
    assert torch.equal(q, q2)
    for s, (n, r) in enumerate(zip(lens, counts)):
        for p in range(n - r, n):
            page = a.m.table[s][p // 32]
            assert torch.equal(a.k[0, page, :, p % 32], b.k[0, page, :, p % 32])
            assert torch.equal(a.v[0, page, :, p % 32], b.v[0, page, :, p % 32])


def test_append_leaves_out_and_reports(ctx):
    from kestrel_b200.cuda import KestrelCudaError
    rope = register(ctx, 64, "half", PLAIN)
    c = Cache(ctx, [20, 3, 40], 16, 2, 64, F16, poison=False)
    k0 = c.k.clone()

    def call(n, seqs, start, code=1, rows=None):
        q, k, v = fused(n, 4, 2, 64, F32, 1)
        q_out = torch.full((n, 4, 64), 9.0, device="cuda")
        ctx.kv_append_dev(c.id, 0, rope, k, v, q=q, q_out=q_out, seqs=seqs, row_start=start)
        with pytest.raises(KestrelCudaError) as e:
            ctx.sync()
        assert e.value.code == code
        return (q_out == 9.0).all((1, 2)).tolist()

    assert call(2, ints([7, 1]), None) == [True, False]        # no such sequence
    assert call(2, ints([-1, 1]), None) == [True, False]
    assert call(5, ints([1, 0]), ints([0, 4, 5]), 1) == [True, False, False, False, False]  # a row before position 0
    assert call(4, ints([1, 0]), ints([1, 2, 3])) == [True, False, False, True]  # rows of no entry
    assert call(2, ints([1, 1]), None) == [False, False]       # given twice
    c.table[2, 2] = 99                                          # outside the pool: the query is turned
    c.k.copy_(k0)
    assert call(1, ints([2]), None) == [False]
    assert torch.equal(c.k, k0)
    q, k, v = fused(2, 4, 2, 64, F32, 1)
    for bad, code in ((lambda: ctx.kv_append_dev(c.id, 0, 5, k, v), 7), (lambda: ctx.kv_append_dev(c.id, 2, rope, k, v), 1),
                      (lambda: ctx.kv_append_dev(c.id, 0, rope, k.bfloat16(), v.bfloat16()), 3),
                      (lambda: ctx.kv_append_dev(c.id, 0, register(ctx, 96, "half", PLAIN), k, v), 2),
                      (lambda: ctx.kv_append_dev(c.id, 0, rope, k, v, q=k, q_out=v), 1)):
        with pytest.raises(KestrelCudaError) as e:
            bad()
        assert e.value.code == code
    for bad in (lambda: ctx.kv_append_dev(c.id, 0, rope, k, v[:1]), lambda: ctx.kv_append_dev(c.id, 0, rope, k, v, q_out=q),
                lambda: ctx.kv_append_dev(c.id, 0, rope, k, v, q=q.half())):
        with pytest.raises(ValueError):
            bad()
    ctx.sync()
