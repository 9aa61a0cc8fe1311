"""Calls of the paged cache and its attention that must be refused, left out or
answered as the definition says where numbers end (run with -m gpu).

Tolerances are test_gpu_paged's: with u the unit roundoff of the query / output
type, 2 u max|v| for 16-bit results and 2^-15 max|v| for f32 ones, values of
unit normal size (max|v| <= 6).
"""
import numpy as np
import pytest

from test_gpu_paged import BF16, F16, F32, PAIRS, Cache, close, ctx, ints, queries, torch, wide  # noqa: F401

pytestmark = pytest.mark.gpu


def pair_id(p):
    return f"{p[0]}-{p[1]}".replace("torch.", "")


def reported(c, code, text):
    from kestrel_b200.cuda import KestrelCudaError
    with pytest.raises(KestrelCudaError, match=text) as e:
        c.sync()
    assert e.value.code == code
    c.sync()  # told once


@pytest.mark.parametrize("pair", PAIRS, ids=pair_id)
@pytest.mark.parametrize("n", [9, 41])
def test_rows_given_to_several_entries(ctx, pair, n):
    """row_start 0, N, 0, N, ...: the first entry has the N rows, the others
    begin before it or end before they begin. Only the first is computed, and
    the context's workspace holds what it should afterwards."""
    rows = 1280
    c = Cache(ctx, [1300] + [1100] * (n - 1), 128, 1, 64, pair[1], n_layer=1, seed=n)
    q = queries(rows + 4, 1, 64, pair[0], 3)
    out = torch.full_like(q.contiguous(), 7.0)
    ctx.attn_prompt_dev(c.id, 0, q, ints([rows * (i % 2) for i in range(n + 1)]), out)
    reported(ctx, 1, "rows that do not ascend")
    want = c.expected(0, wide(q)[:rows], [0], [rows], 0.125, 0, 0)
    close(wide(out)[:rows], want, pair[0])
    assert (out[rows:] == 7).all()
    # An entry after a later one's beginning, and one that goes on in order.
    out.fill_(7)
    start = [0] * n + [0]
    start[1:4] = [40, 20, 60]
    start[4:] = [60] * (n - 3)
    ctx.attn_prompt_dev(c.id, 0, q, ints(start), out)  # entries 0: 0 .. 40, 1: 40 .. 20, 2: 20 .. 60
    reported(ctx, 1, "rows that do not ascend")
    close(wide(out)[:40], c.expected(0, wide(q)[:40], [0], [40], 0.125, 0, 0), pair[0])
    assert (out[40:] == 7).all()
    # What came after is as it was before.
    again = torch.full_like(out, 7.0)
    for o in (out, again):
        ctx.attn_prompt_dev(c.id, 0, q, ints([0] + [rows] * n), o)
        one = torch.empty_like(q[:n].contiguous())
        ctx.attn_decode_dev(c.id, 0, q[:n], one)
    ctx.sync()
    close(wide(out)[:rows], want, pair[0])
    assert torch.equal(out, again)
    close(wide(one), c.expected(0, wide(q)[:n], range(n), [1] * n, 0.125, 0, 0), pair[0])


def same_numbers(got, want, t):
    """NaN and infinities where they belong, the rest within the tolerance."""
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)].astype(got.dtype))
    close(np.where(fine, got, 0.0), np.where(fine, want, 0.0), t)


@pytest.mark.parametrize("heads", [(2, 1, 64), (8, 2, 64), (20, 1, 64), (6, 2, 40), (3, 1, 256), (16, 1, 128)], ids=str)
@pytest.mark.parametrize("pair", PAIRS, ids=pair_id)
def test_infinities_in_view(ctx, heads, pair):
    """Keys and values that hold infinities, seen by the row: a score of minus
    infinity gives no weight, one of plus infinity NaN, an infinite value an
    infinity (or NaN with no weight or beside one of the other sign). A weight
    of exp(-40) is a weight. Short sequences and ones of many parts."""
    nh, nkv, hd = heads
    lens = [40, 3000, 9, 700]
    c = Cache(ctx, lens, 16, nkv, hd, pair[1], n_layer=1, seed=nh)
    at = lambda s, j: (0, c.m.table[s][j // 16], slice(None), j % 16)
    for s, n in enumerate(lens):
        c.k[at(s, 2)][:, 5] = float("inf")       # scores of both infinities, by the head
        c.v[at(s, 3)][:, 9] = float("inf")
        c.v[at(s, 4)][:, 10] = float("-inf")
        c.v[at(s, n - 1)][:, 11] = float("inf")
        c.v[at(s, 3)][:, 11] = float("-inf")
        c.v[at(s, 2)][:, 12] = float("inf")      # where the score is minus infinity: NaN
        c.k[at(s, 6)] = 0                        # a score of -40
        c.k[at(s, 6)][:, 7] = -40
        c.v[at(s, 6)][:, 13] = float("inf")
    for s, n in enumerate(lens):
        for j in range(n):
            if j != 6:
                c.k[at(s, j)][:, 7] = 0
    c.m.k, c.m.v = wide(c.k), wide(c.v)
    q = 0.3 * queries(len(lens), nh, hd, F32, 5)
    q[..., 7] = 1
    q[:, ::2, 5] = -q[:, ::2, 5].abs() - 0.01    # these heads leave position 2 out
    q[:, 1::2, 5] = q[:, 1::2, 5].abs() + 0.01   # these come to NaN
    q = q.to(pair[0])
    with np.errstate(invalid="ignore"):
        want = c.expected(0, wide(q), range(len(lens)), [1] * len(lens), 1.0, 0, 0)
    assert np.isnan(want[:, 1::2]).all() and np.isposinf(want[:, ::2, [9, 13]]).all()
    assert np.isneginf(want[:, ::2, 10]).all() and np.isnan(want[:, ::2, 11:13]).all()
    assert np.isfinite(want[:, ::2, 14:]).all() and np.isfinite(want[:, ::2, :9]).all()
    out = torch.full_like(q, 7.0)
    ctx.attn_decode_dev(c.id, 0, q, out, scale=1.0)
    ctx.sync()
    same_numbers(wide(out), want, pair[0])
    out.fill_(7)
    ctx.attn_prompt_dev(c.id, 0, q, ints(range(len(lens) + 1)), out, scale=1.0)
    ctx.sync()
    same_numbers(wide(out), want, pair[0])


@pytest.mark.parametrize("n_kv,hd", [(1, 8), (3, 40), (4, 128)])
def test_write_to_a_sequence_given_twice(ctx, n_kv, hd):
    """It is reported; the rows of all other sequences are written, and nothing
    else is touched."""
    n_seq = 70
    lens = [40 + s for s in range(n_seq)]
    c = Cache(ctx, lens, 16, n_kv, hd, F16, n_layer=1, spare=1, poison=False)
    rng = np.random.default_rng(hd)
    for counts in (None, [int(x) for x in rng.integers(1, 40, n_seq)]):
        for n, pairs in ((n_seq, ((69, 3), (40, 39), (36, 0), (20, 3))), (5, ((4, 2),)), (2, ((1, 0),))):
            rows = (counts or [1] * n_seq)[:n]
            seqs = [int(s) for s in rng.permutation(n_seq)][:n]
            for a, b in pairs:
                seqs[a] = seqs[b]
            x = torch.randn((2, sum(rows), n_kv, hd), device="cuda")
            start = None if counts is None else ints([0] + list(np.cumsum(rows)))
            ctx.kv_write_dev(c.id, 0, x[0], x[1], seqs=ints(seqs), row_start=start)
            reported(ctx, 1, "given twice")
            at = 0
            for s, m in zip(seqs, rows):
                if seqs.count(s) == 1:
                    c.m.write(0, [s], [m], wide(x[0, at:at + m].half()), wide(x[1, at:at + m].half()))
                at += m
            # Either entry's rows: taken over into the model.
            for s in {s for s in seqs if seqs.count(s) > 1}:
                most = max(m for t, m in zip(seqs, rows) if t == s)
                for j in range(lens[s] - most, lens[s]):
                    p = c.m.table[s][j // 16]
                    c.m.k[0, p, :, j % 16] = wide(c.k[0, p, :, j % 16])
                    c.m.v[0, p, :, j % 16] = wide(c.v[0, p, :, j % 16])
            c.same()
            # The marks are clear again: each once is no error.
            once = [int(s) for s in rng.permutation(n_seq)][:n]
            ctx.kv_write_dev(c.id, 0, x[0], x[1], seqs=ints(once), row_start=start)
            c.m.write(0, once, rows, wide(x[0].half()), wide(x[1].half()))
            c.same()
            ctx.kv_extend_dev(c.id, ints(once), ints([0] * n))
            c.same()


@pytest.mark.parametrize("pair", PAIRS, ids=pair_id)
def test_rows_computed_alone_over_a_long_cache(ctx, pair):
    """An infinite value near the beginning of 160000 positions makes every row
    one that is computed by itself: that takes its time, and no wait expires."""
    n, rows, nh, hd, page = 160000, 32, 4, 64, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn((1, n // page, 1, page, hd), generator=g, device="cuda").to(pair[1]) for _ in range(2))
    v[0, 2, 0, 5, 9], v[0, 2, 0, 6, 10] = float("inf"), float("nan")
    ctx.kv_cache(9998, k, v, torch.arange(n // page, dtype=torch.int32, device="cuda")[None], ints([n]),
                 torch.ones(n // page, dtype=torch.int32, device="cuda"))
    q = queries(rows, nh, hd, pair[0], 9)
    out = torch.empty_like(q.contiguous())
    ctx.attn_prompt_dev(9998, 0, q, ints([0, rows]), out)
    ctx.sync()
    kk, vv = k.reshape(n, hd).double(), v.reshape(n, hd).double()
    score = torch.einsum("rhd,jd->rhj", q.double(), kk) * hd ** -0.5
    hidden = torch.arange(n, device="cuda") > (n - rows + torch.arange(rows, device="cuda"))[:, None, None]
    want = torch.softmax(score.masked_fill(hidden, float("-inf")), -1) @ vv
    # (The hidden positions are finite: their weight of zero adds nothing.)
    same_numbers(wide(out), want.cpu().numpy(), pair[0])
    assert torch.isinf(out[..., 9]).all() and torch.isnan(out[..., 10]).all() and torch.isfinite(out[..., 11:]).all()
    ctx.kv_drop(9998)


def arrival_counts(c):
    """The attention kernels' arrival counts in a context's workspace, as an
    int32 CUDA tensor: their place is found in the context by what surrounds it
    (parts, counts behind them, the bytes of the counts and of both)."""
    start, data = c.h.value if hasattr(c.h, "value") else c.h, b""
    with open("/proc/self/mem", "rb", 0) as mem:
        try:
            for at in range(start, start + (1 << 13), 256):
                mem.seek(at)
                data += mem.read(256)
        except OSError:  # past the heap's end
            pass
    words = np.frombuffer(data[:len(data) // 8 * 8], dtype=np.int64)
    at = [i for i in range(len(words) - 3) if words[i] and words[i + 1] > words[i] and 0 < words[i + 2] < 1 << 16 and
          words[i + 1] - words[i] + words[i + 2] == words[i + 3]]
    assert len(at) == 1
    address, size = int(words[at[0] + 1]), int(words[at[0] + 2]) // 4

    class Counts:
        __cuda_array_interface__ = {"shape": (size,), "typestr": "<i4", "data": (address, False), "version": 3}

    return torch.as_tensor(Counts(), device="cuda")


def test_counts_after_an_expired_wait(ctx):
    """What an attention call that gave up waiting leaves in the arrival counts is
    cleared with the status, so that later calls join their parts in full. (The
    counts are set here, and the status by an index out of range.)"""
    c = Cache(ctx, [3000, 2500], 64, 1, 64, F16, seed=3)
    q = queries(2 * 40, 4, 64, F32, 4)
    one = torch.empty_like(q[:2].contiguous())
    rows = torch.empty_like(q.contiguous())
    counts = arrival_counts(ctx)
    ctx.attn_decode_dev(c.id, 0, q[:2], one)
    ctx.attn_prompt_dev(c.id, 0, q, ints([0, 40, 80]), rows)
    ctx.sync()
    assert not counts.any()  # put back by the kernels
    want = one.clone(), rows.clone()
    close(wide(one), c.expected(0, wide(q[:2]), [0, 1], [1, 1], 0.125, 0, 0), F32)
    for left in (1, 3):
        counts.fill_(left)
        ctx.attn_decode_dev(c.id, 0, q[:1], one[:1], seqs=ints([99]))
        reported(ctx, 1, "out of range")
        assert not counts.any()
        one.fill_(7)
        rows.fill_(7)
        ctx.attn_decode_dev(c.id, 0, q[:2], one)
        ctx.attn_prompt_dev(c.id, 0, q, ints([0, 40, 80]), rows)
        ctx.sync()
        assert torch.equal(one, want[0]) and torch.equal(rows, want[1])


def test_rows_of_a_sequence_out_of_range(ctx):
    """Both kernels leave them as they are, and zero those of an empty one."""
    c = Cache(ctx, [70, 0, 33], 16, 1, 64, F16, seed=1)
    q = queries(5, 2, 64, F32, 2)
    out = torch.full_like(q.contiguous(), 7.0)
    ctx.attn_decode_dev(c.id, 0, q[:3], out[:3], seqs=ints([2, 3, 1]))
    reported(ctx, 1, "out of range")
    close(wide(out)[:1], c.expected(0, wide(q)[:1], [2], [1], 0.125, 0, 0), F32)
    assert (out[1] == 7).all() and (out[2] == 0).all()
    out.fill_(7)
    ctx.attn_prompt_dev(c.id, 0, q, ints([0, 2, 4, 5]), out, seqs=ints([2, -1, 1]))
    reported(ctx, 1, "out of range")
    close(wide(out)[:2], c.expected(0, wide(q)[:2], [2], [2], 0.125, 0, 0), F32)
    assert (out[2:4] == 7).all() and (out[4] == 0).all()


@pytest.mark.parametrize("pair", PAIRS, ids=pair_id)
def test_windows_and_sinks_of_any_size(ctx, pair):
    """Up to the largest int, longer than the sequence, and with more rows than
    positions (the first rows then see nothing)."""
    most = 2 ** 31 - 1
    c = Cache(ctx, [40, 200, 1, 0], 16, 1, 64, pair[1], seed=2)
    counts = [90, 200, 3, 2]
    q = queries(sum(counts), 2, 64, pair[0], 3)
    for window, sinks in ((most, 0), (most, most), (most - 5, 3), (c.table.shape[1] * 16, 1),
                          (c.table.shape[1] * 16 - 1, 1), (30, most), (1, most), (200, 300), (199, 0)):
        out = torch.full_like(q.contiguous(), 7.0)
        ctx.attn_prompt_dev(c.id, 0, q, ints([0] + list(np.cumsum(counts))), out, window=window, sinks=sinks)
        one = torch.full_like(q[:4].contiguous(), 7.0)
        ctx.attn_decode_dev(c.id, 0, q[:4], one, window=window, sinks=sinks)
        ctx.sync()
        close(wide(out), c.expected(0, wide(q), range(4), counts, 0.125, window, sinks), pair[0])
        close(wide(one), c.expected(0, wide(q)[:4], range(4), [1] * 4, 0.125, window, sinks), pair[0])


def test_write_to_thousands_of_sequences(ctx):
    """A list of more sequences than the looking block holds at a time: one given
    twice is found wherever the two are, and none where each is given once."""
    n = 2500
    k = torch.zeros((1, n, 1, 16, 8), dtype=F16, device="cuda")
    v = torch.zeros_like(k)
    table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].contiguous()
    ctx.kv_cache(9997, k, v, table, torch.ones(n, dtype=torch.int32, device="cuda"),
                 torch.ones(n, dtype=torch.int32, device="cuda"))
    x = torch.randn((2, n, 1, 8), device="cuda").half()
    order = torch.randperm(n).int()
    for a, b in ((None, None), (2499, 0), (1025, 1024), (1300, 70), (None, None)):
        seqs = order.clone()
        if a is not None:
            seqs[a] = seqs[b]
        k.zero_()
        ctx.kv_write_dev(9997, 0, x[0], x[1], seqs=seqs.cuda())
        if a is None:
            ctx.sync()
            at = order.long().cuda()
            assert torch.equal(k[0, at, :, 0], x[0]) and torch.equal(v[0, at, :, 0], x[1])
        else:
            reported(ctx, 1, "given twice")
            alone = torch.tensor([i for i in range(n) if i not in (a, b)])
            assert torch.equal(k[0, order[alone].long().cuda(), :, 0], x[0][alone.cuda()])
    ctx.kv_drop(9997)
