"""f32-grade sums however long the cache is (run with -m gpu).

What accumulates on the tensor cores loses a little of the sum per step, always
towards zero: values with a mean of 1 show it, since nothing cancels. The bound on
the 2-norm of a call's f32 error relative to the result's: 192 such steps at
most, at 2^-24.5 of the result each, 8e-6, queries and weights good to 2^-22 each
and f32 sums of few 2^-24, together below 1e-5. For 16-bit results the rounding of
the result and, where they are 16-bit, of the weights: 2 u as in
test_gpu_paged_paths, where u is the type's unit roundoff, and the loss towards
zero of up to 2048 steps at 2^-24, 1.2e-4.
"""
import pytest

from test_gpu_paged import BF16, F16, F32, ctx, ints, torch  # noqa: F401

pytestmark = pytest.mark.gpu
BOUND = {F32: 1e-5, F16: 2.0 ** -10 + 1.3e-4, BF16: 2.0 ** -7 + 1.3e-4}


class Shared:
    """n_seq sequences of n positions that all hold the same pages."""

    def __init__(self, ctx, n_seq, n, n_kv, hd, t, mean, page=256):
        w = -(-n // page)
        g = torch.Generator(device="cuda").manual_seed(n)
        shape = (1, w, n_kv, page, hd)
        self.k = torch.randn(shape, generator=g, device="cuda").to(t)
        self.v = (torch.randn(shape, generator=g, device="cuda") + mean).to(t)
        self.n, self.hd = n, hd
        self.table = torch.arange(w, dtype=torch.int32, device="cuda").repeat(n_seq, 1)
        self.length = torch.full((n_seq,), n, dtype=torch.int32, device="cuda")
        self.refs = torch.full((w,), n_seq, dtype=torch.int32, device="cuda")
        ctx.kv_cache(7000, self.k, self.v, self.table, self.length, self.refs)

    def error(self, got, q, group):
        """Relative 2-norm of the error of the last rows (one sequence's): every
        key-value head."""
        rows, off, size = q.shape[0], 0.0, 0.0
        hidden = torch.arange(self.n, device="cuda") > torch.arange(self.n - rows, self.n, device="cuda")[:, None, None]
        for h in range(self.k.shape[2]):
            k, v = (x[0, :, h].reshape(-1, self.hd)[:self.n].double() for x in (self.k, self.v))
            heads = slice(h * group, (h + 1) * group)
            score = torch.einsum("rhd,jd->rhj", q[:, heads].double(), k) * self.hd ** -0.5
            want = torch.softmax(score.masked_fill_(hidden, float("-inf")), -1) @ v
            off += float((got[:, heads].double() - want).square().sum())
            size += float(want.square().sum())
        return (off / size) ** 0.5


def queries(rows, nh, hd, t):
    g = torch.Generator(device="cuda").manual_seed(rows)
    return (1.5 * torch.randn((rows, nh, hd), generator=g, device="cuda")).to(t)


@pytest.mark.parametrize("mean", [0.0, 1.0])
@pytest.mark.parametrize("types", [(F32, F16), (F16, F16), (BF16, BF16)], ids=str)
@pytest.mark.parametrize("heads", [(8, 1, 128), (8, 2, 64), (40, 2, 96), (4, 1, 256)], ids=str)
def test_decode_of_long_batches(ctx, heads, types, mean):
    """Hundreds of chunks of one sequence and head to a warp."""
    nh, nkv, hd = heads
    c = Shared(ctx, 296, 32768, nkv, hd, types[1], mean)
    q = queries(296, nh, hd, types[0])
    out = torch.empty_like(q)
    ctx.attn_decode_dev(7000, 0, q, out)
    ctx.sync()
    for s in (0, 100, 295):
        assert c.error(out[s:s + 1], q[s:s + 1], nh // nkv) <= BOUND[types[0]]
    ctx.kv_drop(7000)


@pytest.mark.parametrize("mean", [0.0, 1.0])
@pytest.mark.parametrize("types", [(F32, F16), (F16, F16), (BF16, BF16)], ids=str)
@pytest.mark.parametrize("heads,rows,n", [((32, 4, 128), 1500, 40000), ((8, 2, 64), 40, 70000),
                                          ((16, 2, 64), 5000, 20000), ((12, 3, 96), 2000, 33001),
                                          ((8, 2, 256), 1300, 20000), ((6, 2, 200), 33, 50000)], ids=str)
def test_prompts_over_long_caches(ctx, heads, rows, n, types, mean):
    """Items of one and two row tiles, of two streams and of one, whole and split
    over their positions."""
    nh, nkv, hd = heads
    c = Shared(ctx, 1, n, nkv, hd, types[1], mean)
    q = queries(rows, nh, hd, types[0])
    outs = [torch.empty_like(q) for _ in range(2)]
    for out in outs:
        ctx.attn_prompt_dev(7000, 0, q, ints([0, rows]), out)
    ctx.sync()
    assert torch.equal(*outs)
    assert c.error(outs[0][-32:], q[-32:], nh // nkv) <= BOUND[types[0]]
    ctx.kv_drop(7000)


@pytest.mark.parametrize("types", [(F32, F16), (F16, F16), (BF16, BF16)], ids=str)
@pytest.mark.parametrize("rise", [3.0, -3.0])
def test_long_caches_of_rising_scores(ctx, types, rise):
    """Scores that rise (or fall) by 3 every 2000 positions: the sums kept of the
    tiles before count the less (or all) beside those that follow. Scores of up to
    60 add 8 steps of 2^-23 of themselves to the bound."""
    n, rows, nh, nkv, hd = 40000, 1200, 8, 2, 128
    c = Shared(ctx, 1, n, nkv, hd, types[1], 1.0)
    pages = torch.arange(c.k.shape[1] * 256, device="cuda").view(-1, 1, 256)
    c.k[0, :, :, :, 7] = (pages // 2000 * rise).to(types[1])
    q = queries(rows, nh, hd, F32)
    q[..., 7] = hd ** 0.5
    q = q.to(types[0])
    out = torch.empty_like(q)
    ctx.attn_prompt_dev(7000, 0, q, ints([0, rows]), out)
    ctx.sync()
    assert c.error(out[-32:], q[-32:], nh // nkv) <= BOUND[types[0]] + 8 * 2.0 ** -23 * 60
    ctx.kv_drop(7000)
