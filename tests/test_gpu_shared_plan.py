"""When attn_shared_dev shares, and that the choice is the same every time (run with
-m gpu). Whether it did shows in the bits: shared, 16-bit results carry the rounding of
16-bit weights, so that many of them round to a neighbour of the decode call's; not
shared, both are f32 sums in different orders (2^-20 apart at most; up to 8 heads to a
key's, whose weights keep their rests), and a result of 11 bits falls on another side
once in a few hundred times."""
import numpy as np
import pytest

from test_gpu_paged import F16, ints
from test_gpu_shared import branches, ctx, run  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def wide_tables(ctx, n, length, nkv, hd, page=64):  # noqa: F811
    """n sequences of `length` positions whose tables name the same pages but for the last."""
    pages = -(-length // page)
    k, v = (torch.randn((1, pages + n, nkv, page, hd), device="cuda").half() for _ in range(2))
    table = torch.arange(pages, device="cuda", dtype=torch.int32)[None].repeat(n, 1)
    table[:, -1] = pages + torch.arange(n, device="cuda", dtype=torch.int32)
    length = torch.full((n,), length, device="cuda", dtype=torch.int32)
    refs = torch.ones(pages + n, device="cuda", dtype=torch.int32)
    ctx.kv_cache(900, k, v, table, length, refs)
    return k, v, table, length, refs


def test_sums_past_24_bits(ctx):  # noqa: F811
    """Plans are made of sums over all entries: 77 million positions here, from whole
    numbers, so that no order of adding changes a plan, and the bits stay the same."""
    from kestrel_b200.cuda import OPT_SHARE_ALWAYS
    ctx.set_option(OPT_SHARE_ALWAYS, 0)
    try:
        held = wide_tables(ctx, 96, 800001, 1, 64)
        q, start = torch.randn((96, 4, 64), device="cuda").half(), ints(list(range(0, 97, 8)))
        outs = []
        for _ in range(4):
            outs.append(torch.empty_like(q))
            ctx.attn_shared_dev(900, 0, q, start, outs[-1])
        ctx.sync()
        assert all(torch.equal(outs[0], x) for x in outs[1:])
        assert torch.isfinite(outs[0]).all()
        del held
    finally:
        ctx.set_option(OPT_SHARE_ALWAYS, 1)


@pytest.mark.parametrize("n", [60, 900])
def test_little_in_common(ctx, n):  # noqa: F811
    """A page in common by twos, as many entries as the workspace takes at a time and
    more: not worth it, and not shared unless the option says so. Groups of fifty with
    almost everything in common are."""
    from kestrel_b200.cuda import OPT_SHARE_ALWAYS
    for groups, shared in (([(1, [150, 131])] * (n // 2), False), ([(40, [650 + i % 9 for i in range(n // 4)])] * 4, n > 100)):
        c, start = branches(ctx, groups, 16, 2, 256, F16, seed=n, poison=False)
        q = torch.randn((start[-1], 16, 256), device="cuda").half()
        alone = torch.empty_like(q)
        ctx.attn_decode_dev(c.id, 1, q, alone)
        always = run(ctx, c, q, start)
        ctx.set_option(OPT_SHARE_ALWAYS, 0)
        try:
            out = run(ctx, c, q, start)
        finally:
            ctx.set_option(OPT_SHARE_ALWAYS, 1)
        off = lambda x: float((x != alone).float().mean())
        assert off(always) > 0.03
        assert off(out) > 0.03 if shared else off(out) < 0.005
        assert (out.double() - alone.double()).norm() <= 2.0 ** -10 * alone.double().norm()


def test_own_parts_that_outweigh_the_prefix(ctx):  # noqa: F811
    """Not shared, own parts are read from memory as they are when shared: 600 entries in
    groups of 8 at 512 and 500 to 1000 of their own took 460 us not shared and 378 shared
    on a B200, 32 and 8 heads of 128. They are shared."""
    from kestrel_b200.cuda import OPT_SHARE_ALWAYS
    rng = np.random.default_rng(3)
    c, start = branches(ctx, [(32, [int(n) for n in rng.integers(1000, 1500, 8)]) for _ in range(75)], 16, 8, 128, F16, poison=False)
    q = torch.randn((start[-1], 32, 128), device="cuda").half()
    alone = torch.empty_like(q)
    ctx.attn_decode_dev(c.id, 1, q, alone)
    ctx.set_option(OPT_SHARE_ALWAYS, 0)
    try:
        out = run(ctx, c, q, start)
    finally:
        ctx.set_option(OPT_SHARE_ALWAYS, 1)
    assert float((out != alone).float().mean()) > 0.03
    assert (out.double() - alone.double()).norm() <= 2.0 ** -10 * alone.double().norm()
