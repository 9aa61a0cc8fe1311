"""When attn_shared_dev shares, and that the choice is the same every time (run with
-m gpu). Where the scores of what is common lie 160 below the others, and one value of
it is infinite, the choice shows: shared, the common part is weighed by itself and the
infinity counts; not shared, its weight next to the others' is zero in f32, and zero
times it is not a number.
"""
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


def is_shared(ctx, groups, page, nkv, nh, hd, always=False):  # noqa: F811
    """Whether each entry of groups (common pages, lengths) is."""
    from kestrel_b200.cuda import OPT_SHARE_ALWAYS
    c, start = branches(ctx, groups, page, nkv, hd, F16, poison=False)
    c.k.mul_(0.05)
    for (pages, _), lead in zip(groups, start):
        common = torch.tensor(c.m.table[lead][:pages], device="cuda")
        c.k[1, common] = -2.5 * 64 / hd
        c.v[1, common[0], :, 0, 3] = -float("inf")
    q = torch.ones((start[-1], nh, hd), device="cuda", dtype=F16)
    ctx.set_option(OPT_SHARE_ALWAYS, int(always))
    try:
        out = run(ctx, c, q, start, scale=1.0)[:, :, 3]
    finally:
        ctx.set_option(OPT_SHARE_ALWAYS, 1)
    assert (out.isneginf() | out.isnan()).all()
    return out.isneginf().all(1)


@pytest.mark.parametrize("n", [60, 900])
def test_little_in_common(ctx, n):  # noqa: F811
    """A page in common by twos, as many entries as the workspace takes at a time and
    more: not worth it, and not shared unless the option says so. Groups with almost
    everything in common are, where there is much of it."""
    pairs = [(1, [150, 131])] * (n // 2)
    assert is_shared(ctx, pairs, 16, 2, 16, 256, always=True).all()
    assert not is_shared(ctx, pairs, 16, 2, 16, 256).any()
    large = [(40, [650 + i % 9 for i in range(n // 4)])] * 4
    assert is_shared(ctx, large, 16, 2, 16, 256, always=True).all()
    assert (is_shared(ctx, large, 16, 2, 16, 256) == (n > 100)).all()


def test_own_parts_that_outweigh_the_prefix(ctx):  # noqa: F811
    """Not shared, own parts are read from memory as they are when shared: 600 entries in
    groups of 8 at 512 and 500 to 1000 of their own took 459 us not shared and 411 shared
    on a B200, 32 and 8 heads of 128. They are shared."""
    rng = np.random.default_rng(3)
    groups = [(32, [int(n) for n in rng.integers(1000, 1500, 8)]) for _ in range(75)]
    assert is_shared(ctx, groups, 16, 8, 32, 128).all()
