"""Attention over shared prefixes where a part weighs next to nothing (run with -m gpu).

The results are the decode call's: a part whose scores lie 100 and more below the
others' weighs e^-100 (3.8e-44), so that values of 1e36 in it count 4e-8 at most,
which is below the roundings of results of about 1. Tolerances: the two calls' of
test_gpu_shared.py, for the values that weigh.
"""
import numpy as np
import pytest

from test_gpu_paged import BF16, F16, F32, close, wide
from test_gpu_shared import branches, ctx, run  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def far_below(c, positions):
    """Keys of those positions of layer 1 at -2.5, the others near nothing: scores of
    queries of ones 160 below. Returns where they are."""
    hide = torch.zeros((c.k.shape[1], 16), dtype=torch.bool)
    for s, row in enumerate(c.m.table):
        for p in positions:
            if p < c.m.length[s]:
                hide[row[p // 16], p % 16] = True
    hide = hide.cuda()[None, :, None, :, None]
    c.k.copy_(torch.where(hide, torch.full_like(c.k, -2.5), c.k * 0.05))
    c.m.k = wide(c.k)
    return hide


def ones(nh, hd, t):
    return torch.ones((3, nh, hd), device="cuda", dtype=t)


@pytest.mark.parametrize("where", [range(2048), range(2048, 2100), range(512, 1024)], ids=["prefix", "own", "part"])
def test_large_values_far_below(ctx, where):  # noqa: F811
    """1e36 in positions that the softmax leaves out: all of the prefix, all of the own
    parts, one part of the prefix."""
    c, start = branches(ctx, [(128, [2100, 2060, 2049])], 16, 1, 64, BF16, poison=False)
    hide, q = far_below(c, where), ones(4, 64, BF16)
    rest = c.expected(1, wide(q), range(3), [1] * 3, 1.0, 0, 0)  # (before the values)
    c.v.copy_(torch.where(hide, torch.full_like(c.v, 1e36), c.v))
    out = run(ctx, c, q, start, scale=1.0)
    close(wide(out), rest, BF16)
    alone = torch.empty_like(out)
    ctx.attn_decode_dev(c.id, 1, q, alone, scale=1.0)
    ctx.sync()
    close(wide(out), wide(alone).astype(np.float64), BF16)


@pytest.mark.parametrize("pair", [(F32, F16), (F16, F16), (BF16, BF16)], ids=str)
def test_an_infinite_value_in_a_part_far_below(ctx, pair):  # noqa: F811
    """However little all of a prefix weighs, an infinity in it counts, in its column
    alone."""
    c, start = branches(ctx, [(128, [2100, 2060, 2052])], 16, 1, 64, pair[1], poison=False)
    far_below(c, range(2048))
    c.v[1, c.m.table[0][1900 // 16], 0, 1900 % 16, 7] = -float("inf")
    out = wide(run(ctx, c, ones(4, 64, pair[0]), start, scale=1.0))
    assert (out[:, :, 7] == -np.inf).all()
    assert np.isfinite(np.delete(out, 7, 2)).all()
