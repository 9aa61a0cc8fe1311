"""Where top-p ends among very many light tokens (run with -m gpu).

Weights are good to 2e-13 of themselves, and the whole numbers that they are summed
in add at most 2e-13 of the largest, however many there are (393216 of 2^-61). So a
decision that was made by more than 8e-13 of the two sums compared cannot fall
otherwise; 1e-12 is asked for here. The rows are made so that each has a border
closer than three billionths to the sum that top_p asks for, and the number draws the
last token kept.
"""
import numpy as np
import pytest

from sample_model import LD, sample
from test_gpu_sample import BF16, F16, F32, ctx, run  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

LAST = 1 - 2.0 ** -24


def borders(row, temperature=1.0, near=2e-12, far=3e-9, most=24):
    """top_p values (f32) whose share of the row's sum lies within near .. far of a
    running sum in the order of the ranks, on both sides."""
    x = (row.astype(LD) - LD(row.max())) / LD(temperature)
    w = np.sort(np.exp(x))[::-1]
    upto = np.cumsum(w)
    p = (upto / upto[-1]).astype(np.float32)
    off = p.astype(LD) * upto[-1] - upto
    size = np.abs(off) / np.maximum(upto, 1)
    # (The last token kept is heavier than what LAST leaves of the sum.)
    good = np.nonzero((size > near) & (size < far) & (p < 1) & (w > 2e-7 * upto[-1]))[0]
    above, below = good[off[good] > 0], good[off[good] < 0]
    pick = [s[np.linspace(0, len(s) - 1, min(len(s), most // 2)).astype(int)] for s in (above, below)]
    return p[np.concatenate(pick)]


def check(ctx, row, t, ps, u=LAST, **settings):  # noqa: F811
    x = torch.tensor(row, dtype=F32, device="cuda").to(t)
    wide = x.float().cpu().numpy()
    tokens, probs = run(ctx, x[None].expand(len(ps), -1), [u] * len(ps), top_p=ps, **settings)
    sure = 0
    for p, token, share in zip(ps, tokens, probs):
        want, part, room = sample(wide, u, top_p=float(p), **settings)
        if room < 1e-12:
            continue
        sure += 1
        assert token == want, (float(p), token, want, room)
        assert abs(share - part) <= 2.0 ** -24 * part + 1e-12
    assert sure


def test_two_rows_by_arithmetic(ctx):  # noqa: F811
    for n, value, p, u, want in ((150000, -13.996, 0.99991393, LAST, 149884), (151935, -15.0625, 0.9986075758934021, 0.96743596, 28779)):
        row = np.full(n + 1, value, np.float32)
        row[0] = 0.0
        u = float(np.float32(u))
        token, _, room = sample(row, u, top_p=float(np.float32(p)))
        assert token == want and room > 1e-9
        assert run(ctx, torch.tensor(row, device="cuda")[None], [u], top_p=p)[0] == [want]


@pytest.mark.parametrize("n,value", [(150000, -13.999913), (150000, -13.991383), (393215, -14.739397), (393215, -14.653283),
                                     (100000, -12.0189705), (65536, -9.044667), (65536, -9.014786)])
def test_equal_light_tokens(ctx, n, value):  # noqa: F811
    """Weights that whole numbers of 2^-44 would round by half of one, all the same way."""
    row = np.full(n + 1, value, np.float32)
    row[n // 2] = 0.0
    ps = borders(row)
    assert len(ps) > 3
    check(ctx, row, F32, ps)


@pytest.mark.parametrize("t", [BF16, F16], ids=str)
def test_ties_of_16_bit_rows(ctx, t):  # noqa: F811
    """Thousands of ties at a few dozen values, in several bins and stretches."""
    rng = np.random.default_rng(2)
    row = (0.05 * rng.standard_normal(120000) - 11.5).astype(np.float32)
    row[[5, 70001]] = 0.0, -1.0
    row = torch.tensor(row).to(t).float().numpy()
    ps = borders(row)
    assert len(ps) > 3
    check(ctx, row, t, ps)


@pytest.mark.parametrize("temperature", [0.02, 3.0])
def test_light_tokens_in_one_bin_with_heavy_ones(ctx, temperature):  # noqa: F811
    """At low temperatures one bin holds weights far apart; at high ones all that is
    far below is in the last bin."""
    temperature = float(np.float32(temperature))
    row = np.full(140001, -13.999913 * temperature, np.float32)
    row[::7] = -13.991383 * temperature
    row[3] = 0.0
    ps = borders(row, temperature)
    assert len(ps) > 3
    check(ctx, row, F32, ps, temperature=temperature)


def test_what_top_k_leaves(ctx):  # noqa: F811
    """Under top-k, whose own sum is what top_p asks a share of."""
    row = np.full(150001, -13.999913, np.float32)
    row[77] = 0.0
    for k in (140000, 120):
        kept = np.sort(row)[::-1][:k]
        ps = borders(kept, far=3e-9 if k > 1000 else 3e-8)
        assert len(ps)
        check(ctx, row, F32, ps, top_k=k)
