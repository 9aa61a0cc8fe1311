"""min_p right beside a token's weight (run with -m gpu).

The weight is good to 2e-13 of itself and min_p is compared as it is, so tokens that
lie further than 1e-12 of min_p off must fall on their side. Rows of one heavy token
and one light one, in the last place, whose weight is within 2e-10 of an f32 min_p,
on either side; the number draws the last token kept.
"""
import numpy as np
import pytest

from sample_model import LD, sample
from test_gpu_sample import F32, ctx, run  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

LAST = 1 - 2.0 ** -24


def beside(count=32):
    """(logits, min_p values) so that exp(logit) is close to min_p."""
    l = np.arange(np.float32(-15.2), np.float32(-14.8), 1e-6).astype(np.float32)
    w = np.exp(l.astype(LD))
    p = w.astype(np.float32)
    off = w / p.astype(LD) - 1
    good = np.nonzero((np.abs(off) > 2e-12) & (np.abs(off) < 2e-10))[0]
    good = np.concatenate([good[off[good] > 0][:count], good[off[good] < 0][:count]])
    assert len(good) == 2 * count
    return l[good], p[good]


@pytest.mark.parametrize("vocab", [300, 9000, 50257])
@pytest.mark.parametrize("settings", [{}, {"top_k": 40}, {"top_k": 270}, {"top_p": LAST}, {"top_k": 7, "top_p": LAST}], ids=str)
def test_beside_a_weight(ctx, vocab, settings):  # noqa: F811
    l, p = beside()
    x = np.full((len(l), vocab), -60.0, np.float32)
    x[:, vocab // 3] = 0.0
    x[:, -1] = l
    tokens, probs = run(ctx, torch.tensor(x, device="cuda"), [LAST] * len(l), min_p=p, **settings)
    kept = 0
    for row, least, token, share in zip(x, p, tokens, probs):
        want, part, room = sample(row, LAST, min_p=float(least), **settings)
        assert room > 1e-12 and token == want, (float(least), token, want, room)
        assert abs(share - part) <= 2.0 ** -24 * part + 1e-12
        kept += want == vocab - 1
    assert kept == len(l) // 2


@pytest.mark.parametrize("settings", [{}, {"top_k": 40}, {"top_p": 0.99}], ids=str)
def test_very_small_min_p(ctx, settings):  # noqa: F811
    """Below the units of the sums: nothing that matters is lost."""
    x = torch.linspace(0, -60, 5000, device="cuda")[None].expand(3, -1)
    for least in (1e-13, 1e-17, 1e-25, 1e-44):
        tokens, probs = run(ctx, x, [0.1, 0.5, 0.99], min_p=least, **settings)
        for u, token, share in zip([0.1, 0.5, 0.99], tokens, probs):
            want, part, _ = sample(x[0].cpu().numpy(), float(np.float32(u)), min_p=float(np.float32(least)), **settings)
            assert token == want and abs(share - part) <= 2.0 ** -24 * part + 1e-12
