"""Sampling by top-p where much of a row lies far from where its sum ends (run with
-m gpu): tokens spread over all of the histogram, masked ones by the thousand.

Compared as in test_gpu_sample.py, whose derivation holds here.
"""
import numpy as np
import pytest

from test_gpu_sample import check, ctx  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("p", [0.3, 0.9, 0.95, 0.999])
@pytest.mark.parametrize("vocab", [2, 76, 300, 2049])
def test_short_rows(ctx, vocab, p):  # noqa: F811
    """A row much shorter than its place in shared memory, most of its tokens in bins of
    their own."""
    rng = np.random.default_rng(vocab)
    x = rng.uniform(2.0, 12.0, (96, 1)) / 3 * rng.standard_normal((96, vocab))
    for t in (0.7, 1.2, 5.0):
        check(ctx, torch.tensor(x, dtype=torch.float32, device="cuda"), rng.random(96), temperature=t, top_p=p)


@pytest.mark.parametrize("masked", [-np.inf, float(np.finfo(np.float32).min), -60.0], ids=str)
def test_masked_rows(ctx, masked):  # noqa: F811
    """All but a few tokens masked: by infinity, the type's lowest value, a low one."""
    rng = np.random.default_rng(5)
    x = np.full((48, 50257), masked)
    for i in range(48):
        few = rng.choice(50257, 1 + 7 * i, replace=False)
        x[i, few] = rng.uniform(0.5, 6.0) * rng.standard_normal(len(few))
    x = torch.tensor(x, dtype=torch.float32, device="cuda")
    for t in (0.5, 2.0, 20.0):
        for settings in ({"top_p": 0.5}, {"top_p": 0.95}, {"top_p": 0.95, "top_k": 200}, {"top_p": 0.8, "min_p": 0.05}):
            check(ctx, x, rng.random(48), temperature=t, **settings)


def test_flat_tails(ctx):  # noqa: F811
    """A few likely tokens before very many unlikely ones that weigh as much together."""
    rng = np.random.default_rng(6)
    x = rng.uniform(-0.5, 0.5, (32, 100277)) - rng.uniform(8.0, 40.0, (32, 1))
    x[:, rng.choice(100277, 60, replace=False)] = 3.0 * rng.standard_normal((32, 60))
    x = torch.tensor(x, dtype=torch.float32, device="cuda")
    for t in (0.9, 2.5, 10.0):
        for p in (0.2, 0.9, 0.99):
            check(ctx, x, rng.random(32), temperature=t, top_p=p)
