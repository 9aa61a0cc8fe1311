"""Temperatures and logits at the ends of f32 (run with -m gpu): weights depend on
(l - m) / T alone, whether the difference passes the largest f32 or 1 / T does.

Compared as in test_gpu_sample.py, whose derivation holds here.
"""
import numpy as np
import pytest

from test_gpu_sample import check, ctx, run  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SETTINGS = [{}, {"top_k": 30}, {"top_k": 400}, {"top_p": 0.6}, {"top_k": 200, "top_p": 0.8}, {"min_p": 0.01}, {"top_p": 0.9, "min_p": 0.001}]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_differences_past_the_largest_value(ctx, settings):  # noqa: F811
    rng = np.random.default_rng(0)
    for vocab in (700, 20000):
        x = rng.uniform(-3.3e38, 3.3e38, (12, vocab)).astype(np.float32)
        x[:, :40] = rng.uniform(2e38, 3.4e38, (12, 40))
        x[6:, 40:] = -np.finfo(np.float32).max
        for t in (3e38, 1e38, 2e37, 1e36):
            check(ctx, torch.tensor(x, device="cuda"), rng.random(12).astype(np.float32), temperature=t, **settings)


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_temperatures_whose_reciprocal_is_infinite(ctx, settings):  # noqa: F811
    rng = np.random.default_rng(1)
    for vocab in (700, 20000):
        for t, spread in ((1e-38, 4e-38), (1e-40, 3e-40), (1e-40, 5e-39), (1.4e-45, 1e-41), (1.4e-45, 1e-44)):
            x = (-np.abs(spread * rng.standard_normal((12, vocab)))).astype(np.float32)
            # (Apart from each other, but for a few: few whole steps of the smallest f32.)
            check(ctx, torch.tensor(x, device="cuda"), rng.random(12).astype(np.float32), temperature=t, **settings)


def test_no_temperature_is_too_high(ctx):  # noqa: F811
    """Everything but minus infinity weighs the same."""
    x = torch.tensor([[3e38, -3e38, 0.0, -np.inf, np.nan, 1e-40, -3.4e38, 7.0]], dtype=torch.float32, device="cuda").expand(6, -1)
    u = [0.0, 0.17, 0.34, 0.51, 0.67, 0.84]
    for settings in ({}, {"top_p": 0.99}, {"top_k": 6}):
        tokens, probs = run(ctx, x, u, temperature=float("inf"), **settings)
        assert tokens == [0, 1, 2, 5, 6, 7] and probs == [float(np.float32(1) / np.float32(6))] * 6
