"""Rows for which some blocks of a cluster have nothing to load, launched one behind
the other (run with -m gpu): the same tokens every time."""
import numpy as np
import pytest

from test_gpu_sample import ctx, floats, logits_of  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("vocab", [16385, 33000, 50257])
def test_blocks_without_a_token(ctx, vocab):  # noqa: F811
    x = logits_of(3, vocab, torch.float32, vocab)
    u = floats(np.random.default_rng(0).random(3))
    p = floats([0.9, 1.0, 0.7])
    out = torch.zeros((200, 3), dtype=torch.int32, device="cuda")
    for row in out:
        ctx.sample_dev(x, u, row, top_p=p)
    ctx.sync()
    assert (out == out[0]).all() and (out >= 0).all()
