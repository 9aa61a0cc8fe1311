"""top-k among more tokens of one bin than are looked through pair by pair, whose
places span all of their 64 bits (run with -m gpu). Equal weights (an infinite
temperature), so shares and borders are exact."""
import numpy as np
import pytest

from test_gpu_sample import ctx, run  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("vocab", [1500, 40000])
@pytest.mark.parametrize("k", [30, 600])
def test_places_near_the_largest(ctx, vocab, k):  # noqa: F811
    rng = np.random.default_rng(vocab)
    x = rng.uniform(-1.6e38, 1.6e38, (4, vocab)).astype(np.float32)
    u = (np.arange(4) * 0.25 + 0.1).astype(np.float32)
    tokens, probs = run(ctx, torch.tensor(x, device="cuda"), u, top_k=k, temperature=float("inf"))
    for row, n, token, share in zip(x, u, tokens, probs):
        kept = np.sort(np.lexsort((np.arange(vocab), -row))[:k])
        assert token == kept[int(k * float(n))] and share == np.float32(1 / k)
