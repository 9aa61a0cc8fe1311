"""CPU checks of attention over shared prefixes: the split that it rests on, in 64
bits, and the refusals that need no GPU."""
import numpy as np
import pytest

from paged_model import attention

torch = pytest.importorskip("torch")


def test_a_softmax_splits_at_any_position():
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal(s) for s in ((1, 2, 8), (30, 1, 8), (30, 1, 8)))
    whole = attention(q, k, v, 29, 0.4)[0]
    for cut in (1, 16, 29):
        parts = []
        for a, b in ((0, cut), (cut, 30)):
            s = 0.4 * np.einsum("hd,jd->hj", q[0], k[a:b, 0])
            m = s.max(1, keepdims=True)
            p = np.exp(s - m)
            parts.append((m, p.sum(1, keepdims=True), p @ v[a:b, 0] / p.sum(1, keepdims=True)))
        top = np.maximum(parts[0][0], parts[1][0])
        w = [l * np.exp(m - top) for m, l, _ in parts]
        np.testing.assert_allclose((w[0] * parts[0][2] + w[1] * parts[1][2]) / (w[0] + w[1]), whole, rtol=1e-12)


def test_refusals_without_a_gpu():
    from kestrel_b200 import cuda
    assert cuda.lib().kc_attn_shared_dev(None, 0, 0, None, 0, None, 0, 8, 0, None, 0, 1.0, None, 0) == 1
    ctx = cuda.Context.__new__(cuda.Context)
    ctx.h, ctx._kv, ctx._kv_dims = None, {}, {}
    with pytest.raises(ValueError, match="not registered"):
        ctx.attn_shared_dev(0, 0, torch.zeros((1, 1, 8)), torch.zeros(2, dtype=torch.int32), torch.zeros((1, 1, 8)))
