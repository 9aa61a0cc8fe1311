"""CPU checks of the paged cache's plain model and of the binding's refusals."""
import numpy as np
import pytest

from paged_model import PageModel, Refused, attention

torch = pytest.importorskip("torch")


def model(n_pages=12, page=16, n_seq=4, max_pages=6):
    z = np.zeros((2, n_pages, 1, page, 8), np.float32)
    return PageModel(2, n_pages, page, 1, 8, n_seq, max_pages, z, z)


def test_model_shares_then_copies():
    m = model(n_pages=11)
    m.extend([0], [20])
    m.k[:, 1, :, :4] = 7  # positions 16 .. 19
    m.fork([0, 0], [1, 2])
    assert m.refs[:3] == [3, 3, 0]
    m.extend([0, 1, 2], [1, 1, 1])  # two holders copy, the last keeps the page
    m.check()
    assert [m.table[s][1] for s in range(3)] == [2, 3, 1] and m.refs[:4] == [3, 1, 1, 1]
    assert (m.k[:, 2, :, :4] == 7).all() and (m.k[:, 2, :, 4:] == 0).all()
    with pytest.raises(Refused):
        m.extend([0, 0], [1, 1])
    with pytest.raises(Refused):
        m.extend([0, 1], [70, 70])
    m.free([0, 2], [5, 0])
    m.check()
    assert m.compact() == 2 and m.length == [5, 21, 0, 0]
    m.check()


def test_attention_model_sees_only_what_is_visible():
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal(s) for s in ((3, 2, 8), (9, 1, 8), (9, 1, 8)))
    k[8], v[8] = np.nan, np.nan  # the last position
    out = attention(q, k, v, 6, 0.3)
    assert np.isfinite(out[:2]).all() and np.isnan(out[2]).all()
    near = attention(q[:1], k, v, 6, 0.3, window=2, sinks=1)
    s = 0.3 * k[[0, 5, 6], 0] @ q[0, 0]
    p = np.exp(s) / np.exp(s).sum()
    np.testing.assert_allclose(near[0, 0], p @ v[[0, 5, 6], 0], rtol=1e-12)
    assert (attention(q, k[:0], v[:0], -3, 0.3) == 0).all()


def test_null_context_is_refused():
    from kestrel_b200 import cuda
    lib = cuda.lib()
    assert lib.kc_kv_drop(None, 0) == 1
    assert lib.kc_kv_compact_dev(None, 0, None) == 1
    assert lib.kc_attn_decode_dev(None, 0, 0, None, 0, 8, 0, None, 0, 1.0, 0, 0, None, 0) == 1


def test_binding_refuses_tensors_it_cannot_pass():
    from kestrel_b200 import cuda
    ctx = cuda.Context.__new__(cuda.Context)  # no GPU here: the checks come before any call
    ctx.h, ctx._kv, ctx._kv_dims = None, {}, {}
    x = torch.zeros((2, 3, 1, 16, 8))
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ctx.kv_cache(0, x, x, i.view(2, 2), i[:2], i[:3])
    with pytest.raises(ValueError, match="int32 CUDA"):
        ctx.kv_fork_dev(0, i, i)
    with pytest.raises(ValueError, match="not registered"):
        ctx.kv_write_dev(0, 0, x[0], x[0])
    with pytest.raises(ValueError, match="not registered"):
        ctx.attn_decode_dev(0, 0, x[0, 0], x[0, 0])
