"""CPU checks of the rotation's plain model and of the refusals that need no GPU."""
import numpy as np
import pytest

from rope_model import LD, frequencies, gain_of, turn

torch = pytest.importorskip("torch")


def test_model_keeps_lengths_and_differences():
    """Without a gain a rotation keeps a pair's length, and scores depend on the
    distance of two positions alone."""
    rng = np.random.default_rng(0)
    q, k = rng.standard_normal((2, 1, 1, 16))
    for layout in ("half", "interleaved"):
        at = lambda x, p: turn(x, [p], 12, layout)[0][0, 0]
        np.testing.assert_allclose(float(np.sum(at(q, 7) ** 2)), float(np.sum(q ** 2)), rtol=1e-15)
        near, far = at(q, 9) @ at(k, 4), at(q, 100009) @ at(k, 100004)
        np.testing.assert_allclose(float(near), float(far), rtol=1e-12)
        assert (at(q, 5)[12:] == q[0, 0, 12:]).all()
        np.testing.assert_allclose(turn(at(q, 5)[None, None], [-5], 12, layout)[0].astype(float), q, rtol=1e-14)


def test_scalings_at_their_ends():
    w = frequencies(64, 1e4)
    assert w[0] == 1 and np.allclose((w / frequencies(64, 1e4, "linear", 4.0)).astype(float), 4)
    for scaling, low, high in (("yarn", 1.0, 32.0), ("bands", 1.0, 4.0)):
        ratio = (w / frequencies(64, 1e4, scaling, 8.0, 4096, low, high)).astype(float)
        assert ratio[0] == 1 and abs(ratio[-1] - 8) < 1e-12 and (np.diff(ratio) >= 0).all()
        assert ((ratio > 1.0) & (ratio < 8.0)).any()
    assert abs(float(gain_of("yarn", 8.0)) - 1.2079441541679836) < 1e-15
    assert gain_of("yarn", 8.0, gain=2.0) == 2 and gain_of("linear", 8.0) == 1
    assert (frequencies(8, 1e4, freq_factors=[1, 2, 4, 8]) == frequencies(8, 1e4) / LD(2) ** np.arange(4)).all()


def test_null_context_is_refused():
    from kestrel_b200 import cuda
    lib = cuda.lib()
    assert lib.kc_rope(None, 0, 64, 0, 1e4, 0, 1.0, 0, 0.0, 0.0, 0.0, None) == 1
    assert lib.kc_rope_dev(None, 0, None, 0, 1, 64, 0, None, 64, None, 64) == 1
    assert lib.kc_kv_append_dev(None, 0, 0, 0, None, None, 0, 0, 0, None, None, 0, 0, 0, None, 0, None, 0) == 1


def test_binding_refuses_what_it_cannot_pass():
    from kestrel_b200 import cuda
    ctx = cuda.Context.__new__(cuda.Context)  # no GPU here: the checks come before any call
    ctx.h, ctx._kv, ctx._kv_dims = None, {}, {}
    x, i = torch.zeros((2, 1, 8)), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="layout"):
        ctx.rope(0, 8, layout="both")
    with pytest.raises(ValueError, match="scaling"):
        ctx.rope(0, 8, scaling="more")
    with pytest.raises(ValueError, match="freq_factors"):
        ctx.rope(0, 8, freq_factors=[1.0])
    with pytest.raises(ValueError, match="CUDA"):
        ctx.rope_dev(0, x, i)
    with pytest.raises(ValueError, match="not registered"):
        ctx.kv_append_dev(0, 0, 0, x, x)
