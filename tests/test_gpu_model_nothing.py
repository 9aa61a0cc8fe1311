"""kc_model_sample on logits that are not numbers (run with -m gpu): what it says where
there is nothing to draw, and temperature 0 against the greedy loop."""
import ctypes

import numpy as np
import pytest

from kestrel_b200 import ggml, synth

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

STATE, NONE = 7, 0xFFFFFFFF
PROMPT = [int(t) for t in np.random.default_rng(4).integers(0, synth.CONFIG0["n_vocab"], 9)]


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from kestrel_b200.cuda import Context
    c = Context(0)
    yield c
    c.close()


def load(ctx, edit):
    """CONFIG0 with one tensor edited by edit(name, data [rows, ...])."""
    model = synth.make_model(synth.CONFIG0, seed=0)
    model["tensors"] = [(l, n, t, edit(n, np.array(data).reshape(rows, -1)) if l < 0 else data, rows, cols)
                        for l, n, t, data, rows, cols in model["tensors"]]
    synth.load_cuda(ctx, model, n_ctx=64)


def no_number(data, rows):
    """Q8_0 rows whose first block's scale is not a number."""
    assert synth.CONFIG0["t_out"] == ggml.Q8_0
    data = data.view(np.uint8).copy()
    data[rows, :2] = np.array([0x00, 0x7E], np.uint8)
    return data


def test_nothing_to_draw(ctx):
    from kestrel_b200.cuda import KestrelCudaError, lib

    load(ctx, lambda name, data: no_number(data, slice(None)) if name == "output" else data)
    ctx.model_truncate(0)
    assert np.isnan(ctx.model_forward(PROMPT)[0]).all()
    for settings in ({}, {"top_k": 3}, {"temperature": 0.5, "top_p": 0.9}):
        ctx.model_truncate(0)
        with pytest.raises(KestrelCudaError, match="minus infinity") as e:
            ctx.model_sample(PROMPT, 5, [0.5] * 5, **settings)
        assert e.value.code == STATE
        assert ctx.model_cached() == len(PROMPT)
    ctx.model_truncate(0)
    p, u = np.array(PROMPT, np.uint32), np.full(5, 0.5, np.float32)
    tokens, probs = np.zeros(5, np.uint32), np.ones(5, np.float32)
    at = lambda a: ctypes.c_void_p(a.ctypes.data)
    assert lib().kc_model_sample(ctx.h, at(p), len(p), 5, 1.0, 0, 1.0, 0.0, at(u), at(tokens), at(probs)) == STATE
    assert (tokens == NONE).all() and (probs == 0).all()
    # The context goes on; the greedy loop takes the first token, and so does temperature 0.
    ctx.model_truncate(0)
    greedy = ctx.model_generate(PROMPT, 5)
    ctx.model_truncate(0)
    assert ctx.model_sample(PROMPT, 5, u, temperature=0.0) == (greedy, [1.0] * 5)


def test_a_first_logit_that_is_not_a_number(ctx):
    load(ctx, lambda name, data: no_number(data, 0) if name == "output" else data)
    ctx.model_truncate(0)
    greedy = ctx.model_generate(PROMPT, 6)
    assert greedy == [0] * 6
    for temperature in (0.0, -1.0, float("nan")):
        ctx.model_truncate(0)
        assert ctx.model_sample(PROMPT, 6, [0.5] * 6, temperature=temperature) == (greedy, [1.0] * 6)
    ctx.model_truncate(0)
    tokens, probs = ctx.model_sample(PROMPT, 6, np.linspace(0.0, 0.99, 6))
    assert 0 not in tokens and all(0 < p < 1 for p in probs)
