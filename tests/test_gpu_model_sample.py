"""kc_model_sample: the whole-model loop with drawn tokens (run with -m gpu).

Every token must be the one that the sampling definition, in the host's widest
type, takes from that step's logits (kc_model_forward after the same tokens gives
them, bit for bit: both run the reference's one-row decode path) with that step's
number. Decisions closer than 1e-9 of the sums compared are left out; shares are f32
and rounded once (2^-24), from weights good to 2e-13.
"""
import numpy as np
import pytest

from kestrel_b200 import synth
from sample_model import sample

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from kestrel_b200.cuda import Context
    c = Context(0)
    synth.load_cuda(c, synth.make_model(synth.CONFIG0, seed=0), n_ctx=160)
    yield c
    c.close()


PROMPT = [int(t) for t in np.random.default_rng(3).integers(0, synth.CONFIG0["n_vocab"], 20)]


@pytest.mark.parametrize("settings", [dict(temperature=0.9), dict(temperature=0.7, top_k=40, top_p=0.9),
                                      dict(temperature=1.2, top_p=0.8, min_p=0.01), dict(top_k=1)], ids=str)
def test_every_token_is_its_logits(ctx, settings):
    u = np.random.default_rng(1).random(24).astype(np.float32)
    ctx.model_truncate(0)
    tokens, probs = ctx.model_sample(PROMPT, 24, u, **settings)
    assert ctx.model_cached() == len(PROMPT) + 23
    ctx.model_truncate(0)
    feed, near = PROMPT, 0
    for i in range(24):
        logits, _ = ctx.model_forward(feed)
        want, share, room = sample(logits, float(u[i]), **{k: float(np.float32(v)) if k != "top_k" else v
                                                             for k, v in settings.items()})
        if room >= 1e-9:
            assert tokens[i] == want, i
            assert abs(probs[i] - share) <= 2.0 ** -24 * share + 1e-12
        else:
            near += 1
        feed = [tokens[i]]
    assert near <= 1


def test_temperature_zero_is_greedy(ctx):
    ctx.model_truncate(0)
    greedy = ctx.model_generate(PROMPT, 20)
    ctx.model_truncate(0)
    assert ctx.model_sample(PROMPT, 20, [0.9] * 20, temperature=0.0) == (greedy, [1.0] * 20)
    ctx.model_truncate(0)
    assert ctx.model_sample(PROMPT, 1, [0.5], temperature=0.0)[0] == greedy[:1]
    ctx.model_truncate(0)
    assert ctx.model_sample(PROMPT, 0, []) == ([], [])
    assert ctx.model_cached() == len(PROMPT)


def test_refusals(ctx):
    from kestrel_b200.cuda import Context, KestrelCudaError, lib
    ctx.model_truncate(0)
    with pytest.raises(ValueError):
        ctx.model_sample(PROMPT, 3, [0.5])
    with pytest.raises(KestrelCudaError):
        ctx.model_sample(PROMPT, 200, [0.5] * 200)  # past n_ctx
    assert lib().kc_model_sample(ctx.h, None, 0, 1, 1.0, 0, 1.0, 0.0, None, None, None) == 1
    empty = Context(0)
    with pytest.raises(KestrelCudaError) as e:
        empty.model_sample(PROMPT, 1, [0.5])
    assert e.value.code == 7
    empty.close()
