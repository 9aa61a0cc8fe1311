"""CPU checks of the sampling model and of the refusals that need no GPU."""
import math

import numpy as np
import pytest

from sample_model import sample

torch = pytest.importorskip("torch")


def test_model_follows_the_definition():
    l = np.log([0.1, 0.4, 0.2, 0.3])
    for u, want in ((0.0, 0), (0.09, 0), (0.11, 1), (0.49, 1), (0.51, 2), (0.71, 3), (1.0, 3), (math.nan, 0)):
        assert sample(l, u)[0] == want
    assert sample(l, 0.99, top_k=2)[:1] == (3,) and abs(sample(l, 0.0, top_k=2)[1] - 4 / 7) < 1e-12
    assert [sample(l, u, top_p=0.8)[0] for u in (0.0, 0.5, 0.9)] == [1, 2, 3]
    assert sample(l, 0.99, top_p=0.0)[0] == 1 and sample(l, 0.3, min_p=0.7)[0] == 1
    assert sample(l, 0.99, temperature=0.0)[0] == 1
    assert sample([1.0, 1.0, 0.0, 1.0], 0.99, top_k=2)[0] == 1  # equal ones by their index
    assert sample([-math.inf, math.nan], 0.5)[:2] == (-1, 0.0)
    assert sample([0.0, math.inf, 5.0, math.inf], 0.6)[:2] == (3, 0.5)
    assert [sample([2.0, -math.inf, 3.0], u, temperature=math.inf)[0] for u in (0.4, 0.6)] == [0, 2]


def test_equal_logits_share_exactly():
    """Halves and quarters of equal weights are borders that arithmetic must not blur."""
    assert sample([0.0] * 8, 0.99, top_p=0.5)[0] == 3
    assert [sample([0.0] * 4, u)[0] for u in (0.25, 0.5, 0.75)] == [1, 2, 3]


def test_null_context_is_refused():
    from kestrel_b200 import cuda
    assert cuda.lib().kc_sample_dev(None, 0, None, 8, 1, 8, None, None, None, None, None, None, None) == 1


def test_binding_refuses_what_it_cannot_pass():
    from kestrel_b200 import cuda
    ctx = cuda.Context.__new__(cuda.Context)  # no GPU here: the checks come before any call
    ctx.h = None
    x = torch.zeros((2, 8))
    with pytest.raises(ValueError, match="CUDA"):
        ctx.sample_dev(x, x[:, 0], x[:, 0].int())
