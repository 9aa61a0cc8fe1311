"""What a plan decides is not to be seen in the results (run with -m gpu): weights of
shared prefixes are as good as the decode call's, 22 bits or 16 of bf16.

At 640 positions of unit normal values results are about 0.04, where a step of f16 is
2^-15 and one of bf16 2^-12. Weights off by 2^-22 (2^-17) of themselves move a result
by that share of a mean of |v|, 0.8, at most, so at most 2 * 0.8 * 2^-22 / 2^-15 = 1.3%
(2 * 0.8 * 2^-17 / 2^-12 = 5%) of the results fall to another neighbour; f32 sums in
another order, 2^-24 of the same a step, add less than as much. Weights rounded to the
type leave a third of them there.
"""
import numpy as np
import pytest

from test_gpu_paged import BF16, F16
from test_gpu_shared import branches, ctx, queries, run  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("t,most", [(F16, 0.03), (BF16, 0.06)], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads", [(8, 2, 64), (32, 4, 128), (6, 2, 80), (16, 2, 256), (4, 4, 200)], ids=str)
def test_results_are_the_decode_calls(ctx, heads, t, most):  # noqa: F811
    nh, nkv, hd = heads
    c, start = branches(ctx, [(40, [650 + 7 * i for i in range(9)]), (39, [660, 640, 700])], 16, nkv, hd, t, poison=False)
    q = queries(start[-1], nh, hd, t, 3).contiguous()
    out, alone = run(ctx, c, q, start), torch.empty_like(q)
    ctx.attn_decode_dev(c.id, 1, q, alone)
    ctx.sync()
    assert float((out != alone).float().mean()) <= most
    exact = c.expected(1, q.float().cpu().numpy(), range(12), [1] * 12, hd ** -0.5, 0, 0)
    off = lambda x: np.linalg.norm(x.double().cpu().numpy() - exact) / np.linalg.norm(exact)
    assert off(out) <= 1.05 * off(alone)
