"""Attention of f32 queries over many short stretches (run with -m gpu): each block
goes through items that last a few microseconds, whose warps must not be two items
behind one another.

Tolerances are those of the kernels (test_gpu_paged.py), which the helpers apply.
"""
import pytest

from test_gpu_paged import F16, F32, Cache, close, ints, queries, wide
from test_gpu_shared import branches

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from kestrel_b200.cuda import OPT_SHARE_ALWAYS, Context
    c = Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    c.set_option(OPT_SHARE_ALWAYS, 1)
    yield c
    c.close()


def test_prefixes(ctx):
    """32 groups with 256 positions in common, 8 heads: 256 items of two tiles."""
    c, start = branches(ctx, [(16, [260 + i for i in range(4)])] * 32, 16, 8, 64, F16, seed=1)
    q, out = queries(start[-1], 32, 64, F32, 2), None
    at = ints(start)
    for turn in range(400):
        out = torch.full_like(q, 7.0)
        ctx.attn_shared_dev(c.id, 0, q, at, out)
    ctx.sync()
    close(wide(out), c.expected(0, wide(q), range(start[-1]), [1] * start[-1], 64 ** -0.5, 0, 0), F32)


def test_prompts(ctx):
    """64 sequences of one to two tiles, 8 heads: 512 items."""
    lens = [100 + i for i in range(64)]
    c = Cache(ctx, lens, 16, 8, 64, F16, seed=2)
    rows = [4] * 64
    q = queries(sum(rows), 16, 64, F32, 3)
    starts = ints([4 * i for i in range(65)])
    out = None
    for turn in range(400):
        out = torch.full_like(q, 7.0)
        ctx.attn_prompt_dev(c.id, 0, q, starts, out)
    ctx.sync()
    close(wide(out), c.expected(0, wide(q), range(64), rows, 64 ** -0.5, 0, 0), F32)
