"""The operators of a sampling step run together, as a server would (run with -m
gpu): prompts, branches, decode steps that append turned keys, share the prompt's
pages and draw tokens; against the same loop from other operators of the library
(rotation alone, then writing; one sequence at a time attention) and plain models.
"""
import numpy as np
import pytest

from paged_model import PageModel
from sample_model import sample
from test_gpu_paged import F16, ints, wide

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("args", [dict(), dict(sequences=2, branches=5, prompt=700, steps=20, page=16, top_k=0, top_p=0.8),
                                  dict(window=64, sinks=4, steps=12), dict(temperature=0.0, steps=8)], ids=str)
def test_example(args):
    from kestrel_b200 import paged_example
    got = paged_example.run(**args)
    assert got["finite"] and got["tokens_drawn"] and got["same_after_compaction"]
    assert got["kernels_differ"] <= 2 * 2.0 ** -15 * 6  # (f32 results: test_gpu_paged.py)
    assert got["pages_live"] < got["pages_without_sharing"]


def test_a_step_in_two_ways():
    """Two contexts on one cache's copies: append, shared attention and drawing in one,
    rotation, writing, attention by itself and the sampling model in the other."""
    from kestrel_b200.cuda import OPT_SHARE_ALWAYS, Context
    page, nq, nkv, hd, kids, vocab = 16, 8, 2, 64, 6, 500
    stream = torch.cuda.current_stream().cuda_stream
    one, two = Context(0), Context(0)
    try:
        sides = []
        for c in (one, two):
            c.set_stream(stream)
            c.rope(3, 48, layout="interleaved", base=5e5, scaling="bands", factor=8.0, original=64, low=1.0, high=4.0)
            k, v = (torch.zeros((1, 60, nkv, page, hd), dtype=F16, device="cuda") for _ in range(2))
            state = (ints([[-1] * 20 for _ in range(kids + 1)]), ints([0] * (kids + 1)), ints([0] * 60))
            c.kv_cache(0, k, v, *state)
            sides.append((c, k, v) + state)
        one.set_option(OPT_SHARE_ALWAYS, 1)
        m = PageModel(1, 60, page, nkv, hd, kids + 1, 20, wide(sides[0][1]), wide(sides[0][2]))
        g = torch.Generator(device="cuda").manual_seed(0)
        rows = lambda n: torch.randn((n, nq + 2 * nkv, hd), generator=g, device="cuda").half().split([nq, nkv, nkv], 1)
        project = torch.randn((nq * hd, vocab), generator=g, device="cuda") * (nq * hd) ** -0.5 * 40

        def positions(seqs, counts):
            return ints([m.length[s] - c + i for s, c in zip(seqs, counts) for i in range(c)])

        # The prompt, then its branches.
        q, k, v = rows(150)
        for c, *_ in sides:
            c.kv_extend_dev(0, ints([0]), ints([150]))
        m.extend([0], [150])
        one.kv_append_dev(0, 0, 3, k, v, seqs=ints([0]), row_start=ints([0, 150]))
        turned = torch.empty(k.shape, dtype=F16, device="cuda")
        two.rope_dev(3, k, positions([0], [150]), turned)
        two.kv_write_dev(0, 0, turned, v, seqs=ints([0]), row_start=ints([0, 150]))
        seqs = list(range(1, kids + 1))
        for c, *_ in sides:
            c.kv_fork_dev(0, ints([0] * kids), ints(seqs))
            c.kv_free_dev(0, ints([0]))
        m.fork([0] * kids, seqs)
        m.free([0])
        for step in range(5):
            q, k, v = rows(kids)
            for c, *_ in sides:
                c.kv_extend_dev(0, ints(seqs), ints([1] * kids))
            m.extend(seqs, [1] * kids)
            q1, a1, a2 = (torch.empty((kids, nq, hd), dtype=F16, device="cuda") for _ in range(3))
            one.kv_append_dev(0, 0, 3, k, v, q=q, q_out=q1, seqs=ints(seqs))
            one.attn_shared_dev(0, 0, q1, ints([0, kids]), a1, seqs=ints(seqs))
            at = positions(seqs, [1] * kids)
            q2, k2 = (torch.empty(x.shape, dtype=F16, device="cuda") for x in (q, k))
            two.rope_dev(3, q, at, q2)
            two.rope_dev(3, k, at, k2)
            two.kv_write_dev(0, 0, k2, v, seqs=ints(seqs))
            two.attn_decode_dev(0, 0, q2, a2, seqs=ints(seqs))
            one.sync()
            two.sync()
            assert torch.equal(q1, q2)
            for x, y in zip(sides[0][1:], sides[1][1:]):
                assert torch.equal(x, y)
            assert sides[0][3].tolist() == m.table and sides[0][5].tolist() == m.refs
            # f16 results: twice the bound of each.
            assert float((a1.float() - a2.float()).abs().max()) <= 4 * 2.0 ** -11 * 6
            logits = a1.flatten(1).float() @ project
            u = torch.rand(kids, generator=g, device="cuda")
            tokens, probs = torch.empty(kids, dtype=torch.int32, device="cuda"), torch.empty(kids, device="cuda")
            one.sample_dev(logits, u, tokens, probs=probs, top_p=torch.full((kids,), 0.9, device="cuda"))
            one.sync()
            for i in range(kids):
                want, share, room = sample(wide(logits)[i], float(u[i]), top_p=float(np.float32(0.9)))
                assert room < 1e-9 or (int(tokens[i]) == want and abs(float(probs[i]) - share) < 2.0 ** -24)
    finally:
        one.close()
        two.close()
