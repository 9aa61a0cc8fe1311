"""The paged key-value cache in a serving loop: prompts, branches, decode steps.

  python -m kestrel_b200.paged_example
  python -m kestrel_b200.paged_example --sequences 8 --branches 4 --prompt 700 --steps 64 --window 256 --sinks 4

A small stack of layers (RMSNorm, fused q/k/v projection, paged attention,
output projection, routed experts, residuals; random weights, hidden rows in
place of token embeddings) is run the way a server runs it:

  1. the prompts go in chunks of at most --chunk rows, all sequences in one
     call: extend the cache, then per layer write the chunk's keys and values
     and attend to everything before;
  2. every sequence branches: the branches share its pages, and the first
     step copies only a partly full last page;
  3. all branches decode in lockstep, one row each, under an optional sliding
     window with first tokens (sinks) that stay visible;
  4. half the branches end, the cache is compacted, the rest go on.

On the way it checks what must hold: the decode and the prompt kernel agree on
a step's rows, and a step's attention is the same, bit for bit, before and
after compaction. Prints one JSON line with the rates, the pages in use and
what they would be without sharing.
"""
from __future__ import annotations

import argparse
import json
import time

import numpy as np

from . import ggml as G


class Stack:
    """Random layers on one Context; caches of `max_len` positions a sequence."""

    def __init__(self, torch, ctx, n_layer=2, d=512, n_head=8, n_kv=2, hd=64, experts=8, top_k=2, ff=512, seed=0):
        self.torch, self.ctx = torch, ctx
        self.n_layer, self.d, self.n_head, self.n_kv, self.hd = n_layer, d, n_head, n_kv, hd
        rng = np.random.default_rng(seed)
        w = lambda rows, cols: rng.standard_normal((rows, cols), dtype=np.float32) * np.float32(cols ** -0.5)
        for l in range(n_layer):
            qkv, o = w((n_head + 2 * n_kv) * hd, d), w(d, n_head * hd)
            ctx.upload_dense(2 * l, G.Q8_0, G.quantize(G.Q8_0, qkv), *qkv.shape)
            ctx.upload_dense(2 * l + 1, G.Q8_0, G.quantize(G.Q8_0, o), *o.shape)
            gate, up, down = (G.quantize(t, w(r, c)) for t, r, c in
                              ((G.Q4_K, experts * ff, d), (G.Q4_K, experts * ff, d), (G.Q6_K, experts * d, ff)))
            ctx.upload_experts(l, experts, d, ff, G.Q4_K, gate, G.Q4_K, up, G.Q6_K, down)
            ctx.upload_router(l, w(experts, d), top_k)

    def cache(self, cache_id, n_seq, max_len, n_pages, page=32):
        t = self.torch
        shape = (self.n_layer, n_pages, self.n_kv, page, self.hd)
        self.k, self.v = (t.zeros(shape, dtype=t.float16, device="cuda") for _ in range(2))
        i32 = dict(dtype=t.int32, device="cuda")
        self.table = t.full((n_seq, -(-max_len // page)), -1, **i32)
        self.length, self.refs = t.zeros(n_seq, **i32), t.zeros(n_pages, **i32)
        self.id, self.page = cache_id, page
        self.ctx.kv_cache(cache_id, self.k, self.v, self.table, self.length, self.refs)

    def norm(self, h):
        return h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()

    def forward(self, h, seqs, row_start=None, window=0, sinks=0, probe=None):
        """Rows h [n, d]: the last positions of `seqs` (already extended), one
        each or row_start's ranges. probe(layer, q, out) sees each attention."""
        t, ctx = self.torch, self.ctx
        nq, nkv, hd = self.n_head, self.n_kv, self.hd
        for l in range(self.n_layer):
            qkv = t.empty((h.shape[0], (nq + 2 * nkv) * hd), device="cuda")
            ctx.matmul_dev(2 * l, self.norm(h), qkv)
            # Queries, keys and values stay slices of the fused rows.
            q, k, v = (x.unflatten(1, (-1, hd)) for x in qkv.split([nq * hd, nkv * hd, nkv * hd], 1))
            ctx.kv_write_dev(self.id, l, k, v, seqs=seqs, row_start=row_start)
            a = t.empty((h.shape[0], nq, hd), device="cuda")
            if row_start is None:
                ctx.attn_decode_dev(self.id, l, q, a, seqs=seqs, window=window, sinks=sinks)
            else:
                ctx.attn_prompt_dev(self.id, l, q, row_start, a, seqs=seqs, window=window, sinks=sinks)
            if probe:
                probe(l, q, a)
            o = t.empty_like(h)
            ctx.matmul_dev(2 * l + 1, a.flatten(1), o)
            h = h + o
            f = t.empty_like(h)
            ctx.moe_ffn_dev(l, self.norm(h), f)
            h = h + f
        return h


def run(sequences=4, branches=3, prompt=300, steps=32, chunk=256, window=0, sinks=0, page=32, seed=0):
    import torch

    from .cuda import Context
    ctx = Context(torch.cuda.current_device())
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    try:
        s = Stack(torch, ctx, seed=seed)
        rng = np.random.default_rng(seed)
        lens = [int(n) for n in rng.integers(max(1, prompt // 2), prompt + 1, sequences)]
        kids = sequences * branches
        held = lambda n: -(-n // page)
        most = sum(held(n) for n in lens) + kids * (held(steps) + 2)
        s.cache(0, sequences + kids, max(lens) + steps, most, page)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        gen = torch.Generator(device="cuda").manual_seed(seed)

        # 1. prompts, chunk by chunk
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        last = torch.empty((sequences, s.d), device="cuda")
        for at in range(0, max(lens), chunk):
            who = [i for i in range(sequences) if lens[i] > at]
            counts = [min(chunk, lens[i] - at) for i in who]
            start = [0] + [int(x) for x in np.cumsum(counts)]
            ctx.kv_extend_dev(0, i32(who), i32(counts))
            h = s.forward(torch.randn((start[-1], s.d), generator=gen, device="cuda"), i32(who), i32(start), window,
                          sinks)
            for j, i in enumerate(who):
                last[i] = h[start[j + 1] - 1]
        ctx.sync()
        t_prompt = time.perf_counter() - t0

        # 2. branches share their parent's pages; the parents end
        kid = i32(list(range(sequences, sequences + kids)))
        ctx.kv_fork_dev(0, i32([i for i in range(sequences) for _ in range(branches)]), kid)
        ctx.kv_free_dev(0, i32(list(range(sequences))))
        h = last.repeat_interleave(branches, 0) + 0.1 * torch.randn((kids, s.d), generator=gen, device="cuda")

        # 3. decode in lockstep
        one, rows = i32([1] * kids), i32(list(range(kids + 1)))
        worst = 0.0

        def both(layer, q, a):
            nonlocal worst
            again = torch.empty_like(a)
            ctx.attn_prompt_dev(0, layer, q, rows, again, seqs=kid, window=window, sinks=sinks)
            worst = max(worst, float((again - a).abs().max() / a.abs().max()))

        t_decode = 0.0
        for step in range(steps // 2):
            torch.cuda.synchronize()
            t0 = time.perf_counter()
            ctx.kv_extend_dev(0, kid, one)
            h = s.norm(s.forward(h, kid, None, window, sinks, both if step == 0 else None))
            ctx.sync()
            t_decode += time.perf_counter() - t0 if step else 0.0
        live = int((s.refs > 0).sum())
        unshared = sum(held(int(n)) for n in s.length.tolist())

        # 4. every other branch ends; the pool is compacted; the rest go on
        gone, stay = kid[::2].contiguous(), kid[1::2].contiguous()
        ctx.kv_free_dev(0, gone)
        q = torch.randn((stay.numel(), s.n_head, s.hd), generator=gen, device="cuda")
        before, after = torch.empty_like(q), torch.empty_like(q)
        ctx.attn_decode_dev(0, 0, q, before, seqs=stay, window=window, sinks=sinks)
        n_live = i32([0])
        ctx.kv_compact_dev(0, n_live)
        ctx.attn_decode_dev(0, 0, q, after, seqs=stay, window=window, sinks=sinks)
        h = h[1::2].contiguous()
        for _ in range(steps - steps // 2):
            ctx.kv_extend_dev(0, stay, one[:stay.numel()])
            h = s.norm(s.forward(h, stay, None, window, sinks))
        ctx.sync()
        return {"prompt_rows_per_s": sum(lens) / t_prompt,
                "decode_rows_per_s": kids * (steps // 2 - 1) / t_decode if t_decode else None,
                "pages_live": live, "pages_without_sharing": unshared, "pages_after_compaction": int(n_live),
                "kernels_differ": worst, "same_after_compaction": bool(torch.equal(before, after)),
                "finite": bool(torch.isfinite(h).all())}
    finally:
        ctx.close()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("sequences", 4), ("branches", 3), ("prompt", 300), ("steps", 32), ("chunk", 256),
                        ("window", 0), ("sinks", 0), ("page", 32), ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=value)
    print(json.dumps(run(**vars(ap.parse_args()))))


if __name__ == "__main__":
    main()
