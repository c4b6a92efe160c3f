"""Retrieve memories on the GPU and attend to them, all on one device.

Every request's question is looked up in the memory store; the rows it finds
become the first tokens of its paged key/value cache (a prefix that all its
tokens see), the question's tokens follow, and then one token a step is
answered.  The projections are one random layer: the point is the path

    query_batch_topk -> plan -> rope_append -> attention -> ... -> release

whose ids, lengths, tables and slots never leave the GPU.  Run it with

    python examples/answer_with_memories.py
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "cuda-multimodal-memory_b200"))
import mars_b200  # noqa: E402
from mars_b200 import datagen  # noqa: E402

PAGE = 32
AXES = 3                                   # time, row, column


class Layer:
    """One attention layer over a paged cache: 768 columns, 12 query heads of 64, 4 key heads."""

    def __init__(self, pages, dim=768, hq=12, hkv=4, d=64, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.hq, self.hkv, self.d = hq, hkv, d
        self.w = (torch.randn(dim, (hq + 2 * hkv) * d, generator=g, device="cuda") * 2.0).to(torch.bfloat16)
        k, v = (torch.zeros(pages, PAGE, hkv, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        self.cache = mars_b200.KvCache(k, v)
        half = d // 2
        self.freq = torch.from_numpy((10000.0 ** (-np.arange(half) / half)).astype(np.float32)).cuda()
        self.axis = torch.arange(half, dtype=torch.int32, device="cuda") % AXES        # time, row, column in turn
        self.decay = 2.0 ** -torch.arange(4, 4 + hq, device="cuda", dtype=torch.float32)

    def project(self, x):
        return (x.to(torch.bfloat16) @ self.w).unflatten(1, (-1, self.d)).split([self.hq, self.hkv, self.hkv], dim=1)

    def step(self, ctx, x, positions, plan, tables, memories, max_new):
        """x: the new tokens of all requests back to back; their attention's output."""
        q, k, v = self.project(x)
        q = mars_b200.rope_append(q, k, v, positions, self.freq, self.axis, self.cache, plan.slots)
        return ctx.attention(q, self.cache, tables, plan.kv_lens, plan.cu_new, max_new=max_new, decay=self.decay,
                             softcap=30.0, prefix_lens=memories)


def text_positions(p):
    """Text stands at the same place on every axis."""
    return p[:, None].expand(-1, AXES).contiguous()


def answer(n_memories=20000, requests=4, top_k=16, question=(9, 1, 30, 17), steps=5, seed=1, keep=None):
    """Answers `steps` tokens for each request; the outputs of every step.  keep: a list that receives
    (x, positions, plan, output) of each step, for checks."""
    E, mod, ts, imp = datagen.gaussian_corpus(n_memories, 768, seed=seed, n_mod=4, ts_max=600.0)
    store = mars_b200.Store(n_memories, 768)
    store.upload(E, mod, ts, imp)
    rows, kinds = torch.from_numpy(E).cuda(), torch.from_numpy(mod).cuda()
    gen = torch.Generator(device="cuda").manual_seed(seed)

    # the questions' embeddings find their memories: [requests, top_k] ids, on the device
    batch = mars_b200.BatchContext(n_memories, 768, max_batch=requests, max_k=top_k)
    Q = torch.from_numpy(datagen.queries(requests, 768, seed=seed + 1)).cuda()
    ids = torch.empty(requests, top_k, dtype=torch.int32, device="cuda")
    vals = torch.empty(requests, top_k, device="cuda")
    batch.query_batch_topk(store, Q, requests, 600.0, 0.01, top_k, ids, vals, use_importance=True)

    pages = requests * 8
    layer = Layer(pages)
    ctx = mars_b200.KvContext(max_requests=requests)
    i32 = dict(dtype=torch.int32, device="cuda")
    lens = torch.zeros(requests, **i32)
    tables = torch.full((requests, 8), -1, **i32)
    free, count = torch.arange(pages, **i32), torch.tensor([pages], **i32)
    memories = torch.full((requests,), top_k, **i32)

    def run(x, positions, new, total, max_new):
        nonlocal lens, count
        plan = ctx.plan(lens, new, tables, free, count, page_size=PAGE, max_tokens=total)
        positions = positions(plan)
        out = layer.step(ctx, x, positions, plan, tables, memories, max_new)
        lens, count = plan.kv_lens, plan.free_count
        if keep is not None:
            keep.append((x, positions, plan, out))
        return out

    # prompt: each request's memories, then its question
    new = torch.tensor([top_k + n for n in question], **i32)
    words = [torch.randn(n, 768, generator=gen, device="cuda") for n in question]
    x = torch.cat([t for b in range(requests) for t in (rows[ids[b].long()], words[b])])
    kind = torch.cat([t for b in range(requests) for t in (kinds[ids[b].long()], torch.full((question[b],), -1, **i32))])

    def prompt_positions(plan):
        p = text_positions(plan.positions)
        p[:, 1] = torch.where(kind >= 0, 100 + 10 * kind, p[:, 1])        # a memory's row: its modality's band
        return p
    outs = [run(x, prompt_positions, new, len(x), int(top_k + max(question)))]

    # answer: the last output of each request makes its next token
    one = torch.ones(requests, **i32)
    last = outs[0][keep_last(new)]
    for _ in range(steps):
        x = last.flatten(1).float()
        out = run(x, lambda plan: text_positions(plan.positions), one, requests, 1)
        outs.append(out)
        last = out
    lens, count = ctx.release(lens, one, tables, free, count, page_size=PAGE)
    return outs, count, pages, layer


def keep_last(new):
    """The place of each request's last new token."""
    return torch.cumsum(new.long(), 0) - 1


if __name__ == "__main__":
    outs, count, pages, _ = answer()
    print(f"prompt {tuple(outs[0].shape)}, {len(outs) - 1} answered tokens a request, "
          f"{count.item()} of {pages} pages free again")
