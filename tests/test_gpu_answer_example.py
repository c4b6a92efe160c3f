"""The retrieval-to-attention example, run whole: its outputs against dense
attention in 64 bits over the same projections, and its pages all free again.

Queries and keys are rounded to bf16 after their rotation there as here, so
what differs is the softmax weights' rounding and the output's (2^-8 each at
most) and a few scores whose rotation falls on the other side of a rounding:
2^-6 in the 2-norm."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def rotate(x, positions, freq, axis):
    import torch
    theta = positions[:, axis.long()].double() * freq.double()
    c, s = torch.cos(theta)[:, None], torch.sin(theta)[:, None]
    a, b = x.double().chunk(2, dim=-1)
    return torch.cat([a * c - b * s, a * s + b * c], dim=-1).to(torch.bfloat16).double()


def test_example_answers_with_its_memories():
    import torch
    import answer_with_memories as ex
    kept = []
    question, top_k = (9, 1, 30, 17), 16
    outs, count, pages, layer = ex.answer(question=question, top_k=top_k, steps=3, keep=kept)
    assert count.item() == pages
    keys, values = [[] for _ in question], [[] for _ in question]
    for x, positions, plan, out in kept:
        assert plan.status.item() == 0
        q, k, v = layer.project(x)
        q, k = rotate(q, positions, layer.freq, layer.axis), rotate(k, positions, layer.freq, layer.axis)
        first = plan.cu_new.tolist()
        for b in range(len(question)):
            rows = slice(first[b], first[b + 1])
            keys[b].append(k[rows])
            values[b].append(v[rows].double())
            kk, vv = torch.cat(keys[b]).repeat_interleave(3, 1), torch.cat(values[b]).repeat_interleave(3, 1)
            n, new = len(kk), first[b + 1] - first[b]
            assert n == plan.kv_lens[b].item()
            s = torch.einsum("ihd,jhd->hij", q[rows], kk) / 8.0
            s = 30.0 * torch.tanh(s / 30.0)
            i, j = torch.arange(n - new, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
            s = s - layer.decay.double()[:, None, None] * (i - j).clamp(min=0)
            s = s.masked_fill(~((j <= i) | (j < top_k)), float("-inf"))
            want = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), vv)
            off = (out[rows].double() - want).norm() / want.norm()
            assert off <= 2.0 ** -6, f"request {b}: {off}"
