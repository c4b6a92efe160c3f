"""What a row of mars_paged_attention must not depend on: the other requests'
queries, padding tokens, what lies in the cache beyond a request's length, and
what the launch before left in shared memory.  The request lengths, and with
them the split of the work, stay as they are, so every bit has to."""
import math

import numpy as np
import pytest

from test_gpu_paged_attention import Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mb():
    import mars_b200
    return mars_b200


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def crowd(torch, mb, ctx, size):
    """A launch that fills every CTA's shared memory with queries and keys of this size."""
    p = Problem(torch, [600] * 8, [256] * 8, 8, 2, 128, 32, "bfloat16", seed=77)
    p.q.fill_(size)
    p.k.nan_to_num_(nan=size)
    p.run(mb, ctx)


# query heads of a key head that fill a row tile (4), and that leave rows of it empty (3: two, 5: three, 12: eight)
@pytest.mark.parametrize("hq,hkv", [(8, 2), (6, 2), (5, 1), (12, 1)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("option", [{}, dict(softcap=20.0), dict(window=300), dict(softcap=30.0, decay=True)])
@pytest.mark.parametrize("new", [[100, 37, 60], [9, 5, 7]])
def test_a_request_has_its_bits_whoever_stands_beside_it(mb, torch, hq, hkv, d, option, new):
    option = dict(option)
    if option.pop("decay", False):
        option["decay"] = torch.linspace(0.001, 0.02, hq, device="cuda")
    cached = [900, 300, 417]
    p = Problem(torch, cached, new, hq, hkv, d, 32, "bfloat16", seed=hq * d)
    ctx = mb.KvContext(max_requests=8)
    q = torch.cat([p.q, torch.zeros(40, hq, d, device="cuda", dtype=p.q.dtype)])      # and padding
    own = slice(0, new[0])

    def answer(neighbours, padding, stale, before):
        """Request 0's rows; the rest of the call is made of the given sizes."""
        x = q.clone()
        x[new[0]:sum(new)] *= neighbours
        x[sum(new):] = padding
        # slots of the pages that lie beyond their request's length, and pages of nobody
        j = torch.arange(p.k.shape[1], device="cuda")
        used = torch.zeros(p.k.shape[:2], dtype=torch.bool, device="cuda")
        for b, n in enumerate(p.lens):
            pages = torch.from_numpy(p.tables[b, :-(-n // p.page)].astype(np.int64)).cuda()
            at = torch.arange(len(pages), device="cuda")[:, None] * p.page + j
            used[pages] = at < n
        p.k[~used], p.v[~used] = stale, stale
        if before is not None:
            crowd(torch, mb, ctx, before)
        out, lse = ctx.attention(x, mb.KvCache(p.k, p.v), p.d_tables, p.d_lens, p.cu, max_new=max(new),
                                 return_lse=True, **option)
        return out[own].clone(), lse[own].clone()

    want = answer(1.0, 0.0, 0.0, 0.0)
    assert want[0].isfinite().all() and want[1].isfinite().all()
    for neighbours, padding, stale, before in [
            (50.0, 0.0, 0.0, 0.0), (-1000.0, 300.0, 0.0, 0.0), (1.0, math.nan, math.nan, 0.0),
            (1.0, math.inf, 1e4, 0.0), (1.0, 0.0, 0.0, 1e3), (1.0, 0.0, 0.0, -20.0), (math.nan, 5.0, -300.0, 40.0)]:
        got = answer(neighbours, padding, stale, before)
        for a, b, name in zip(got, want, ("out", "lse")):
            assert torch.equal(a, b), f"{name} differs in {(a != b).sum().item()} of {a.numel()} places " \
                                      f"(neighbours {neighbours}, padding {padding}, stale {stale}, before {before})"
