"""Capped scores of mars_paged_attention, from caps far below the scores to caps
so far above that they cap nothing: the error has to follow the score, not the
cap.

Tolerances, from the definition, before any run, as in
test_gpu_paged_attention.py but for the cap's term: a score is off by at most
e = 2 ((D + 4) 2^-24 max|q||k| |scale| + 2^-20 + 2^-20 max|capped score|): the
product's error passes through the cap unamplified (the slope of tanh is at
most 1); the capped score itself is relative to its own size, a polynomial fit
to 2^-24.5 in eight fp32 operations where |score| is at most half the cap, and
1 - 2 / (1 + e^2x) beyond it, whose few units of 2^-24 stand beside tanh 1/2 =
0.46."""
import math

import pytest

from test_gpu_paged_attention import UNIT, Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mb():
    import mars_b200
    return mars_b200


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def check(torch, p, out, lse, softcap, scale):
    d, hq = p.q.shape[2], p.q.shape[1]
    group = hq // p.k.shape[2]
    u = UNIT[p.dtype]
    tokens = 0
    for b, n in enumerate(p.lens):
        rows = slice(tokens, tokens + p.new[b])
        tokens += p.new[b]
        q = p.q[rows].double().transpose(0, 1)
        kd = p.keys[b].double().permute(1, 2, 0).repeat_interleave(group, 0)
        vd = p.values[b].double().transpose(0, 1).repeat_interleave(group, 0)
        seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - p.new[b], n, device="cuda")[:, None]
        s = softcap * torch.tanh(q @ kd * scale / softcap)
        e = 2 * ((d + 4) * 2.0 ** -24 * abs(scale) * (q.norm(dim=-1).max() * kd.norm(dim=1).max()).item() + 2.0 ** -20 +
                 2.0 ** -20 * s.abs().max().item())
        s = torch.where(seen, s, -math.inf)
        want_lse = torch.logsumexp(s, -1)
        w = torch.exp(s - want_lse[..., None])
        want, mean = w @ vd, w @ vd.abs()
        limit = u * mean + u * want.abs() + 2 * e * mean + 1e-12
        if p.dtype == "float16":
            limit = limit + n * 2.0 ** -25 * vd.abs().max().item() + 2.0 ** -25
        off = (lse[rows].double().T - want_lse).abs()
        assert (off <= e + 2.0 ** -21 * (1 + want_lse.abs())).all(), f"request {b}: lse off by {off.max().item()}, e {e}"
        err = (out[rows].double().transpose(0, 1) - want).abs()
        assert (err <= limit).all(), f"request {b}: out off by {(err / limit).max().item()} of the limit"


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 2, 1], [150, 40, 70]])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("softcap", [0.3, 5.0, 50.0, 1e3, 1e5, 1e8, 1e20, 1e36, 3.4e38])
@pytest.mark.parametrize("qscale", [1.0, 40.0])
def test_the_error_follows_the_score(mb, torch, softcap, qscale, d, new, dtype):
    p = Problem(torch, [700, 0, 90], new, 4, 2, d, 16, dtype, qscale=qscale)
    for scale in (d ** -0.5, -d ** -0.5):
        out, lse = p.run(mb, softcap=softcap, scale=scale)
        check(torch, p, out, lse, softcap, scale)


@pytest.mark.parametrize("new", [[1, 1], [70, 5]])
def test_a_prompt_row_and_the_same_row_alone_agree(mb, torch, new):
    """The kernel for chunks and the one for single tokens, both within the bound of one score."""
    p = Problem(torch, [300, 40], new, 4, 2, 64, 16, "bfloat16")
    out, lse = p.run(mb, softcap=1e6)
    out1, lse1 = p.run(mb, softcap=1e6, max_new=1)
    e = 2 * (68 * 2.0 ** -24 * 0.125 * 2 * 64 + 2.0 ** -20 + 2.0 ** -20 * 16)      # norms of 64 normal values: below 11.3
    assert (lse - lse1).abs().max().item() <= 2 * (e + 2.0 ** -21 * (1 + lse.abs().max().item()))


@pytest.mark.parametrize("new", [[1, 1], [70, 5]])
@pytest.mark.parametrize("softcap", [1e-30, 1e-42])
def test_caps_that_leave_no_score(mb, torch, new, softcap):
    """scale / softcap is beyond fp32 for the smaller one: scores of zero stay zero, the others are at most the cap."""
    p = Problem(torch, [300, 40], new, 4, 2, 64, 16, "bfloat16")
    p.q[0].zero_()
    out, lse = p.run(mb, softcap=softcap)
    check(torch, p, out, lse, softcap, 0.125)
