"""A score that is not a number, of mars_paged_attention: the rows that see it
answer NaN in out and lse (lse = -inf says that a row sees nothing); every
other row keeps its answer.  Its last bits may move: rows that share a warp
move their maximum together.  Both answers are within their bound of the
definition (weights and result rounded to bf16, 2^-8 each, of at most max|v|;
scores off by e), so they are within twice that of one another."""
import math

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


def check_others(torch, p, got, want, got_lse, want_lse, bad):
    d = p.q.shape[2]
    norms = max(k.float().norm(dim=-1).nan_to_num().max().item() for k in p.keys) * 2 * d ** 0.5
    e = 2 * ((d + 4) * 2.0 ** -24 * norms * 0.125 + 2.0 ** -20 + 2.0 ** -20 * 20)
    top = max(v.abs().max().item() for v in p.values)
    assert ((got[~bad].float() - want[~bad].float()).abs() <= 2 * (2.0 ** -7 + 2 * e) * top).all()
    off = (got_lse[~bad] - want_lse[~bad]).abs()
    assert (off <= 2 * (e + 2.0 ** -21 * (1 + want_lse[~bad].abs()))).all()


# one part of a unit, and several that are joined
CACHED = [[40, 5], [3000, 5], [20000, 700]]
OPTIONS = [{}, dict(softcap=20.0), dict(scale=-0.1)]


@pytest.mark.parametrize("option", OPTIONS)
@pytest.mark.parametrize("cached", CACHED)
@pytest.mark.parametrize("new", [[1, 1], [90, 30]])
@pytest.mark.parametrize("d", [64, 128])
def test_a_query_of_nan(mb, torch, cached, new, d, option):
    p = Problem(torch, cached, new, 6, 2, d, 16, "bfloat16")
    want, want_lse = p.run(mb, **option)
    bad = torch.zeros(want_lse.shape, dtype=torch.bool, device="cuda")
    for token, head in [(0, 4), (new[0] - 1, 0), (sum(new) - 1, 5)]:
        p.q[token, head, d // 2] = math.nan
        bad[token, head] = True
    out, lse = p.run(mb, **option)
    assert out[bad].isnan().all()
    assert lse[bad].isnan().all()
    check_others(torch, p, out, want, lse, want_lse, bad)


@pytest.mark.parametrize("option", OPTIONS)
@pytest.mark.parametrize("cached", CACHED)
@pytest.mark.parametrize("new", [[1, 1], [90, 30]])
@pytest.mark.parametrize("d", [64, 128])
def test_a_key_of_nan(mb, torch, cached, new, d, option):
    """Key head 1 of request 0 has one in the middle of the cache, and one that only its last rows see."""
    p = Problem(torch, cached, new, 6, 2, d, 16, "bfloat16")
    want, want_lse = p.run(mb, **option)
    last = p.lens[0] - 1
    first = 0 if new[0] == 1 else last - 20            # seen by rows at and beyond it
    for at in (last, first):
        p.k[p.d_tables[0, at // 16].long(), at % 16, 1, 3] = math.nan
    out, lse = p.run(mb, **option)
    bad = torch.zeros(want_lse.shape, dtype=torch.bool, device="cuda")
    rows = torch.arange(new[0], device="cuda") + cached[0]
    bad[:new[0], 3:] = (rows >= first)[:, None]
    assert out[bad].isnan().all()
    assert lse[bad].isnan().all()
    check_others(torch, p, out, want, lse, want_lse, bad)
