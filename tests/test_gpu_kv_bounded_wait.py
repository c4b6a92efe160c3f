"""The attention kernels' bounded waits give up cleanly.

The test hook mars_kv_ctx_debug_wait makes the next call's first CTA load
nothing, so that its waits (barriers that nothing completes) run out after a
few milliseconds.  No GPU fault is involved: the kernel records the wait, ends
and leaves the context usable.  The test checks that

* rows without a result are NaN in out and lse, the others keep their bits;
* the status reaches the host as MARS_ERR_TIMEOUT, once, through
  mars_kv_ctx_status or through the next call, which does nothing;
* calls that were queued behind the failed one, the call after the report and
  replays of captured calls are bit-identical to those of an untouched context."""
import pytest

from test_gpu_paged_attention import Problem

pytestmark = pytest.mark.gpu

LIMIT = 20_000_000                   # 20 ms; a call takes microseconds


@pytest.fixture(scope="module")
def mb():
    import mars_b200
    return mars_b200


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


# few tokens and chunks; units of one part, and cut into several
CASES = [([40, 90, 5], [1, 1, 1]), ([9000, 300, 5000], [1, 2, 1]), ([0, 40, 3], [100, 30, 1]), ([6000, 900, 0], [90, 200, 400])]


def make(mb, torch, cached, new):
    p = Problem(torch, cached, new, 8, 2, 128, 32, "bfloat16")
    ctx = mb.KvContext(max_requests=3)
    want = p.run(mb, ctx)
    ctx.status()
    return p, ctx, want


def same(torch, got, want):
    return torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def marked(torch, got, want):
    """Some rows are NaN, in out and lse alike; the others are as they should be."""
    out, lse = got
    bad = lse.isnan()
    assert bad.any()
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad)
    assert torch.equal(out[~bad], want[0][~bad]) and torch.equal(lse[~bad], want[1][~bad])


def timed_out(mb, call, *args):
    with pytest.raises(mb.MarsError) as e:
        call(*args)
    assert e.value.status == mb.MARS_ERR_TIMEOUT and "gave up" in str(e.value)


@pytest.mark.parametrize("cached,new", CASES)
def test_a_wait_that_gives_up_is_marked_and_reported_once(mb, torch, cached, new):
    p, ctx, want = make(mb, torch, cached, new)
    ctx.debug_wait(LIMIT, True)
    got = p.run(mb, ctx)
    timed_out(mb, ctx.status)
    marked(torch, got, want)
    ctx.status()
    assert same(torch, p.run(mb, ctx), want)              # the hook held for one call
    ctx.status()


@pytest.mark.parametrize("cached,new", CASES)
def test_the_next_call_reports_it_and_does_nothing(mb, torch, cached, new):
    p, ctx, want = make(mb, torch, cached, new)
    ctx.debug_wait(LIMIT, True)
    p.run(mb, ctx)
    torch.cuda.synchronize()
    out = torch.full_like(p.q, 7.0)
    timed_out(mb, lambda: p.run(mb, ctx, out=out))
    torch.cuda.synchronize()
    assert (out == 7).all()
    assert same(torch, p.run(mb, ctx), want)
    # and a call of another operator
    ctx.debug_wait(LIMIT, True)
    p.run(mb, ctx)
    torch.cuda.synchronize()
    i32 = dict(dtype=torch.int32, device="cuda")
    args = (torch.zeros(1, **i32), torch.ones(1, **i32), torch.full((1, 1), -1, **i32), torch.arange(1, **i32),
            torch.ones(1, **i32))
    timed_out(mb, lambda: ctx.plan(*args, page_size=8, max_tokens=1))
    assert ctx.plan(*args, page_size=8, max_tokens=1).slots.item() == 0


@pytest.mark.parametrize("cached,new", CASES)
def test_calls_queued_behind_it_find_nothing_of_it(mb, torch, cached, new):
    p, ctx, want = make(mb, torch, cached, new)
    for _ in range(3):
        ctx.debug_wait(LIMIT, True)
        got = [p.run(mb, ctx) for _ in range(4)]          # issued within the first one's 20 ms
        timed_out(mb, ctx.status)
        marked(torch, got[0], want)
        for again in got[1:]:
            assert same(torch, again, want)
        ctx.status()


@pytest.mark.parametrize("cached,new", [CASES[1], CASES[3]])
def test_replays(mb, torch, cached, new):
    p, ctx, want = make(mb, torch, cached, new)
    cache, outs = mb.KvCache(p.k, p.v), [torch.empty_like(p.q) for _ in range(3)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        for i, out in enumerate(outs):
            ctx.debug_wait(LIMIT, i == 1)                 # the second of three
            ctx.attention(p.q, cache, p.d_tables, p.d_lens, p.cu, max_new=max(new), out=out)
    for _ in range(2):
        for out in outs:
            out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[2], want[0])
        assert outs[1].isnan().any()
        timed_out(mb, ctx.status)
        ctx.status()
    assert same(torch, p.run(mb, ctx), want)


def test_refusals(mb):
    L = mb.lib()
    assert L.mars_kv_ctx_status(None) == mb.MARS_ERR_INVALID
    assert L.mars_kv_ctx_debug_wait(None, 0, 0) == mb.MARS_ERR_INVALID
