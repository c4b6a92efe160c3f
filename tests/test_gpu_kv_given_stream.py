"""Calls on a given stream whose outputs the call allocates: the memory stays
the call's until it has run, and the caller's until its own stream has read it."""
import pytest

from test_gpu_paged_attention import Problem

pytestmark = pytest.mark.gpu

BUSY = 40_000_000                    # cycles: some 20 ms, while a call takes microseconds


@pytest.fixture(scope="module")
def mb():
    import mars_b200
    return mars_b200


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def calls(mb, torch):
    """name -> (a call with stream=, that returns its outputs; their values)"""
    p = Problem(torch, [300, 40], [70, 5], 8, 2, 64, 16, "bfloat16")
    ctx = mb.KvContext(max_requests=2)
    i32 = dict(dtype=torch.int32, device="cuda")
    freq, axis, pos = torch.rand(32, device="cuda"), torch.zeros(32, **i32), torch.arange(75, **i32)
    spare = mb.KvCache(*(torch.zeros(5, 16, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)))
    lens, new = torch.tensor([3, 9], **i32), torch.tensor([40, 2], **i32)
    tables = torch.tensor([[0, -1, -1], [1, -1, -1]], **i32)
    free, count = torch.arange(2, 9, **i32), torch.tensor([7], **i32)
    stack, gone = torch.full((9,), -1, **i32), torch.tensor([1, 0], **i32)
    none = torch.zeros(1, **i32)
    x = torch.randn(75, 4, 64, device="cuda")
    made = {
        "attention": lambda stream: ctx.attention(p.q, mb.KvCache(p.k, p.v), p.d_tables, p.d_lens, p.cu, max_new=70,
                                                  return_lse=True, stream=stream),
        "rope": lambda stream: (mb.rope(x, pos, freq, axis, stream=stream),),
        "rope_append": lambda stream: (mb.rope_append(p.q, p.q[:, :2], p.q[:, :2], pos, freq, axis, spare, pos,
                                                      stream=stream),),
        "plan": lambda stream: ctx.plan(lens, new, tables.clone() if stream is None else tables, free, count, page_size=16,
                                        max_tokens=42, stream=stream),
        "release": lambda stream: ctx.release(lens, gone, tables, stack, none, page_size=16, stream=stream),
    }
    out = {}
    for name, call in made.items():
        want = [t.clone() for t in call(None)]
        torch.cuda.synchronize()
        out[name] = call, want
    return ctx, out


def handles(mb, torch, ctx):
    """A stream of torch's, and the context's own (NULL)."""
    s = torch.cuda.Stream()
    own = torch.cuda.ExternalStream(mb.lib().mars_kv_ctx_stream(ctx.handle))
    return [(s.cuda_stream, s), (0, own)]


NAMES = ["attention", "rope", "rope_append", "plan", "release"]


@pytest.mark.parametrize("name", NAMES)
def test_a_dropped_result_goes_to_nobody_before_the_call_has_run(mb, torch, name):
    ctx, all_calls = calls(mb, torch)
    call, want = all_calls[name]
    for handle, s in handles(mb, torch, ctx):
        if handle == 0 and name.startswith("rope"):
            continue                                       # no context: NULL is the default stream
        with torch.cuda.stream(s):
            torch.cuda._sleep(BUSY)
        got = call(handle)
        sizes = [t.untyped_storage().nbytes() for t in got]
        del got
        mine = [torch.full((n,), 77, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(4)]
        assert not s.query()                               # the call has still to run
        torch.cuda.synchronize()
        assert all((t == 77).all() for t in mine)


@pytest.mark.parametrize("name", NAMES)
def test_the_callers_stream_reads_before_the_next_call_writes(mb, torch, name):
    ctx, all_calls = calls(mb, torch)
    call, want = all_calls[name]
    for handle, s in handles(mb, torch, ctx):
        if handle == 0 and name.startswith("rope"):
            continue
        got = call(handle)
        here = torch.cuda.current_stream()
        here.wait_stream(s)
        torch.cuda._sleep(BUSY)
        copies = [t.clone() for t in got]
        places = {t.untyped_storage().data_ptr() for t in got}
        del got
        again = call(handle)                               # while the copies are still to be made
        assert not here.query()
        assert not places & {t.untyped_storage().data_ptr() for t in again}
        torch.cuda.synchronize()
        for a, b in zip(copies, want):
            assert torch.equal(a, b)
