"""Calls of one mars_kv_ctx on several streams: each starts after the one
before it, which is still pending when it is issued, also where the stream's
handle tells nothing (a destroyed stream's handle given to a new one, the
per-thread default stream)."""
import ctypes
import threading

import numpy as np
import pytest

from test_gpu_kv_plan import dev, plain_plan, state
from test_gpu_paged_attention import Problem

pytestmark = pytest.mark.gpu

PER_THREAD = 2                       # cudaStreamPerThread
BUSY = 40_000_000                    # cycles: some 20 ms, while a call takes microseconds


@pytest.fixture(scope="module")
def mb():
    import mars_b200
    return mars_b200


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def cudart():
    """The runtime that the library has loaded."""
    import mars_b200
    mars_b200.lib()
    with open("/proc/self/maps") as f:
        paths = {line.split()[-1] for line in f if "libcudart" in line}
    lib = ctypes.CDLL(sorted(paths)[0])
    lib.cudaStreamCreateWithFlags.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_uint]
    lib.cudaStreamDestroy.argtypes = [ctypes.c_void_p]
    return lib


def new_stream(cudart):
    h = ctypes.c_void_p()
    assert cudart.cudaStreamCreateWithFlags(ctypes.byref(h), 1) == 0      # cudaStreamNonBlocking
    return h.value


class Steps:
    """Two plans, the second of the first's lengths, count and tables; each with the arrays that it writes."""

    def __init__(self, mb, torch, seed):
        self.B, self.page = 300, 16
        rng = np.random.default_rng(seed)
        lens, new, tables, free, count = state(seed, self.B, self.page, 200, 40, spare=self.B * 4)
        more = rng.integers(0, 30, self.B)
        width = -(-(200 + 40 + 30) // self.page)
        wide = np.full((self.B, width), -1)
        wide[:, :tables.shape[1]] = tables[:, :width]
        self.total = [int(new.sum()), int(more.sum())]
        after, t, *_, left = plain_plan(lens, new, wide, free, count, self.page, self.total[0])
        self.want = plain_plan(after, more, t, free, left, self.page, self.total[1])
        self.ctx = mb.KvContext(max_requests=self.B)
        self.lens, self.new, self.more, self.tables, self.free, self.count = (
            dev(x) for x in (lens, new, more, wide, free, [count]))
        self.L = mb.lib()
        i32 = dict(dtype=torch.int32, device="cuda")
        self.out = [dict(lens=torch.zeros(self.B, **i32), count=torch.zeros(1, **i32), cu=torch.zeros(self.B + 1, **i32),
                         slots=torch.zeros(n, **i32), positions=torch.zeros(n, **i32), status=torch.zeros(1, **i32))
                    for n in self.total]
        torch.cuda.synchronize()

    def call(self, step, stream):
        p = lambda t: ctypes.c_void_p(t.data_ptr())
        o = self.out[step]
        lens, count = (self.lens, self.count) if step == 0 else (self.out[0]["lens"], self.out[0]["count"])
        new = self.new if step == 0 else self.more
        assert self.L.mars_kv_plan(self.ctx.handle, self.B, p(lens), p(new), p(self.tables), self.tables.shape[1], self.page,
                                   p(self.free), len(self.free), p(count), self.total[step], p(o["lens"]), p(o["count"]),
                                   p(o["cu"]), p(o["slots"]), p(o["positions"]), p(o["status"]), stream) == 0

    def check(self):
        after, tables, first, slots, positions, left = self.want
        o = self.out[1]
        assert o["status"].item() == 0
        assert o["lens"].tolist() == after and o["count"].item() == left and o["cu"].tolist() == first
        assert self.tables.tolist() == [list(r) for r in tables]
        assert o["slots"].tolist() == slots and o["positions"].tolist() == positions


def busy(torch, stream):
    with torch.cuda.stream(torch.cuda.ExternalStream(stream)):
        torch.cuda._sleep(BUSY)


def test_a_call_on_another_stream_follows_the_pending_one(mb, torch):
    for seed in range(3):
        s = Steps(mb, torch, seed)
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        busy(torch, a.cuda_stream)
        s.call(0, a.cuda_stream)
        s.call(1, b.cuda_stream)
        assert not a.query()                      # the first call was still pending
        torch.cuda.synchronize()
        s.check()


def test_a_new_stream_with_a_destroyed_ones_handle(mb, torch, cudart):
    s = Steps(mb, torch, 7)
    first = new_stream(cudart)
    busy(torch, first)
    s.call(0, first)
    marker = torch.cuda.Event()
    with torch.cuda.stream(torch.cuda.ExternalStream(first)):
        marker.record()
    assert cudart.cudaStreamDestroy(first) == 0   # its work goes on
    others = []
    second = new_stream(cudart)
    while second != first and len(others) < 32:   # where no handle comes back, this is the test before
        others.append(second)
        second = new_stream(cudart)
    s.call(1, second)
    assert not marker.query()
    torch.cuda.synchronize()
    s.check()
    for h in others + [second]:
        assert cudart.cudaStreamDestroy(h) == 0
    # the context's last stream is gone: the next call works
    t = Steps(mb, torch, 8)
    t.ctx = s.ctx
    t.call(0, torch.cuda.current_stream().cuda_stream or 1)
    t.call(1, torch.cuda.current_stream().cuda_stream or 1)
    torch.cuda.synchronize()
    t.check()


def test_the_default_streams_of_two_threads(mb, torch):
    s = Steps(mb, torch, 9)
    errors, marker = [], torch.cuda.Event()

    def work(step):
        try:
            if step == 0:
                with torch.cuda.stream(torch.cuda.ExternalStream(PER_THREAD)):
                    torch.cuda._sleep(BUSY)
            s.call(step, PER_THREAD)
            if step == 0:
                with torch.cuda.stream(torch.cuda.ExternalStream(PER_THREAD)):
                    marker.record()
            else:
                assert not marker.query()
        except BaseException as e:                # noqa: B902 -- shown by the test's thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:                             # one after the other; the first's work is pending
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    s.check()


@pytest.mark.parametrize("new", [1, 150])
def test_attention_of_two_problems_in_turn(mb, torch, new):
    """Units cut into parts, whose memory and counters the calls share: 24 calls on four streams, nothing waited for
    in between, give each problem's own bits."""
    problems = [Problem(torch, [5000, 77, 9000], [new, 1, new], 8, 2, 128, 32, "bfloat16", seed=1),
                Problem(torch, [300, 12000], [1, new], 12, 4, 64, 16, "bfloat16", seed=2)]
    want = [p.run(mb) for p in problems]
    ctx = mb.KvContext(max_requests=3)
    for p in problems:
        p.run(mb, ctx)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    with torch.cuda.stream(streams[0]):
        torch.cuda._sleep(BUSY)
    for i in range(24):
        p = problems[i % 2]
        with torch.cuda.stream(streams[i % 4]):
            got.append((i % 2, p.run(mb, ctx)))
    torch.cuda.synchronize()
    for which, (out, lse) in got:
        assert torch.equal(out, want[which][0]) and torch.equal(lse, want[which][1])
