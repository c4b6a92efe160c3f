"""mars_kv_release / mars_kv_plan against the rules written out with Python
integers: every value is a whole number and has to be equal."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def plain_release(lens, gone, tables, free, count, page):
    lens, free = list(lens), list(free)
    for b, g in enumerate(gone):
        if g:
            pages = -(-lens[b] // page)
            free[count:count + pages] = tables[b][:pages]
            count += pages
            lens[b] = 0
    return lens, free, count


def plain_plan(lens, new, tables, free, count, page, max_tokens):
    tables = [list(r) for r in tables]
    slots, positions, first, after = [], [], [0], []
    for b, (n, add) in enumerate(zip(lens, new)):
        for col in range(-(-n // page), -(-(n + add) // page)):
            count -= 1
            tables[b][col] = free[count]
        for pos in range(n, n + add):
            slots.append(tables[b][pos // page] * page + pos % page)
            positions.append(pos)
        first.append(first[-1] + add)
        after.append(n + add)
    pad = [-1] * (max_tokens - len(slots))
    return after, tables, first, slots + pad, positions + pad, count


@pytest.fixture(scope="module")
def mb():
    import mars_b200
    return mars_b200


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def state(seed, B, page, longest, most_new, spare=3):
    """Lengths with zeros and ones among them, pages in no order, columns past a request's pages -1."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, longest + 1, B)
    new = rng.integers(0, most_new + 1, B)
    lens[rng.random(B) < 0.2] = 0
    new[rng.random(B) < 0.2] = 1
    lens[rng.random(B) < 0.2] //= page
    lens[rng.random(B) < 0.2] *= page            # ends on a page's edge
    lens = np.minimum(lens, longest)
    held = -(-lens // page)
    need = int((-(-(lens + new) // page) - held).sum())
    ids = rng.permutation(int(held.sum()) + need + spare)
    width = max(1, -(-(longest + most_new) // page))
    tables = np.full((B, width), -1)
    at = 0
    for b in range(B):
        tables[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    free = np.full(len(ids), -1)
    free[:len(ids) - at] = ids[at:]
    return lens, new, tables, free, len(ids) - at


CASES = [(1, 1, 5, 4), (1, 16, 0, 1), (3, 7, 40, 9), (17, 16, 100, 33), (64, 16, 4096, 1), (513, 32, 700, 64),
         (1000, 48, 300, 150), (2, 128, 1000, 100000), (8192, 64, 200, 20)]


@pytest.mark.parametrize("B,page,longest,most_new", CASES)
def test_plan_equals_the_rules(mb, B, page, longest, most_new):
    lens, new, tables, free, count = state(B, B, page, longest, most_new)
    total = int(new.sum())
    ctx = mb.KvContext(max_requests=B)
    for pad in (0, 5):
        t = dev(tables)
        p = ctx.plan(dev(lens), dev(new), t, dev(free), dev([count]), page_size=page, max_tokens=total + pad)
        after, want_t, first, slots, positions, left = plain_plan(lens, new, tables, free, count, page, total + pad)
        assert p.status.item() == 0
        assert p.kv_lens.tolist() == after
        assert p.cu_new.tolist() == first
        assert p.free_count.item() == left
        assert t.tolist() == want_t
        assert p.slots.tolist() == slots
        assert p.positions.tolist() == positions


@pytest.mark.parametrize("B,page,longest,most_new", CASES)
def test_release_equals_the_rules(mb, B, page, longest, most_new):
    lens, new, tables, free, count = state(100 + B, B, page, longest, most_new)
    gone = (np.random.default_rng(B).random(B) < 0.4).astype(np.int32) * 3
    gone[0] = 1
    ctx = mb.KvContext(max_requests=B)
    f = dev(free)
    status = dev([77])
    got_lens, got_count = ctx.release(dev(lens), dev(gone), dev(tables), f, dev([count]), page_size=page, status=status)
    want_lens, want_free, want_count = plain_release(lens.tolist(), gone, tables.tolist(), free.tolist(), count, page)
    assert status.item() == 0
    assert got_lens.tolist() == want_lens
    assert got_count.item() == want_count
    assert f.tolist() == want_free


def test_steps_in_place_return_every_page(mb):
    """A server's life on the same arrays: the pages in tables and on the stack stay a permutation."""
    import ctypes as C
    import torch
    B, page, pages = 33, 16, 900
    rng = np.random.default_rng(5)
    ctx = mb.KvContext(max_requests=B)
    lens, tables, free, count = dev(np.zeros(B)), dev(np.full((B, 40), -1)), dev(rng.permutation(pages)), dev([pages])
    cu, slots, status = dev(np.zeros(B + 1)), dev(np.zeros(4000)), dev([0])
    L, p = mb.lib(), lambda t: C.c_void_p(t.data_ptr())
    st = torch.cuda.current_stream().cuda_stream or 1
    for step in range(40):
        gone = dev(rng.random(B) < 0.1)
        assert L.mars_kv_release(ctx.handle, B, p(lens), p(gone), p(tables), 40, page, p(free), pages, p(count),
                                 p(lens), p(count), p(status), st) == 0
        assert status.item() == 0
        room = 640 - lens.cpu().numpy()
        new = np.minimum(room, rng.integers(0, 60, B))
        assert L.mars_kv_plan(ctx.handle, B, p(lens), p(dev(new)), p(tables), 40, page, p(free), pages, p(count),
                              4000, p(lens), p(count), p(cu), p(slots), None, p(status), st) == 0
        assert status.item() == 0
        held = -(-lens.cpu().numpy() // page)
        t = tables.cpu().numpy()
        used = np.concatenate([t[b, :held[b]] for b in range(B)] + [free.cpu().numpy()[:count.item()]])
        assert sorted(used.tolist()) == list(range(pages)), f"step {step}"


@pytest.mark.parametrize("what,bit", [("pages", "KV_NO_PAGES"), ("table", "KV_TABLE_FULL"),
                                      ("tokens", "KV_TOO_MANY_TOKENS"), ("negative", "KV_BAD_LENGTH"),
                                      ("huge", "KV_BAD_LENGTH"), ("count", "KV_STACK_FULL")])
def test_a_plan_that_does_not_fit_changes_nothing(mb, what, bit):
    B, page = 9, 16
    lens, new, tables, free, count = state(3, B, page, 100, 40)
    new[4] = 30
    limit = int(new.sum())
    if what == "pages":
        count = int((-(-(lens + new) // page) + (-lens // page)).sum()) - 1
    if what == "table":
        tables = tables[:, :int((-(-(lens + new) // page)).max()) - 1]
    if what == "tokens":
        limit -= 1
    if what == "negative":
        new[2] = -1
    if what == "huge":
        lens[2], new[2] = 2 ** 31 - 1, 1
    if what == "count":
        count = len(free) + 1
    ctx = mb.KvContext(max_requests=B)
    t = dev(tables)
    p = ctx.plan(dev(lens), dev(new), t, dev(free), dev([count]), page_size=page, max_tokens=limit)
    assert p.status.item() & getattr(mb, bit)
    assert p.kv_lens.tolist() == lens.tolist()
    assert p.free_count.item() == count
    assert t.tolist() == tables.tolist()
    assert set(p.cu_new.tolist()) == {0} and set(p.slots.tolist()) == {-1} and set(p.positions.tolist()) == {-1}
    # and the context still works
    lens, new, tables, free, count = state(4, B, page, 100, 40)
    p = ctx.plan(dev(lens), dev(new), dev(tables), dev(free), dev([count]), page_size=page, max_tokens=int(new.sum()))
    assert p.status.item() == 0


def test_a_release_that_does_not_fit_changes_nothing(mb):
    lens, _, tables, free, _ = state(8, 6, 16, 200, 1)
    lens[1] = 50
    full = dev(np.arange(len(free)))
    status = dev([0])
    ctx = mb.KvContext(max_requests=6)
    got, count = ctx.release(dev(lens), dev(np.ones(6)), dev(tables), full, dev([len(free)]), page_size=16, status=status)
    assert status.item() == mb.KV_STACK_FULL
    assert got.tolist() == lens.tolist() and count.item() == len(free)
    assert full.tolist() == list(range(len(free)))


def test_empty_calls(mb):
    ctx = mb.KvContext(max_requests=4)
    none, tables = dev(np.zeros(0)), dev(np.zeros((0, 1)))
    p = ctx.plan(none, none, tables, none, dev([0]), page_size=16, max_tokens=3)
    assert p.status.item() == 0 and p.cu_new.tolist() == [0] and p.slots.tolist() == [-1] * 3
    p = ctx.plan(dev([5, 0]), dev([0, 0]), dev([[2], [-1]]), none, dev([0]), page_size=8, max_tokens=0)
    assert p.status.item() == 0 and p.kv_lens.tolist() == [5, 0] and p.cu_new.tolist() == [0, 0, 0]


def test_calls_on_two_streams_are_ordered(mb):
    """The second call reads what the first, on another stream, has written with the context's memory."""
    import torch
    B, page = 512, 16
    lens, new, tables, free, count = state(11, B, page, 300, 40)
    want = plain_plan(lens, new, tables, free, count, page, int(new.sum()))
    ctx = mb.KvContext(max_requests=B)
    args = (dev(lens), dev(new), dev(tables), dev(free), dev([count]))
    torch.cuda.synchronize()
    plans = []
    for _ in range(6):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            plans.append(ctx.plan(*args, page_size=page, max_tokens=int(new.sum())))
    torch.cuda.synchronize()
    for p in plans:
        assert p.slots.tolist() == want[3] and p.free_count.item() == want[5]


def test_refusals(mb):
    with pytest.raises(mb.MarsError) as e:
        mb.KvContext(max_requests=0)
    assert e.value.status == mb.MARS_ERR_INVALID
    with pytest.raises(mb.MarsError) as e:
        mb.KvContext(max_requests=mb.KV_MAX_REQUESTS + 1)
    assert e.value.status == mb.MARS_ERR_INVALID
    ctx = mb.KvContext(max_requests=2)
    ok = dict(kv_lens=dev([1, 2]), new_lens=dev([1, 1]), tables=dev([[0], [1]]), free_pages=dev([2]),
              free_count=dev([1]), page_size=16, max_tokens=2)
    ctx.plan(**ok)
    with pytest.raises(mb.MarsError) as e:
        ctx.plan(**dict(ok, page_size=0))
    assert e.value.status == mb.MARS_ERR_INVALID
    with pytest.raises(mb.MarsError) as e:
        ctx.plan(**dict(ok, kv_lens=dev([1, 2, 3]), new_lens=dev([1, 1, 1]), tables=dev([[0], [1], [2]])))
    assert e.value.status == mb.MARS_ERR_CAPACITY
    with pytest.raises(ValueError):
        ctx.plan(**dict(ok, new_lens=dev([1])))
    with pytest.raises(ValueError):
        ctx.plan(**dict(ok, new_lens=dev([1, 1]).long()))
    with pytest.raises(ValueError):
        ctx.plan(**dict(ok, tables=dev(np.zeros((2, 4)))[:, ::2]))
