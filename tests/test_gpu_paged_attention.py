"""mars_paged_attention against its definition in 64 bits.

Tolerances, from the definition, before any run.  With u the unit roundoff of
the type (2^-11 fp16, 2^-8 bf16), w_j the softmax's weights and A = sum_j w_j
|v_j|: the weights are rounded to the type once (u A), the result is rounded
once (u |out|), and a score is off by at most e = 2 ((D + 4) 2^-24 max|q||k|
|scale| + 2^-20 + 2^-21 |bias| + 2^-20 cap), which moves a weight by the factor 1 +- 2e (2 e A).
fp16 weights below 2^-14 keep 2^-25 absolute: n 2^-25 max|v| over n keys, and
the result 2^-25.  lse: e + 2^-21 (1 + |lse|)."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def mb():
    import mars_b200
    return mars_b200


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


class Problem:
    """Requests of cached[b] + new[b] tokens on shuffled pages.  Whatever no row may see is poisoned: NaN in every
    slot beyond a request's length and in pages of nobody, wild ids in the tables' unused columns."""

    def __init__(self, torch, cached, new, hq, hkv, d, page, dtype, layout="tokens", seed=0, qscale=1.0):
        rng = np.random.default_rng(seed)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.cached, self.new, self.page, self.dtype = cached, new, page, dtype
        dt = getattr(torch, dtype)
        lens = [c + n for c, n in zip(cached, new)]
        need = [-(-x // page) for x in lens]
        ids = rng.permutation(sum(need) + 5)
        width = max(1, max(need)) + 2
        self.tables = rng.choice([-1, 10 ** 9, -2 ** 31, 2 ** 31 - 1], (len(lens), width)).astype(np.int32)
        pages = len(ids)
        if layout == "heads":
            k, v = (torch.full((pages, hkv, page, d), math.nan, device="cuda", dtype=dt).transpose(1, 2) for _ in range(2))
        elif layout == "both":
            kv = torch.full((pages, 2, page, hkv, d), math.nan, device="cuda", dtype=dt)
            k, v = kv[:, 0], kv[:, 1]
        elif layout == "wide":
            k, v = (torch.full((pages, page, hkv, d + 16), math.nan, device="cuda", dtype=dt)[..., 8:8 + d] for _ in range(2))
        else:
            k, v = (torch.full((pages, page, hkv, d), math.nan, device="cuda", dtype=dt) for _ in range(2))
        self.keys, self.values, at = [], [], 0
        for b, n in enumerate(lens):
            mine = ids[at:at + need[b]]
            at += need[b]
            self.tables[b, :need[b]] = mine
            kb, vb = (torch.randn(n, hkv, d, generator=gen, device="cuda").to(dt) for _ in range(2))
            j = torch.arange(n, device="cuda")
            slot = torch.from_numpy(mine.astype(np.int64)).cuda()[j // page]
            k[slot, j % page] = kb
            v[slot, j % page] = vb
            self.keys.append(kb)
            self.values.append(vb)
        self.k, self.v, self.lens = k, v, lens
        total = sum(new)
        if layout == "wide":
            self.q = (torch.randn(total, hq + 2, d, generator=gen, device="cuda") * qscale).to(dt)[:, 1:hq + 1]
        else:
            self.q = (torch.randn(total, hq, d, generator=gen, device="cuda") * qscale).to(dt)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.d_lens = torch.tensor(lens, **i32)
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), **i32)
        self.d_tables = torch.from_numpy(self.tables).cuda()
        self.torch = torch

    def run(self, mb, ctx=None, **kw):
        ctx = ctx or mb.KvContext(max_requests=len(self.lens))
        kw.setdefault("max_new", max(self.new))
        return ctx.attention(self.q, mb.KvCache(self.k, self.v), self.d_tables, self.d_lens, self.cu, return_lse=True, **kw)

    def check(self, out, lse, scale=None, softcap=0.0, window=0, decay=None, prefix_lens=None, **_):
        torch = self.torch
        d, hq = self.q.shape[2], self.q.shape[1]
        group = hq // self.k.shape[2]
        scale = d ** -0.5 if scale is None else scale
        u = UNIT[self.dtype]
        tokens = 0
        for b, n in enumerate(self.lens):
            rows = slice(tokens, tokens + self.new[b])
            tokens += self.new[b]
            if self.new[b] == 0:
                continue
            q = self.q[rows].double().transpose(0, 1)                                         # hq, rows, d
            kd = self.keys[b].double().permute(1, 2, 0).repeat_interleave(group, 0)
            vd = self.values[b].double().transpose(0, 1).repeat_interleave(group, 0)
            i = torch.arange(n - self.new[b], n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            seen = j <= i
            if window:
                seen &= i - j < window
            if prefix_lens is not None:
                seen |= j < int(prefix_lens[b])
            s = q @ kd * scale
            e = 2 * ((d + 4) * 2.0 ** -24 * abs(scale) * (q.norm(dim=-1).max() * kd.norm(dim=1).max()).item() + 2.0 ** -20) \
                if n else 0.0
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                e += 2 * 2.0 ** -20 * softcap
            top_bias = 0.0
            if decay is not None:
                bias = decay.double()[:, None, None] * (i - j).clamp(min=0)
                s = s - bias
            s = torch.where(seen, s, -math.inf)
            want_lse = torch.logsumexp(s, -1) if n else torch.full(s.shape[:2], -math.inf, device="cuda", dtype=torch.float64)
            w = torch.exp(s - torch.where(want_lse.isfinite(), want_lse, 0.0)[..., None])
            if decay is not None:
                # the bias of the keys that weigh anything, by their weight
                top_bias = ((w * bias).sum(-1)).max().item()
                e += 2 * 2.0 ** -21 * top_bias
            want, mean = w @ vd, w @ vd.abs()
            limit = u * mean + u * want.abs() + 2 * e * mean + 1e-12
            if self.dtype == "float16":
                limit = limit + (n * 2.0 ** -25 * vd.abs().max().item() if n else 0) + 2.0 ** -25
            err = (out[rows].double().transpose(0, 1) - want).abs()
            assert (err <= limit).all(), f"request {b}: out off by {(err / limit).max().item()} of the limit"
            got = lse[rows].double().T
            assert torch.equal(got.isfinite(), want_lse.isfinite()), f"request {b}: finite lse"
            fin = want_lse.isfinite()
            assert (got[~fin] == -math.inf).all() and (out[rows].transpose(0, 1)[~fin] == 0).all()
            off = (got[fin] - want_lse[fin]).abs()
            assert (off <= e + 2.0 ** -21 * (1 + want_lse[fin].abs())).all(), f"request {b}: lse off by {off.max().item()}"


def check(mb, torch, cached, new, hq, hkv, d, page, dtype, layout="tokens", seed=0, qscale=1.0, ctx=None, **kw):
    p = Problem(torch, cached, new, hq, hkv, d, page, dtype, layout, seed, qscale)
    out, lse = p.run(mb, ctx, **kw)
    p.check(out, lse, **kw)
    return p, out, lse


DTYPES = ["float16", "bfloat16"]
# heads: no sharing, 2, 3, 5, 8 and 16 queries a key head, odd head counts
HEADS = [(1, 1), (4, 2), (9, 3), (5, 1), (8, 1), (16, 1), (12, 12)]
DIMS = [8, 16, 40, 64, 72, 80, 96, 120, 128]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_single_tokens_ragged(mb, torch, hq, hkv, dtype):
    """One new token each, caches from nothing to several splits, ends on and beside page and tile edges."""
    check(mb, torch, [0, 1, 7, 15, 16, 31, 63, 64, 65, 127, 128, 500, 1023, 2500], [1] * 14, hq, hkv, 64, 16, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", DIMS)
def test_head_dims(mb, torch, d, dtype):
    check(mb, torch, [100, 3, 260], [1, 1, 1], 6, 2, d, 16, dtype, seed=d)
    check(mb, torch, [100, 0, 260], [70, 33, 1], 6, 2, d, 16, dtype, seed=d + 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [8, 16, 24, 40, 48, 64, 128, 200, 256])
def test_page_sizes(mb, torch, page, dtype):
    check(mb, torch, [300, 0, 515], [1, 1, 1], 4, 2, 64, page, dtype, seed=page)
    check(mb, torch, [300, 0, 515], [90, 300, 17], 4, 2, 128, page, dtype, seed=page + 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["heads", "both", "wide"])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 140, 1]])
def test_layouts(mb, torch, layout, new, dtype):
    check(mb, torch, [77, 300, 129], new, 8, 2, 80, 32, dtype, layout=layout)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv", HEADS + [(32, 1), (7, 1), (48, 2), (128, 1), (65, 1)])
def test_chunks(mb, torch, hq, hkv, dtype):
    check(mb, torch, [0, 200, 64, 1], [130, 5, 64, 1], hq, hkv, 64, 16, dtype, seed=hq)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[0, 1, 0, 2], [1, 0, 1, 1], [3, 16, 1, 0], [128, 127, 129, 0], [256, 0, 257, 255], [600, 1, 0, 33]])
@pytest.mark.parametrize("cached", [[0, 0, 0, 0], [100, 0, 1, 1000]])
def test_requests_without_new_tokens_and_edges(mb, torch, new, cached, dtype):
    check(mb, torch, cached, new, 6, 2, 128, 32, dtype)


OPTIONS = [dict(softcap=5.0), dict(softcap=50.0, decay=True), dict(decay=True), dict(window=1), dict(window=37),
           dict(window=300, decay=True), dict(prefix=[0, 150, 1000, 3]), dict(prefix=[10, 64, 300, 1], window=20),
           dict(prefix=[90, 128, 129, 400], window=100, softcap=20.0, decay=True), dict(scale=0.0), dict(scale=-0.3)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [2, 4, 1, 3], [90, 300, 140, 5]])
@pytest.mark.parametrize("option", OPTIONS)
def test_options(mb, torch, option, new, dtype):
    option = dict(option)
    cached = [150, 600, 0, 900]
    if option.pop("decay", False):
        option["decay"] = torch.tensor([0.5, 0.03, 0.0, 0.2, 0.001, 2.0], device="cuda")
    if "prefix" in option:
        lens = [c + n for c, n in zip(cached, new)]
        option["prefix_lens"] = torch.tensor([min(p, n) for p, n in zip(option.pop("prefix"), lens)],
                                             dtype=torch.int32, device="cuda")
    check(mb, torch, cached, new, 6, 2, 64, 16, dtype, **option)
    check(mb, torch, cached, new, 6, 2, 128, 48, dtype, **option)


@pytest.mark.parametrize("dtype", DTYPES)
def test_peaked_scores(mb, torch, dtype):
    """Scores of hundreds: one key decides, the running maximum jumps."""
    check(mb, torch, [700, 0], [1, 1], 4, 2, 64, 16, dtype, qscale=40.0)
    check(mb, torch, [700, 0], [60, 500], 4, 2, 128, 16, dtype, qscale=40.0)


@pytest.mark.parametrize("growing", [True, False])
@pytest.mark.parametrize("new", [1, 40, 300])
def test_scores_in_order(mb, torch, new, growing):
    """Scores that rise (or fall) along the cache by 0.2 a key: the maximum moves at every step, or never."""
    p = Problem(torch, [2000], [new], 2, 1, 64, 16, "bfloat16")
    n = 2000 + new
    ramp = torch.arange(n, device="cuda").float() * 0.2 * (1 if growing else -1)
    kb = torch.zeros(n, 1, 64, device="cuda", dtype=torch.bfloat16)
    hi = ramp.bfloat16()
    kb[:, 0, 0], kb[:, 0, 1] = hi, (ramp - hi.float()).bfloat16()
    p.keys[0] = kb
    j = torch.arange(n, device="cuda")
    p.k[p.d_tables[0].long()[j // 16], j % 16] = kb
    p.q.zero_()
    p.q[..., :2] = 1.0
    out, lse = p.run(mb, scale=1.0)
    p.check(out, lse, scale=1.0)


@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_rows_that_see_nothing(mb, torch, new):
    """More new tokens than the cache holds: the first rows stand before its start.  And a request of length 0."""
    p = Problem(torch, [20, 50], new, 4, 2, 64, 16, "bfloat16")
    short = [max(0, n - 7) if n > 1 else 0 for n in new]      # as if only these were there
    p.d_lens.copy_(torch.tensor(short))
    p.lens = short
    p.keys = [k[:n] for k, n in zip(p.keys, short)]
    p.values = [v[:n] for v, n in zip(p.values, short)]
    out, lse = p.run(mb)
    p.check(out, lse)
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()


def test_a_wrong_bound_on_new_tokens_is_only_slow(mb, torch):
    p = Problem(torch, [10, 300, 0], [1, 200, 40], 8, 2, 64, 16, "bfloat16")
    for bound in (1, 2, 200, 10 ** 6):
        out, lse = p.run(mb, max_new=bound)
        p.check(out, lse)


@pytest.mark.parametrize("new", [1, 200])
def test_long_cache_and_offsets_past_32_bits(mb, torch, new):
    """A cache of 5 GB (2.6e9 values): the request's pages lie at both ends."""
    page, hkv, d = 64, 8, 128
    pages = 40000
    k = torch.zeros(pages, page, hkv, d, device="cuda", dtype=torch.bfloat16)
    v = torch.zeros(pages, page, hkv, d, device="cuda", dtype=torch.bfloat16)
    p = Problem(torch, [3000], [new], 16, hkv, d, page, "bfloat16")
    need = -(-p.lens[0] // page)
    ids = [pages - 1 - i if i % 2 else i for i in range(need)]
    for i, at in enumerate(ids):
        k[at], v[at] = p.k[p.d_tables[0, i].long()], p.v[p.d_tables[0, i].long()]
    p.k, p.v = k, v
    p.d_tables[0, :need] = torch.tensor(ids, dtype=torch.int32)
    out, lse = p.run(mb)
    p.check(out, lse)


def test_many_requests_and_long_ones(mb, torch):
    rng = np.random.default_rng(3)
    check(mb, torch, rng.integers(0, 400, 300).tolist(), [1] * 300, 8, 2, 64, 16, "float16")
    check(mb, torch, [70000, 5, 30000], [1, 1, 1], 8, 2, 64, 64, "bfloat16")
    check(mb, torch, [20000, 5, 9000], [30, 100, 1], 8, 2, 128, 64, "bfloat16")
    check(mb, torch, rng.integers(0, 200, 60).tolist(), rng.integers(0, 60, 60).tolist(), 4, 2, 128, 16, "bfloat16")


@pytest.mark.parametrize("new", [1, 150])
def test_the_same_bits_every_time_and_on_any_stream(mb, torch, new):
    p = Problem(torch, [5000, 77, 900], [new, 1, new], 8, 2, 128, 32, "bfloat16")
    ctx = mb.KvContext(max_requests=3)
    out, lse = p.run(mb, ctx)
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(torch.cuda.Stream()):
            again, lse2 = p.run(mb, ctx)
        torch.cuda.synchronize()
        assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("new", [1, 100])
def test_graph_replay_with_other_lengths(mb, torch, new):
    """A captured call reads its lengths on the GPU: a replay after they grew answers for the new ones."""
    p = Problem(torch, [900, 400], [new, new], 4, 2, 64, 16, "float16")
    ctx = mb.KvContext(max_requests=2)
    cache = mb.KvCache(p.k, p.v)
    out = torch.empty_like(p.q)
    lens = p.d_lens.clone()
    lens -= torch.tensor([700, 300], dtype=torch.int32, device="cuda")
    ctx.attention(p.q, cache, p.d_tables, lens, p.cu, max_new=new, out=out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        ctx.attention(p.q, cache, p.d_tables, lens, p.cu, max_new=new, out=out)
    lens.copy_(p.d_lens)
    g.replay()
    want, lse = p.run(mb, ctx)
    assert torch.equal(out, want)
    p.check(want, lse)


def test_padding_tokens_and_pages_out_of_range(mb, torch):
    p = Problem(torch, [40, 90], [1, 3], 4, 2, 64, 16, "bfloat16")
    ctx = mb.KvContext(max_requests=2)
    q = torch.cat([p.q, torch.full_like(p.q, math.nan)])
    out = torch.full_like(q, 7.0)
    ctx.attention(q, mb.KvCache(p.k, p.v), p.d_tables, p.d_lens, p.cu, max_new=3, out=out)
    want, lse = p.run(mb, ctx)
    assert torch.equal(out[:4], want) and (out[4:] == 7).all()
    # a page of nowhere reads as zeros
    for page in (-1, len(p.k), 2 ** 31 - 1):
        p.d_tables[1, 2] = page
        p.keys[1][32:48] = 0
        p.values[1][32:48] = 0
        got, lse = p.run(mb, ctx)
        p.check(got, lse)


def test_parts_join_by_their_lse(mb, torch):
    """A row's attention over the prefix alone and over the rest, joined, is the whole."""
    p, out, lse = check(mb, torch, [600], [1], 4, 2, 64, 8, "float16")
    ctx = mb.KvContext(max_requests=1)
    cache = mb.KvCache(p.k, p.v)
    first = torch.tensor([304], dtype=torch.int32, device="cuda")
    a, la = ctx.attention(p.q, cache, p.d_tables, first, p.cu, max_new=1, return_lse=True)
    b, lb = ctx.attention(p.q, cache, p.d_tables[:, 38:].contiguous(), p.d_lens - 304, p.cu, max_new=1, return_lse=True)
    both = torch.logaddexp(la, lb)
    joined = a.float() * torch.exp(la - both)[..., None] + b.float() * torch.exp(lb - both)[..., None]
    p.check(joined, both)


def test_no_tokens(mb, torch):
    p = Problem(torch, [5, 9], [1, 1], 4, 2, 64, 16, "bfloat16")
    ctx = mb.KvContext(max_requests=2)
    out, lse = ctx.attention(p.q[:0], mb.KvCache(p.k, p.v), p.d_tables, p.d_lens, p.cu * 0, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_refusals(mb, torch):
    p = Problem(torch, [5, 9], [1, 1], 4, 2, 64, 16, "bfloat16")
    ctx = mb.KvContext(max_requests=2)
    bf = dict(device="cuda", dtype=torch.bfloat16)

    def call(q=p.q, cache=None, tables=p.d_tables, lens=p.d_lens, cu=p.cu, **kw):
        return ctx.attention(q, cache or mb.KvCache(p.k, p.v), tables, lens, cu, **kw)
    call()
    for status, kw in [
            (mb.MARS_ERR_INVALID, dict(q=torch.zeros(2, 3, 64, **bf))),                          # heads
            (mb.MARS_ERR_INVALID, dict(window=-1)), (mb.MARS_ERR_INVALID, dict(softcap=-2.0)),
            (mb.MARS_ERR_INVALID, dict(softcap=math.nan)), (mb.MARS_ERR_INVALID, dict(scale=math.inf)),
            (mb.MARS_ERR_INVALID, dict(q=torch.zeros(2, 4, 72, **bf)[..., 4:68])),               # starts at 8 bytes
            (mb.MARS_ERR_INVALID, dict(q=torch.zeros(2, 4, 68, **bf)[..., :64])),                # strides of 136 bytes
            (mb.MARS_ERR_UNSUPPORTED, dict(q=torch.zeros(2, 258, 64, **bf))),                    # 129 a key head
            (mb.MARS_ERR_UNSUPPORTED, dict(q=torch.zeros(2, 4, 60, **bf), cache=mb.KvCache(*(torch.zeros(4, 16, 2, 60, **bf),) * 2))),
            (mb.MARS_ERR_UNSUPPORTED, dict(q=torch.zeros(2, 4, 136, **bf), cache=mb.KvCache(*(torch.zeros(4, 16, 2, 136, **bf),) * 2))),
            (mb.MARS_ERR_UNSUPPORTED, dict(cache=mb.KvCache(*(torch.zeros(4, 12, 2, 64, **bf),) * 2))),
            (mb.MARS_ERR_CAPACITY, dict(lens=torch.zeros(3, dtype=torch.int32, device="cuda"),
                                        cu=torch.zeros(4, dtype=torch.int32, device="cuda"),
                                        tables=torch.zeros(3, 2, dtype=torch.int32, device="cuda")))]:
        with pytest.raises(mb.MarsError) as e:
            call(**kw)
        assert e.value.status == status, f"{kw}: {e.value}"
    for kw in (dict(q=p.q.half()), dict(q=p.q.cpu()), dict(q=p.q[..., :32]), dict(lens=p.d_lens.long()),
               dict(cu=p.cu[:2]), dict(tables=p.d_tables[:1]), dict(decay=torch.zeros(3, device="cuda")),
               dict(prefix_lens=torch.zeros(1, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            call(**kw)
    out, lse = call(return_lse=True)
    p.check(out, lse)
