"""The answering step's operators on a paged key/value cache, as measured cases.

An agent that answers with retrieved memories keeps the keys and values of its
requests in pages.  Three operators run there:

* plan:   block tables, slots and positions from the requests' lengths, with
          pages given back by finished requests (kv_release, kv_plan);
* rope:   rotary positions with several axes on queries and keys, which also
          writes keys and values into their pages (rope_append), and the
          rotation alone in both directions (rope: its inverse is its gradient);
* attend: attention of each request's new tokens over its pages, with capped
          scores, a decay with the distance, a prefix that every row sees and a
          window over the rest (paged_attention).

Lengths follow from the case alone (so work() knows them); which request has
which, the pages and all values come from the seed.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def _mars():
    path = os.path.abspath("cuda-multimodal-memory_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mars_b200
    return mars_b200


# ---- cases -----------------------------------------------------------------

def _plan(name, **kw):
    return dict(dict(name=name, op="plan", requests=64, cached=4096, new=1, page=16, release=0), **kw)


def _append(name, **kw):
    return dict(dict(name=name, op="append", tokens=32, hq=12, hkv=12, d=64, rot=64, axes=1, interleaved=False,
                     page=16, longest=4096, dtype="f16"), **kw)


def _rope(name, **kw):
    return dict(dict(name=name, op="rope", tokens=1024, hq=12, d=64, rot=64, axes=2, interleaved=False,
                     inverse=False, longest=4096, dtype="f32"), **kw)


def _attend(name, **kw):
    return dict(dict(name=name, op="attend", requests=4, cached=700, new=1, hq=12, hkv=12, d=64, page=16,
                     cap=0.0, decay=False, prefix=0, window=0, dtype="f16"), **kw)


def listed():
    return [
        # one decode step of 64 running requests: the call before every generated token
        _plan("plan_decode_64"),
        # a busy server's step: 1,023 slots, a quarter finished and refilled, chunks of up to 128 tokens
        _plan("plan_mixed_1023", requests=1023, cached=8000, new=128, page=32, release=4),
        # a bulk load of prompts, 300 K new tokens
        _plan("plan_prompts_300", requests=300, cached=0, new=2000, page=64),
        # the decode step of a small encoder-sized head layout (12 heads of 64: the 768 columns of the stored rows)
        _append("append_step_32"),
        # a prefill chunk with three axes (time, height, width), grouped heads
        _append("append_chunk_8192", tokens=8192, hq=32, hkv=8, d=128, rot=128, axes=3, page=64, longest=32768,
                dtype="bf16"),
        # training: the gradient of a rotation in fp32, interleaved pairs, part of the head rotated, odd count
        _rope("rope_grad_16381", tokens=16381, hq=12, d=64, rot=48, axes=3, interleaved=True, inverse=True,
              longest=16384),
        # the smallest decode step: four short requests
        _attend("decode_4_short"),
        # a decode step of 64 ragged requests, grouped heads
        _attend("decode_64_ragged", requests=64, cached=8000, hq=32, hkv=8, d=128, page=32, dtype="bf16"),
        # two very long caches: the split over the long axis carries it
        _attend("decode_2_long", requests=2, cached=250000, hq=16, hkv=4, d=128, page=128, dtype="bf16"),
        # prefill chunks over a cache, capped scores and a decay with the distance
        _attend("chunk_8_capped", requests=8, cached=4000, new=512, hq=16, hkv=4, d=128, page=64, cap=30.0,
                decay=True, dtype="bf16"),
        # whole prompts whose first 1,000 tokens (the memories) everyone sees
        _attend("prompt_2_prefix", requests=2, cached=0, new=8192, hq=32, hkv=8, d=128, page=64, prefix=1000,
                dtype="bf16"),
        # odd everything: 3 queries a key head, 80 columns, pages of 48, a window behind a short prefix
        _attend("chunk_5_window", requests=5, cached=3001, new=217, hq=15, hkv=5, d=80, page=48, prefix=70,
                window=1500),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


_MOST_FLOPS = 7e11        # the largest listed case's
_MOST_SCORES = 4.2e9      # rows x columns of the plain form's padded scores


def draw(rng):
    op = rng.choice(["plan", "append", "rope", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "plan":
        requests = _log(rng, 1, 2000)
        return {k: v for k, v in _plan("", requests=requests, cached=rng.choice([0, _log(rng, 1, 8000)]),
                                       new=_log(rng, 1, max(1, min(4000, 600000 // requests))),
                                       page=rng.choice([8, 16, 32, 48, 64, 128]),
                                       release=rng.choice([0, 0, 2, 5])).items() if k != "name"}
    d = rng.choice([64, 128, 128, 8 * rng.randint(3, 16)])
    hkv = rng.choice([1, 2, 3, 4, 5, 8, 12])
    hq = hkv * rng.choice([1, 1, 2, 3, 4, 8] if hkv < 8 else [1, 2, 4])
    if op in ("append", "rope"):
        axes = rng.randint(1, 3)
        rot = rng.choice([d, d, max(2 * axes, d // 4 * 2)])
        most = 32 << 20
        tokens = _log(rng, 1, max(1, most // ((hq + 2 * hkv) * d)))
        if op == "append":
            case = _append("", tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, axes=axes,
                           interleaved=rng.random() < 0.4, page=rng.choice([8, 16, 32, 48, 64, 128]),
                           longest=_log(rng, 64, 32768), dtype=dtype)
        else:
            case = _rope("", tokens=tokens, hq=hq, d=d, rot=rot, axes=axes, interleaved=rng.random() < 0.4,
                         inverse=rng.random() < 0.6, longest=_log(rng, 64, 32768),
                         dtype=rng.choice(["f32", dtype]))
        return {k: v for k, v in case.items() if k != "name"}
    while True:
        new = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 8192)])
        requests = _log(rng, 1, 96 if new < 10 else 12)
        cached = rng.choice([0, 1, 1]) * _log(rng, 16, 250000 if new < 10 else 30000)
        case = _attend("", requests=requests, cached=cached, new=new, hq=hq, hkv=hkv, d=d,
                       page=rng.choice([8, 16, 32, 48, 64, 128]), cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                       decay=rng.random() < 0.3, prefix=rng.choice([0, 0, _log(rng, 8, 2000)]),
                       window=rng.choice([0, 0, 0, _log(rng, 16, 4000)]), dtype=dtype)
        most = cached + new
        if requests * hq * new * most > _MOST_SCORES or requests * hkv * most * d * 2 > 1 << 29:
            continue
        if work(case)["flops"] > _MOST_FLOPS:
            continue
        return {k: v for k, v in case.items() if k != "name"}


def _spread(n, most, least):
    """n lengths between least and most, the first of them `most`: the same for every seed."""
    at = (np.arange(n) * 0.6180339887) % 1.0
    return np.maximum(least, np.round(most * (1.0 - 0.8 * at))).astype(np.int64)


def _lengths(case):
    """(cached before, new) tokens of each request."""
    n = case["requests"]
    cached = _spread(n, case["cached"], 0)
    return cached, np.roll(_spread(n, case["new"], 1), n // 3)


# ---- inputs ----------------------------------------------------------------

def _tables(case, total, rng):
    """Pages in no order for requests of `total` tokens: (tables, pages in all)."""
    page = case["page"]
    need = -(-total // page)
    spare = 3
    order = rng.permutation(int(need.sum()) + spare)
    tables = np.full((len(total), max(1, int(need.max()))), -1, np.int64)
    first = np.cumsum(need) - need
    for b in range(len(total)):
        tables[b, :need[b]] = order[first[b]:first[b] + need[b]]
    return tables, len(order)


def _freq(case):
    """Frequencies of the pairs, and the axis each pair turns with (axes in bands)."""
    half = case["rot"] // 2
    freq = (10000.0 ** (-np.arange(half) / half)).astype(np.float32)
    axis = np.minimum(np.arange(half) * case["axes"] // half, case["axes"] - 1).astype(np.int32)
    return torch.from_numpy(freq).cuda(), torch.from_numpy(axis).cuda()


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def normal(*shape, dtype=None):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype or _DTYPES[case["dtype"]])

    s = {"case": case}
    if op == "plan":
        cached, new = _lengths(case)
        page = case["page"]
        gone = np.zeros(len(cached), np.int64)
        if case["release"]:
            gone[::case["release"]] = 1
        order = rng.permutation(len(cached))
        cached, new, gone = cached[order], new[order], gone[order]
        after = np.where(gone, 0, cached) + new
        held = -(-cached // page)
        width = int(max(1, (-(-np.maximum(after, cached) // page)).max()))
        need = int((-(-after // page) - np.where(gone, 0, held)).sum())
        pages = rng.permutation(int(held.sum()) + need + 7)
        tables = np.full((len(cached), width), -1, np.int64)
        first = np.cumsum(held) - held
        for b in range(len(cached)):
            tables[b, :held[b]] = pages[first[b]:first[b] + held[b]]
        free = np.full(len(pages), -1, np.int64)
        free[:need + 7] = pages[int(held.sum()):]
        s.update(lens=_i32(cached), new=_i32(new), gone=_i32(gone), tables=_i32(tables), free=_i32(free),
                 count=_i32([need + 7]), tokens=int(new.sum()))
        return s
    if op in ("append", "rope"):
        n = case["tokens"]
        s["freq"], s["axis"] = _freq(case)
        s["positions"] = _i32(rng.integers(0, case["longest"], (n, case["axes"])))
        if op == "rope":
            s["x"] = normal(n, case["hq"], case["d"])
            return s
        # the three parts of one projection's output, as a program has them
        qkv = normal(n, (case["hq"] + 2 * case["hkv"]) * case["d"])
        q, k, v = qkv.split([case["hq"] * case["d"], case["hkv"] * case["d"], case["hkv"] * case["d"]], dim=1)
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, case["d"])) for x in (q, k, v))
        pages = -(-n // case["page"]) + 5
        s["keys"], s["values"] = (normal(pages, case["page"], case["hkv"], case["d"]) for _ in range(2))
        slots = rng.permutation(pages * case["page"])[:n]
        s["slots"] = _i32(slots)
        return s
    cached, new = _lengths(case)
    order = rng.permutation(len(cached))
    cached, new = cached[order], new[order]
    total = cached + new
    tables, pages = _tables(case, total, rng)
    s["tables"] = _i32(tables)
    s["lens"] = _i32(total)
    s["first"] = _i32(np.concatenate([[0], np.cumsum(new)]))
    s["most_new"], s["most_len"] = int(new.max()), int(total.max())
    s["q"] = normal(int(new.sum()), case["hq"], case["d"])
    s["keys"] = normal(pages, case["page"], case["hkv"], case["d"])
    s["values"] = normal(pages, case["page"], case["hkv"], case["d"])
    s["decay"] = None
    if case["decay"]:
        s["decay"] = torch.from_numpy(2.0 ** (-8.0 * np.arange(1, case["hq"] + 1) / case["hq"]))
        s["decay"] = s["decay"].to(device="cuda", dtype=torch.float32)
    s["prefix"] = None
    if case["prefix"]:
        s["prefix"] = _i32(np.minimum(total, np.maximum(1, case["prefix"] - 13 * np.arange(len(total)))))
    return s


# ---- the operators ---------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "rope": _own_rope, "attend": _own_attend}[op](s)
    return {"plan": _plain_plan, "append": _plain_append, "rope": _plain_rope, "attend": _plain_attend}[op](s)


def _own_plan(s):
    mars = _mars()
    case = s["case"]
    ctx = s.get("ctx") or s.setdefault("ctx", mars.KvContext(max_requests=case["requests"]))
    lens, free, count = s["lens"], s["free"], s["count"]
    if case["release"]:
        lens, count = ctx.release(lens, s["gone"], s["tables"], free, count, page_size=case["page"])
    p = ctx.plan(lens, s["new"], s["tables"], free, count, page_size=case["page"], max_tokens=s["tokens"])
    return {"lens": p.kv_lens, "tables": s["tables"], "free": free, "count": p.free_count, "first": p.cu_new,
            "slots": p.slots, "positions": p.positions, "status": p.status}


def _plain_plan(s):
    case = s["case"]
    page, lens, free, count, tables = case["page"], s["lens"].long(), s["free"], s["count"].long(), s["tables"]
    column = torch.arange(tables.shape[1], device="cuda")
    if case["release"]:
        back = (s["gone"] != 0)[:, None] & (column < ((lens + page - 1) // page)[:, None])
        pushed = tables[back]
        free[count + torch.arange(len(pushed), device="cuda")] = pushed
        count = count + len(pushed)
        lens = torch.where(s["gone"] != 0, 0, lens)
    after = lens + s["new"]
    held, want = (lens + page - 1) // page, (after + page - 1) // page
    fresh = (column >= held[:, None]) & (column < want[:, None])
    number = torch.cumsum(fresh.flatten(), 0) - 1
    tables[fresh] = free[(count - 1 - number)[fresh.flatten()]]
    first = torch.cat([torch.zeros_like(count), torch.cumsum(s["new"].long(), 0)])
    which = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), s["new"].long(), output_size=s["tokens"])
    position = lens[which] + torch.arange(s["tokens"], device="cuda") - first[which]
    slots = tables[which, position // page].long() * page + position % page
    i32 = torch.int32
    return {"lens": after.to(i32), "tables": tables, "free": free, "count": (count - fresh.sum()).to(i32),
            "first": first.to(i32), "slots": slots.to(i32), "positions": position.to(i32),
            "status": torch.zeros(1, dtype=i32, device="cuda")}


def _own_append(s):
    mars = _mars()
    cache = mars.KvCache(s["keys"], s["values"])
    q = mars.rope_append(s["q"], s["k"], s["v"], s["positions"], s["freq"], s["axis"], cache, s["slots"],
                         interleaved=s["case"]["interleaved"])
    return {"q": q, "keys": s["keys"], "values": s["values"]}


def _own_rope(s):
    case = s["case"]
    return {"y": _mars().rope(s["x"], s["positions"], s["freq"], s["axis"], interleaved=case["interleaved"],
                              inverse=case["inverse"])}


def _turn(x, positions, freq, axis, interleaved, inverse):
    """x [tokens, heads, d] in 32 bits, the first columns' pairs turned by position * frequency.

    The product of a position below 2^15 and a frequency's leading 9 bits is exact in 32 bits; what the
    other bits add to the angle is small, and the two are joined by the addition theorem."""
    lead = (freq.view(torch.int32) & -32768).view(torch.float32)
    p = positions[:, axis.long()].float()
    big, small = p * lead, p * (freq - lead)
    cos = (torch.cos(big) * torch.cos(small) - torch.sin(big) * torch.sin(small))[:, None, :]
    sin = (torch.sin(big) * torch.cos(small) + torch.cos(big) * torch.sin(small))[:, None, :]
    if inverse:
        sin = -sin
    x = x.float()
    rot = 2 * len(freq)
    turned, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _plain_append(s):
    how = (s["positions"], s["freq"], s["axis"], s["case"]["interleaved"], False)
    slots = s["slots"].long()
    s["keys"].flatten(0, 1)[slots] = _turn(s["k"], *how).to(s["keys"].dtype)
    s["values"].flatten(0, 1)[slots] = s["v"]
    return {"q": _turn(s["q"], *how).to(s["q"].dtype), "keys": s["keys"], "values": s["values"]}


def _plain_rope(s):
    case = s["case"]
    y = _turn(s["x"], s["positions"], s["freq"], s["axis"], case["interleaved"], case["inverse"])
    return {"y": y.to(s["x"].dtype)}


def _own_attend(s):
    mars = _mars()
    case = s["case"]
    ctx = s.get("ctx") or s.setdefault("ctx", mars.KvContext(max_requests=case["requests"]))
    cache = mars.KvCache(s["keys"], s["values"])
    out, lse = ctx.attention(s["q"], cache, s["tables"], s["lens"], s["first"], max_new=s["most_new"],
                             softcap=case["cap"], window=case["window"], decay=s["decay"],
                             prefix_lens=s["prefix"], return_lse=True)
    return {"out": out, "lse": lse}


def _plain_attend(s):
    """All requests at once, padded to the longest: products, sums and exponentials in 32 bits."""
    case = s["case"]
    n, hq, hkv, d = case["requests"], case["hq"], case["hkv"], case["d"]
    group, rows, columns = hq // hkv, s["most_new"], s["most_len"]
    lens, first = s["lens"].long(), s["first"].long()
    new = first[1:] - first[:-1]
    j = torch.arange(columns, device="cuda")
    tables = s["tables"].long().clamp(min=0)
    slot = tables[:, j // case["page"]] * case["page"] + j % case["page"]
    keys = s["keys"].flatten(0, 1)[slot].float().permute(0, 2, 3, 1)                   # n, hkv, d, columns
    row = torch.arange(rows, device="cuda")
    token = (first[:-1, None] + row).clamp(max=len(s["q"]) - 1)
    q = s["q"][token].float().unflatten(2, (hkv, group)).permute(0, 2, 3, 1, 4)        # n, hkv, group, rows, d
    score = torch.matmul(q.flatten(2, 3) * d ** -0.5, keys).unflatten(2, (group, rows))
    del keys
    if case["cap"]:
        score.div_(case["cap"]).tanh_().mul_(case["cap"])
    position = (lens - new)[:, None] + row                                             # n, rows
    age = position[:, :, None] - j
    if case["decay"]:
        score.sub_(s["decay"].view(1, hkv, group, 1, 1) * age.clamp(min=0)[:, None, None].float())
    seen = age >= 0
    if case["window"]:
        seen &= age < case["window"]
    if s["prefix"] is not None:
        seen |= (j < s["prefix"][:, None])[:, None, :]
    seen &= (j < lens[:, None])[:, None, :]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    values = s["values"].flatten(0, 1)[slot].float().transpose(1, 2)                   # n, hkv, columns, d
    out = torch.matmul(score.flatten(2, 3), values).unflatten(2, (group, rows))
    out = out / torch.where(total > 0, total, 1.0)
    lse = torch.log(total) + top
    which = torch.repeat_interleave(torch.arange(n, device="cuda"), new, output_size=len(s["q"]))
    at = torch.arange(len(s["q"]), device="cuda") - first[which]
    out = out.permute(0, 3, 1, 2, 4)[which, at].flatten(1, 2)
    return {"out": out.to(s["q"].dtype), "lse": lse[..., 0].permute(0, 3, 1, 2)[which, at].flatten(1, 2)}


# ---- what a pass cannot do without -----------------------------------------

def work(case):
    op = case["op"]
    if op == "plan":
        cached, new = _lengths(case)
        page, n = case["page"], len(new)
        start = cached.copy()
        if case["release"]:
            start[::case["release"]] = 0
        fresh = int((-(-(start + new) // page) - -(-start // page)).sum())
        size = 4 * (2 * n + 1) + 4 * (2 * n + 2) + 2 * 4 * fresh + 2 * 4 * int(new.sum())
        if case["release"]:
            size += 4 * 2 * n + 2 * 4 * int((-(-cached[::case["release"]] // page)).sum())
        return {"bytes": size, "flops": int(new.sum())}
    if op in ("append", "rope"):
        heads = case["hq"] + (2 * case["hkv"] if op == "append" else 0)
        turned = case["hq"] + (case["hkv"] if op == "append" else 0)
        size = 2 * case["tokens"] * heads * case["d"] * _SIZE[case["dtype"]]
        size += case["tokens"] * 4 * (case["axes"] + (op == "append")) + 4 * case["rot"]
        return {"bytes": size, "flops": 3 * case["tokens"] * turned * case["rot"]}
    cached, new = _lengths(case)
    size = pairs = 0
    for b in range(case["requests"]):
        length = int(cached[b] + new[b])
        prefix = min(length, max(1, case["prefix"] - 13 * b)) if case["prefix"] else 0
        window = case["window"] or length
        i = np.arange(cached[b], length)
        low, high = np.maximum(prefix, i + 1 - window), np.maximum(prefix, i + 1)
        pairs += int((high - np.minimum(low, high) + prefix).sum())
        size += prefix + max(0, length - max(prefix, int(cached[b]) + 1 - window))
    tokens = int(new.sum())
    size = 2 * size * case["hkv"] * case["d"] * 2 + 2 * tokens * case["hq"] * case["d"] * 2 + tokens * case["hq"] * 4
    return {"bytes": size + 4 * int((-(-(cached + new) // case["page"])).sum()), "flops": 4 * case["d"] * case["hq"] * pairs}


# ---- the definitions in 64 bits --------------------------------------------

def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None                       # whole numbers only
    s = prepare(case, seed)
    if op in ("append", "rope"):
        half = case["rot"] // 2
        theta = s["positions"].double()[:, s["axis"].long()] * s["freq"].double()
        unit = torch.polar(torch.ones_like(theta), -theta if case.get("inverse") else theta)[:, None, :]

        def turned(x):
            y = x.double().clone()
            at = (slice(0, case["rot"], 2), slice(1, case["rot"], 2)) if case["interleaved"] else \
                (slice(0, half), slice(half, case["rot"]))
            z = torch.complex(y[..., at[0]].clone(), y[..., at[1]].clone()) * unit
            y[..., at[0]], y[..., at[1]] = z.real, z.imag
            return y
        if op == "rope":
            return {"y": turned(s["x"])}
        keys, values = s["keys"].double(), s["values"].double()
        place = s["slots"].long()
        keys[place // case["page"], place % case["page"]] = turned(s["k"])
        values[place // case["page"], place % case["page"]] = s["v"].double()
        return {"q": turned(s["q"]), "keys": keys, "values": values}
    group, page = case["hq"] // case["hkv"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    lens, first = s["lens"].tolist(), s["first"].tolist()
    for b, length in enumerate(lens):
        pages = s["tables"][b, :-(-length // page)].long()
        begin, end = first[b], first[b + 1]
        i = torch.arange(length - (end - begin), length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None, :]
        seen = (j <= i) & ((i - j < case["window"]) if case["window"] else True)
        if case["prefix"]:
            seen = seen | (j < int(s["prefix"][b]))
        for h in range(case["hkv"]):
            k = s["keys"][pages, :, h].double().reshape(-1, case["d"])[:length]
            v = s["values"][pages, :, h].double().reshape(-1, case["d"])[:length]
            for g in range(h * group, (h + 1) * group):
                z = s["q"][begin:end, g].double() @ k.T / math.sqrt(case["d"])
                if case["cap"]:
                    z = torch.tanh(z / case["cap"]) * case["cap"]
                if case["decay"]:
                    z = z - float(s["decay"][g]) * (i - j).clamp(min=0)
                z = torch.where(seen, z, -math.inf)
                lse[begin:end, g] = torch.logsumexp(z, 1)
                out[begin:end, g] = torch.softmax(z, 1) @ v
    return {"out": out, "lse": lse}
