"""mars_rope / mars_rope_append against the rotation written out in 64 bits.

Tolerances: the result is one rounding of a value computed in fp32 with an
angle good to 2^-24 of a turn of pi (the reduced argument's rounding, at most
pi * 2^-24, and sincospi's 2 units in the last place): for a pair of norm r
at most 6 * 2^-24 * r in fp32 (angle 3.2, two products and a sum 1.5, spare),
plus half a unit of the output type, 2^-11 (fp16) or 2^-8 (bf16) of the value
at most; fp16 also 2^-25 below its normal range."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_UNIT = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def mb():
    import mars_b200
    return mars_b200


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def plain(x, positions, freq, axis, interleaved, inverse=False):
    """x [tokens, heads, d] float64 numpy."""
    half = len(freq)
    theta = positions[:, axis].astype(np.float64) * freq.astype(np.float64)
    c, s = np.cos(theta)[:, None], np.sin(theta)[:, None] * (-1 if inverse else 1)
    y = x.copy()
    i = np.arange(half)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ia] * s + x[..., ib] * c
    norm = np.zeros_like(x)
    norm[..., ia] = norm[..., ib] = np.hypot(x[..., ia], x[..., ib])
    return y, norm


def close(got, want, norm, dtype):
    limit = 6 * 2.0 ** -24 * norm + HALF_UNIT[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "float16" else 0)
    err = np.abs(got - want)
    assert (err <= limit).all(), f"largest excess {(err - limit).max()} at {np.argmax(err - limit)}"


def table(torch, rot, axes, seed):
    half = rot // 2
    rng = np.random.default_rng(seed)
    freq = (10000.0 ** (-np.arange(half) / max(half, 1))).astype(np.float32)
    axis = rng.integers(0, axes, half).astype(np.int32)
    return freq, axis, torch.from_numpy(freq).cuda(), torch.from_numpy(axis).cuda()


SHAPES = [  # tokens, heads, d, rot, axes
    (1, 1, 2, 2, 1), (1, 12, 64, 64, 1), (7, 3, 128, 128, 3), (33, 5, 80, 40, 2), (1300, 4, 64, 48, 3), (5, 2, 7, 4, 2),
    (64, 2, 24, 24, 1), (9, 3, 72, 12, 2), (3, 2, 16, 0, 1), (2, 1, 1024, 1024, 2), (2500, 1, 36, 20, 1), (4, 2, 130, 128, 1)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotation_and_its_inverse(mb, torch, shape, interleaved, dtype):
    n, h, d, rot, axes = shape
    rng = np.random.default_rng(n * d)
    freq, axis, dfreq, daxis = table(torch, rot, axes, d)
    pos = rng.integers(0, 200000, (n, axes)).astype(np.int32)
    pos[0] = 0
    x = torch.from_numpy(rng.standard_normal((n, h, d)).astype(np.float32)).cuda().to(getattr(torch, dtype))
    x64 = x.double().cpu().numpy()
    for inverse in (False, True):
        y = mb.rope(x, torch.from_numpy(pos).cuda(), dfreq, daxis, interleaved=interleaved, inverse=inverse)
        want, norm = plain(x64, pos, freq, axis, interleaved, inverse)
        close(y.double().cpu().numpy(), want, norm, dtype)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(mb, torch, interleaved):
    """d/dx of <w, rope(x)> by central differences; the rotation is linear, so a step of 1 has no truncation
    error: what is left is 8 fp32 values' rounding (each 2^-24 of at most 4.5 sigma) times the 14 terms a row adds."""
    n, h, d, rot, axes = 3, 2, 14, 10, 2
    rng = np.random.default_rng(0)
    _, _, dfreq, daxis = table(torch, rot, axes, 1)
    pos = torch.from_numpy(rng.integers(0, 5000, (n, axes)).astype(np.int32)).cuda()
    x, w = (torch.from_numpy(rng.standard_normal((n, h, d)).astype(np.float32)).cuda() for _ in range(2))
    grad = mb.rope(w, pos, dfreq, daxis, interleaved=interleaved, inverse=True).double()
    for k in range(n * h * d):
        e = torch.zeros(n * h * d, device="cuda")
        e[k] = 1.0
        e = e.view(n, h, d)
        up, down = (mb.rope(x + s * e, pos, dfreq, daxis, interleaved=interleaved).double() for s in (1.0, -1.0))
        diff = ((up - down) * w.double()).sum() / 2
        assert abs(diff.item() - grad.flatten()[k].item()) <= 14 * 8 * 4.5 * 4.5 * 2.0 ** -24


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,hq,hkv,d,rot,page,layout", [
    (1, 4, 1, 64, 64, 16, "tokens"), (50, 12, 12, 64, 64, 16, "heads"), (700, 6, 2, 128, 64, 48, "tokens"),
    (33, 3, 3, 80, 80, 7, "both"), (5, 2, 1, 18, 6, 3, "tokens"), (17, 5, 5, 40, 24, 8, "odd")])
def test_append_writes_its_slots_and_nothing_else(mb, torch, n, hq, hkv, d, rot, page, layout, interleaved, dtype):
    rng = np.random.default_rng(n + d)
    gen = torch.Generator(device="cuda").manual_seed(n)
    dt = getattr(torch, dtype)
    freq, axis, dfreq, daxis = table(torch, rot, 3, d)
    pos = rng.integers(0, 40000, (n, 3)).astype(np.int32)
    pages = -(-n // page) + 4
    if layout == "heads":              # [pages, heads, page, d] in memory
        k, v = (torch.randn(pages, hkv, page, d, generator=gen, device="cuda").to(dt).transpose(1, 2) for _ in range(2))
    elif layout == "both":             # keys and values of a page side by side
        both = torch.randn(pages, 2, page, hkv, d, generator=gen, device="cuda").to(dt)
        k, v = both[:, 0], both[:, 1]
    elif layout == "odd":              # starts and strides that no 16-byte load can use
        k, v = (torch.randn(pages, page, hkv, d + 3, generator=gen, device="cuda").to(dt)[..., 1:d + 1] for _ in range(2))
    else:
        k, v = (torch.randn(pages, page, hkv, d, generator=gen, device="cuda").to(dt) for _ in range(2))
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=gen, device="cuda").to(dt)
    q3, k3, v3 = (t.unflatten(1, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], dim=1))
    slots = rng.permutation(pages * page)[:n].astype(np.int32)
    skipped = rng.random(n) < 0.2
    slots[skipped] = rng.choice([-1, pages * page, 2 ** 31 - 1, -2 ** 31], skipped.sum())
    want_k, want_v = k.double().cpu().numpy(), v.double().cpu().numpy()
    norm_k = np.zeros_like(want_k)
    yk, nk = plain(k3.double().cpu().numpy(), pos, freq, axis, interleaved)
    at = slots[~skipped]
    want_k[at // page, at % page], norm_k[at // page, at % page] = yk[~skipped], nk[~skipped]
    want_v[at // page, at % page] = v3.double().cpu().numpy()[~skipped]
    out = mb.rope_append(q3, k3, v3, torch.from_numpy(pos).cuda(), dfreq, daxis, mb.KvCache(k, v),
                         torch.from_numpy(slots).cuda(), interleaved=interleaved)
    want_q, norm_q = plain(q3.double().cpu().numpy(), pos, freq, axis, interleaved)
    close(out.double().cpu().numpy(), want_q, norm_q, dtype)
    got_k = k.double().cpu().numpy()
    touched = np.zeros(got_k.shape[:2], bool)
    touched[at // page, at % page] = True
    close(got_k[touched], want_k[touched], norm_k[touched], dtype)
    assert np.array_equal(got_k[~touched], want_k[~touched])
    assert np.array_equal(v.double().cpu().numpy(), want_v)
    # in place gives the same
    mb.rope_append(q3, k3, v3, torch.from_numpy(pos).cuda(), dfreq, daxis, mb.KvCache(k, v),
                   torch.from_numpy(slots).cuda(), interleaved=interleaved, out=q3)
    assert torch.equal(q3, out)


def test_padded_columns_stay(mb, torch):
    """Head 'odd' above: the columns beside the view are not the view's."""
    base = torch.full((2, 4, 1, 24), 7.0, device="cuda", dtype=torch.float16)
    k, v = base[..., 1:9], torch.zeros(2, 4, 1, 8, device="cuda", dtype=torch.float16)
    x = torch.ones(3, 1, 8, device="cuda", dtype=torch.float16)
    z = torch.zeros(4, dtype=torch.int32, device="cuda")
    mb.rope_append(x, x, x, z[:3], torch.ones(4, device="cuda"), z, mb.KvCache(k, v),
                   torch.tensor([0, 5, 7], dtype=torch.int32, device="cuda"))
    assert (base[..., 0] == 7).all() and (base[..., 9:] == 7).all()
    assert (k.reshape(8, 8)[[0, 5, 7]] == 1).all() and (k.reshape(8, 8)[[1, 2, 3, 4, 6]] == 7).all()


def test_strided_tokens_long_positions_and_streams(mb, torch):
    freq, axis, dfreq, daxis = table(torch, 16, 1, 0)
    base = torch.randn(40, 3, 64, device="cuda")
    x = base[::2, :, 8:40]
    pos = np.array([2 ** 31 - 1 - i for i in range(20)], np.int32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = mb.rope(x, torch.from_numpy(pos).cuda(), dfreq, daxis)
    s.synchronize()
    want, norm = plain(x.double().cpu().numpy(), pos[:, None], freq, axis, False)
    close(y.double().cpu().numpy(), want, norm, "float32")


def test_no_tokens(mb, torch):
    z = torch.zeros(0, 2, 8, device="cuda", dtype=torch.float16)
    pos = torch.zeros(0, dtype=torch.int32, device="cuda")
    f, a = torch.ones(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    assert mb.rope(z, pos, f, a).shape == (0, 2, 8)
    c = mb.KvCache(*(torch.zeros(1, 4, 2, 8, device="cuda", dtype=torch.float16) for _ in range(2)))
    assert mb.rope_append(z, z, z, pos, f, a, c, pos).shape == (0, 2, 8)


def test_refusals(mb, torch):
    f16 = dict(device="cuda", dtype=torch.float16)
    x, pos = torch.zeros(3, 2, 8, **f16), torch.zeros(3, dtype=torch.int32, device="cuda")
    f, a = torch.ones(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    cache = mb.KvCache(torch.zeros(1, 4, 2, 8, **f16), torch.zeros(1, 4, 2, 8, **f16))
    mb.rope(x, pos, f, a)
    with pytest.raises(mb.MarsError) as e:                      # rot_dim 8 > head_dim 6
        mb.rope(x[..., :6], pos, f, a)
    assert e.value.status == mb.MARS_ERR_INVALID
    with pytest.raises(mb.MarsError) as e:
        mb.rope(torch.zeros(3, 1, 1026, **f16), pos, torch.ones(513, device="cuda"),
                torch.zeros(513, dtype=torch.int32, device="cuda"))
    assert e.value.status == mb.MARS_ERR_UNSUPPORTED
    for bad in (dict(x=x.double()), dict(x=x.cpu()), dict(x=x.transpose(1, 2)), dict(positions=pos.long()),
                dict(positions=pos[:2]), dict(freq=f.half()), dict(axis=a[:3])):
        with pytest.raises(ValueError):
            mb.rope(**dict(dict(x=x, positions=pos, freq=f, axis=a), **bad))
    ok = dict(q=x, k=x, v=x, positions=pos, freq=f, axis=a, cache=cache, slots=pos)
    mb.rope_append(**ok)
    for bad in (dict(k=x[:, :1]), dict(v=x[:2]), dict(q=x.float()), dict(slots=pos[:1])):
        with pytest.raises(ValueError):
            mb.rope_append(**dict(ok, **bad))
    with pytest.raises(ValueError):
        mb.KvCache(torch.zeros(1, 4, 2, 8, device="cuda"), torch.zeros(1, 4, 2, 8, device="cuda"))
    with pytest.raises(ValueError):
        mb.KvCache(cache.k, cache.v[:, :2])
