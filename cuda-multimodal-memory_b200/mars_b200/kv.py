"""The operators of an answering step on a paged key/value cache.

A step of a program that answers with retrieved memories:

    lens, count = ctx.release(lens, finished, tables, free, count, page_size=64)
    plan = ctx.plan(lens, new_lens, tables, free, count, page_size=64, max_tokens=n)
    for each layer, with q, k, v its new tokens' projections:
        q = rope_append(q, k, v, positions, freq, axis, cache, plan.slots)
        out = ctx.attention(q, cache, tables, plan.kv_lens, plan.cu_new, max_new=1)

rope is the rotation by itself, for programs that train: autograd records it,
and its gradient is rope(..., inverse=True) of the output's gradient.  The calls
on a cache are for answering and record no gradient.

All arguments are torch CUDA tensors; calls run on torch's current stream
unless one is given (its handle, an integer), and return without waiting.  On a
given stream the caller orders the call after what makes its inputs, and keeps
them (record_stream) while it runs, as with torch's own operators; what the call
allocates itself belongs to that stream, and may be dropped at any time.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _STREAM_LEGACY, _check, lib

_raw_stream = torch._C._cuda_getCurrentRawStream      # torch.cuda.current_stream(...).cuda_stream without its objects
_current_device = torch._C._cuda_getDevice

KV_MAX_REQUESTS = 8192   # MARS_KV_MAX_REQUESTS
_INT32_MAX = 2 ** 31 - 1

# bits of KvPlan.status
KV_BAD_LENGTH = 1
KV_NO_PAGES = 2
KV_TABLE_FULL = 4
KV_TOO_MANY_TOKENS = 8
KV_STACK_FULL = 16


class KvPlan(NamedTuple):
    """What KvContext.plan returns (int32 CUDA tensors)."""
    kv_lens: torch.Tensor      # [B] tokens in the cache after the step
    cu_new: torch.Tensor       # [B + 1] new tokens before each request
    slots: torch.Tensor        # [max_tokens] place of each new token in the cache (-1: none)
    positions: torch.Tensor    # [max_tokens] its place in its request (-1: none)
    free_count: torch.Tensor   # [1] pages left on the free stack
    status: torch.Tensor       # [1] 0, or KV_* bits: then nothing was handed out


def _stream(stream, t):
    """The given stream, or torch's current one on t's device (as the other calls of this package do)."""
    if stream is not None:
        return stream
    return _raw_stream(t.get_device()) or _STREAM_LEGACY


def _empty(stream, t, shape, dtype):
    """An output of a call on the given stream (None: torch's current one on t's device).  The memory belongs to that
    stream, so that it goes to nobody else before the call has run; and the current stream, where the caller goes on, is
    recorded, so that a later call on the given one does not get it too early."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=t.device)
    handle = getattr(stream, "value", stream) or 0
    on = torch.cuda.default_stream(t.device) if handle in (0, _STREAM_LEGACY) else \
        torch.cuda.ExternalStream(handle, device=t.device)
    here = torch.cuda.current_stream(t.device)
    with torch.cuda.stream(on):
        made = torch.empty(shape, dtype=dtype, device=t.device)
    if here != on:
        made.record_stream(here)
    return made


def _on_device_of(t, call, args):
    """call(*args) with t's device as the current one, for entry points without a context."""
    if t.get_device() == _current_device():
        _check(call(*args))
    else:
        with torch.cuda.device(t.device):
            _check(call(*args))


def _ints(name, t, device, n=None, dims=1):
    """The address of a contiguous int32 tensor of n entries (n None: any) on the CUDA device of that number."""
    shape = t.shape
    if t.dtype is not torch.int32 or t.get_device() != device or len(shape) != dims or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {dims} dimension(s) on cuda:{device}")
    if n is not None and shape[0] != n:
        raise ValueError(f"{name} must have {n} entries, has {shape[0]}")
    return t.data_ptr()


def _floats(name, t, device, n=None):
    """The same of a float32 tensor of one dimension."""
    shape = t.shape
    if t.dtype is not torch.float32 or t.get_device() != device or len(shape) != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of 1 dimension on cuda:{device}")
    if n is not None and shape[0] != n:
        raise ValueError(f"{name} must have {n} entries, has {shape[0]}")
    return t.data_ptr()


_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # MARS_DTYPE_*


class _Cache(C.Structure):
    """mars_kv_cache."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("dtype", C.c_int32), ("num_pages", C.c_int32),
                ("page_size", C.c_int32), ("kv_heads", C.c_int32), ("head_dim", C.c_int32), ("reserved", C.c_int32),
                ("k_page_stride", C.c_int64), ("k_slot_stride", C.c_int64), ("k_head_stride", C.c_int64),
                ("v_page_stride", C.c_int64), ("v_slot_stride", C.c_int64), ("v_head_stride", C.c_int64)]


class _Table(C.Structure):
    """mars_rope_table."""
    _fields_ = [("freq", C.c_void_p), ("axis", C.c_void_p), ("rot_dim", C.c_int32), ("n_axes", C.c_int32),
                ("interleaved", C.c_int32), ("reserved", C.c_int32)]


class _Config(C.Structure):
    """mars_attn_config."""
    _fields_ = [("scale", C.c_float), ("softcap", C.c_float), ("window", C.c_int32), ("max_new", C.c_int32)]


class KvCache:
    """The caller's pages: k and v are [pages, page_size, kv_heads, head_dim] CUDA tensors (fp16 or bf16) of any
    strides with contiguous columns -- a permuted view where memory has the heads before the tokens."""

    def __init__(self, k, v):
        shape, dtype = k.shape, k.dtype
        if v.shape != shape or v.dtype is not dtype or len(shape) != 4 or not k.is_cuda or k.device != v.device:
            raise ValueError("k and v must be CUDA tensors [pages, page_size, kv_heads, head_dim] of one shape and type")
        if dtype is not torch.float16 and dtype is not torch.bfloat16:
            raise ValueError("the cache holds fp16 or bf16")
        ks, vs = k.stride(), v.stride()
        if ks[3] != 1 or vs[3] != 1:
            raise ValueError("the cache's columns must be contiguous")
        self.k, self.v = k, v
        self._c = _Cache(k.data_ptr(), v.data_ptr(), _DTYPES[dtype], *shape, 0, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])
        self._ref = C.byref(self._c)


def _heads(name, x, like=None):
    """Checks [tokens, heads, head_dim] with contiguous columns; its address and (token, head) strides."""
    shape, strides = x.shape, x.stride()
    if len(shape) != 3 or not x.is_cuda or (strides[2] != 1 and shape[2] != 1):
        raise ValueError(f"{name} must be a CUDA tensor [tokens, heads, head_dim] with contiguous columns")
    if like is not None and (shape[0] != like.shape[0] or x.dtype is not like.dtype or x.device != like.device):
        raise ValueError(f"{name} must have {like.shape[0]} tokens of {like.dtype}")
    return x.data_ptr(), strides[0], strides[1]


def _table(tokens, positions, freq, axis, interleaved, device):
    _ints("positions", positions, device, tokens, positions.dim())
    if positions.dim() not in (1, 2):
        raise ValueError("positions must be [tokens] or [tokens, axes]")
    pairs = freq.shape[0] if freq.dim() == 1 else None
    freq = _floats("freq", freq, device)
    axes = 1 if positions.dim() == 1 else positions.shape[1]
    return _Table(freq, _ints("axis", axis, device, pairs), 2 * pairs, axes, int(interleaved), 0)


def _out(out, x, stream):
    if out is None:
        return _empty(stream, x, x.shape, x.dtype)
    if out.shape != x.shape:
        raise ValueError("out must have the input's shape")
    return out


class _Rope(torch.autograd.Function):
    """rope on an x that requires a gradient: the rotation is orthogonal, so dx is dy turned the other way."""

    @staticmethod
    def forward(ctx, x, positions, freq, axis, interleaved, inverse, stream):
        ctx.save_for_backward(positions, freq, axis)
        ctx.how = interleaved, inverse
        return rope(x, positions, freq, axis, interleaved=interleaved, inverse=inverse, stream=stream)

    @staticmethod
    def backward(ctx, dy):
        interleaved, inverse = ctx.how
        if dy.stride(2) != 1:
            dy = dy.contiguous()                   # an expanded gradient (of a sum) has strides of 0
        return rope(dy, *ctx.saved_tensors, interleaved=interleaved, inverse=not inverse), None, None, None, None, None, None


def rope(x, positions, freq, axis, *, interleaved=False, inverse=False, out=None, stream=None):
    """Rotary positions of x [tokens, heads, head_dim] (fp32, fp16 or bf16): pair i turns by positions[:, axis[i]]
    * freq[i].  positions: int32 [tokens, axes].  inverse: turns back, the gradient of the forward rotation.  x has a
    gradient (its backward pass runs on autograd's stream, also where stream is given), freq has none."""
    if x.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("rope into out records no gradient: leave out away, or detach x")
        return _Rope.apply(x, positions, freq, axis, interleaved, inverse, stream)
    xp = _heads("x", x)
    dtype = _DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError("x must be fp32, fp16 or bf16")
    n, heads, dim = x.shape
    table = _table(n, positions, freq, axis, interleaved, x.get_device())
    out = _out(out, x, stream)
    _on_device_of(x, lib().mars_rope, (C.byref(table), dtype, *xp, *_heads("out", out, x), n, heads, dim,
                                       positions.data_ptr(), int(inverse), _stream(stream, x)))
    return out


def rope_append(q, k, v, positions, freq, axis, cache, slots, *, interleaved=False, out=None, stream=None):
    """q rotated (returned, or into out, which may be q), k rotated and v copied into the cache's slots.  No gradient.
    q: [tokens, q_heads, head_dim], k and v: [tokens, kv_heads, head_dim], all of the cache's type."""
    qp, kp, vp = _heads("q", q), _heads("k", k, q), _heads("v", v, q)
    n, heads, dim = q.shape
    c = cache._c
    if q.dtype is not cache.k.dtype or q.device != cache.k.device or dim != c.head_dim or \
            k.shape[1:] != (c.kv_heads, dim) or v.shape != k.shape:
        raise ValueError("q, k and v must have the cache's type, device, heads and columns")
    table = _table(n, positions, freq, axis, interleaved, q.get_device())
    slots = _ints("slots", slots, q.get_device(), n)
    out = _out(out, q, stream)
    _on_device_of(q, lib().mars_rope_append, (C.byref(table), cache._ref, *qp, *kp, *vp, *_heads("out", out, q), n, heads,
                                              positions.data_ptr(), slots, _stream(stream, q)))
    return out


class KvContext:
    """Working memory of the cache's operators on one device."""

    def __init__(self, max_requests: int, device: int = 0):
        h = C.c_void_p()
        _check(lib().mars_kv_ctx_create(device, max_requests, C.byref(h)))
        self.handle = h
        self.device = device

    def _given(self, stream):
        """The handle of a given stream (0: the context's own)."""
        return getattr(stream, "value", stream) or lib().mars_kv_ctx_stream(self.handle)

    def status(self):
        """Waits for the context's last call; raises MarsError (MARS_ERR_TIMEOUT) if a bounded wait of an attention call
        has given up since the last report.  Rows that it left without a result are NaN in out and lse."""
        _check(lib().mars_kv_ctx_status(self.handle))

    def debug_wait(self, limit_ns: int = 0, stall: bool = False) -> None:
        """Test hook: the attention kernels' waits give up after limit_ns (0: the default); stall: the next attention
        call's first CTA loads nothing, so that its waits run out."""
        _check(lib().mars_kv_ctx_debug_wait(self.handle, limit_ns, int(stall)))

    def release(self, kv_lens, finished, tables, free_pages, free_count, *, page_size, status=None, stream=None):
        """Push the pages of the requests with finished != 0 onto the free stack; returns the new
        (kv_lens, free_count).  A failure (status, one int32, if given) leaves everything as it was."""
        d, B = self.device, kv_lens.shape[0]
        pointers = (_ints("kv_lens", kv_lens, d), _ints("finished", finished, d, B), _ints("tables", tables, d, B, 2),
                    tables.shape[1], page_size, _ints("free_pages", free_pages, d), free_pages.shape[0],
                    _ints("free_count", free_count, d, 1))
        status = None if status is None else _ints("status", status, d, 1)
        if stream is None:
            lens_out, count_out = torch.empty_like(kv_lens), torch.empty_like(free_count)
        else:
            stream = self._given(stream)
            lens_out, count_out = (_empty(stream, x, x.shape, torch.int32) for x in (kv_lens, free_count))
        _check(lib().mars_kv_release(
            self.handle, B, *pointers, lens_out.data_ptr(), count_out.data_ptr(), status, _stream(stream, kv_lens)))
        return lens_out, count_out

    def plan(self, kv_lens, new_lens, tables, free_pages, free_count, *, page_size, max_tokens, stream=None) -> KvPlan:
        """Pages (into tables, in place), slots and positions for new_lens more tokens of each request."""
        d, B = self.device, kv_lens.shape[0]
        pointers = (_ints("kv_lens", kv_lens, d), _ints("new_lens", new_lens, d, B), _ints("tables", tables, d, B, 2),
                    tables.shape[1], page_size, _ints("free_pages", free_pages, d), free_pages.shape[0],
                    _ints("free_count", free_count, d, 1))
        if stream is not None:
            stream = self._given(stream)
        # one allocation for all that comes back
        lens_out, cu_new, slots, positions, count_out, status = _empty(
            stream, kv_lens, 2 * (B + max_tokens) + 3, torch.int32).split((B, B + 1, max_tokens, max_tokens, 1, 1))
        _check(lib().mars_kv_plan(
            self.handle, B, *pointers, max_tokens, lens_out.data_ptr(), count_out.data_ptr(),
            cu_new.data_ptr(), slots.data_ptr(), positions.data_ptr(), status.data_ptr(), _stream(stream, kv_lens)))
        return KvPlan(lens_out, cu_new, slots, positions, count_out, status)

    def attention(self, q, cache, tables, kv_lens, cu_new, *, max_new=None, scale=None, softcap=0.0, window=0,
                  decay=None, prefix_lens=None, out=None, return_lse=False, stream=None):
        """Attention of q [tokens, q_heads, head_dim], the requests' new tokens back to back (request b's from
        cu_new[b] to cu_new[b+1], already in the cache), over the pages of tables [B, pages].  kv_lens counts the
        new tokens.  A row at position i sees key j when j < prefix_lens[b], or j <= i and (window 0 or i - j <
        window); scores are scale * q.k (scale None: head_dim ** -0.5), capped by softcap * tanh(. / softcap), minus
        decay[head] * max(0, i - j).  No gradient.
        max_new: the most new tokens of one request.  It chooses the kernel, not the answer: up to 16 rows (max_new times
        the query heads of a key head) the one for single tokens.  Without it the call has to count on one request's having
        all tokens, and takes the one for chunks as soon as it has more than a few: give it to every step of single tokens.
        Returns out (q's shape and type), with return_lse also the fp32 [tokens, q_heads] log of the scores'
        exponentials' sum."""
        qp = _heads("q", q)
        n, heads, dim = q.shape
        if q.dtype is not cache.k.dtype or q.device != cache.k.device or dim != cache._c.head_dim:
            raise ValueError("q must have the cache's type, device and columns")
        d, B = self.device, kv_lens.shape[0]
        if q.get_device() != d:
            raise ValueError(f"the context works on cuda:{d}, q and the cache are on {q.device}")
        if decay is not None:
            decay = _floats("decay", decay, d, heads)
        pointers = (_ints("cu_new", cu_new, d, B + 1), _ints("kv_lens", kv_lens, d), _ints("tables", tables, d, B, 2),
                    tables.shape[1])
        if prefix_lens is not None:
            prefix_lens = _ints("prefix_lens", prefix_lens, d, B)
        if stream is not None:
            stream = self._given(stream)
        out = _out(out, q, stream)
        lse = _empty(stream, q, (n, heads), torch.float32) if return_lse else None
        # a window or bound beyond 32 bits is none (a C field would keep its low bits)
        cfg = _Config(dim ** -0.5 if scale is None else scale, softcap, min(window, _INT32_MAX),
                      min(n if max_new is None else max_new, _INT32_MAX))
        _check(lib().mars_paged_attention(
            self.handle, cache._ref, *qp, n, heads, B, *pointers, C.byref(cfg), decay, prefix_lens, *_heads("out", out, q),
            None if lse is None else lse.data_ptr(), _stream(stream, q)))
        return (out, lse) if return_lse else out

    def close(self):
        if getattr(self, "handle", None):
            lib().mars_kv_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
