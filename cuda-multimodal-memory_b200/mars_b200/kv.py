"""The operators of an answering step on a paged key/value cache.

A step of a program that answers with retrieved memories:

    lens, count = ctx.release(lens, finished, tables, free, count, page_size=64)
    plan = ctx.plan(lens, new_lens, tables, free, count, page_size=64, max_tokens=n)

All arguments are torch CUDA tensors; calls run on torch's current stream
unless one is given, and return without waiting.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _check, _stream, lib

KV_MAX_REQUESTS = 8192   # MARS_KV_MAX_REQUESTS

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


def _ints(name, t, n=None, dims=1):
    """The address of a contiguous int32 CUDA tensor of n entries (n None: any)."""
    if t.dtype is not torch.int32 or not t.is_cuda or not t.is_contiguous() or t.dim() != dims:
        raise ValueError(f"{name} must be a contiguous int32 CUDA tensor of {dims} dimension(s)")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{name} must have {n} entries, has {t.shape[0]}")
    return t.data_ptr()


class KvContext:
    """Working memory of the cache's operators on one device."""

    def __init__(self, max_requests: int, device: int = 0):
        h = C.c_void_p()
        _check(lib().mars_kv_ctx_create(device, max_requests, C.byref(h)))
        self.handle = h
        self.device = device

    def release(self, kv_lens, finished, tables, free_pages, free_count, *, page_size, status=None, stream=None):
        """Push the pages of the requests with finished != 0 onto the free stack; returns the new
        (kv_lens, free_count).  A failure (status, one int32, if given) leaves everything as it was."""
        B = kv_lens.shape[0]
        lens_out, count_out = torch.empty_like(kv_lens), torch.empty_like(free_count)
        _check(lib().mars_kv_release(
            self.handle, B, _ints("kv_lens", kv_lens), _ints("finished", finished, B),
            _ints("tables", tables, B, 2), tables.shape[1], page_size, _ints("free_pages", free_pages),
            free_pages.shape[0], _ints("free_count", free_count, 1), lens_out.data_ptr(), count_out.data_ptr(),
            None if status is None else _ints("status", status, 1), _stream(stream, kv_lens)))
        return lens_out, count_out

    def plan(self, kv_lens, new_lens, tables, free_pages, free_count, *, page_size, max_tokens, stream=None) -> KvPlan:
        """Pages (into tables, in place), slots and positions for new_lens more tokens of each request."""
        B = kv_lens.shape[0]
        dev = kv_lens.device
        lens_out, count_out = torch.empty_like(kv_lens), torch.empty_like(free_count)
        cu_new = torch.empty(B + 1, dtype=torch.int32, device=dev)
        slots = torch.empty(max_tokens, dtype=torch.int32, device=dev)
        positions = torch.empty(max_tokens, dtype=torch.int32, device=dev)
        status = torch.empty(1, dtype=torch.int32, device=dev)
        _check(lib().mars_kv_plan(
            self.handle, B, _ints("kv_lens", kv_lens), _ints("new_lens", new_lens, B), _ints("tables", tables, B, 2),
            tables.shape[1], page_size, _ints("free_pages", free_pages), free_pages.shape[0],
            _ints("free_count", free_count, 1), max_tokens, lens_out.data_ptr(), count_out.data_ptr(),
            cu_new.data_ptr(), slots.data_ptr(), positions.data_ptr(), status.data_ptr(), _stream(stream, kv_lens)))
        return KvPlan(lens_out, cu_new, slots, positions, count_out, status)

    def close(self):
        if getattr(self, "handle", None):
            lib().mars_kv_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
