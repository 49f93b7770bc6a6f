"""A paged KV cache on the device and the attention over it (ck_kv_* and ck_paged_attention in
include/ck_b200.h).

The cache is `n_blocks` pages of `block_tokens` tokens, K and V each a tensor
[n_blocks, block_tokens, n_kv_heads, head_dim]; a request's tokens lie in the pages its table row
names.  Per step, on the current stream and without a host wait:

    plan = cache.plan(new_tokens, ntok)       # pages, slots and row offsets from the lengths
    cache.append(k, v, plan)                  # the step's K/V rows into the cache
    out = cache.attend(q, plan)               # every request's rows over its cached tokens

The state (lengths, tables, free pages) lives on the device and is advanced by `plan`, so a step
captured in a CUDA graph advances it at each replay.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from . import _lib
from .ops import TYPE_NUMBERS, _dev, _ptr, _stream


@dataclass
class Plan:
    """What ck_kv_plan wrote: one step's view of the cache."""
    length: torch.Tensor      # int32 [nreq] tokens held
    kv_len: torch.Tensor      # int32 [nreq] tokens the request's rows attend over (0: not served)
    q_start: torch.Tensor     # int32 [nreq + 1] first row of each request
    slots: torch.Tensor       # int64 [ntok] cache slot of every row, -1 for none
    positions: torch.Tensor   # int32 [ntok] position in its request, -1 for none
    free_count: torch.Tensor  # int32 [1] free pages left


def plan_buffers(nreq: int, ntok: int, device) -> Plan:
    """Output buffers of `plan` for steps of nreq requests and ntok rows."""
    i = lambda *n: torch.empty(n, dtype=torch.int32, device=device)
    return Plan(i(nreq), i(nreq), i(nreq + 1), torch.empty(ntok, dtype=torch.int64, device=device), i(ntok), i(1))


def _same_device(*tensors):
    dev = tensors[0].device
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors on {dev} and {t.device}")
    return torch.cuda.device(dev)


def _rows(t, name, dtype, *inner):
    """A tensor [n, *inner] whose rows are contiguous; returns its row stride in elements."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.dim() != 1 + len(inner) or tuple(t.shape[1:]) != tuple(inner):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected [n, {', '.join(map(str, inner))}]")
    step = 1
    for size, stride in zip(reversed(inner), reversed(t.stride()[1:])):
        if size != 1 and stride != step:
            raise ValueError(f"{name}'s rows must be contiguous")
        step *= size
    if t.shape[0] > 1 and t.stride(0) < step:
        raise ValueError(f"{name}'s rows overlap")
    return t.stride(0) if t.shape[0] > 1 else step


def plan(table, length, new_tokens, free_blocks, free_count, block_tokens: int, ntok: int, out: Plan | None = None) -> Plan:
    """Block tables and slot maps of one step (ck_kv_plan): table int32 [nreq, max_blocks] and
    free_blocks int32 [n_blocks] are updated in place; length and free_count are read, and the new
    ones are in the returned plan (whose tensors may be these)."""
    nreq, max_blocks = table.shape
    stride = _rows(table, "table", torch.int32, max_blocks)
    _dev(length, "length", torch.int32, nreq)
    _dev(new_tokens, "new_tokens", torch.int32, nreq)
    _dev(free_blocks, "free_blocks", torch.int32, 1)
    _dev(free_count, "free_count", torch.int32, 1)
    o = out if out is not None else plan_buffers(nreq, ntok, table.device)
    for t, n, dt, k in ((o.length, "out.length", torch.int32, nreq), (o.kv_len, "out.kv_len", torch.int32, nreq),
                        (o.q_start, "out.q_start", torch.int32, nreq + 1), (o.slots, "out.slots", torch.int64, ntok),
                        (o.positions, "out.positions", torch.int32, ntok),
                        (o.free_count, "out.free_count", torch.int32, 1)):
        _dev(t, n, dt, k)
    with _same_device(table, length, new_tokens, free_blocks, free_count, o.length, o.kv_len, o.q_start, o.slots,
                      o.positions, o.free_count):
        _lib.check(_lib.load().ck_kv_plan(_ptr(length), _ptr(new_tokens), nreq, _ptr(table), stride, max_blocks,
                                          _ptr(free_blocks), _ptr(free_count), free_blocks.numel(), block_tokens, ntok,
                                          _ptr(o.length), _ptr(o.free_count), _ptr(o.kv_len), _ptr(o.q_start),
                                          _ptr(o.slots), _ptr(o.positions), _stream()), "ck_kv_plan")
    return o


def _config(k_cache, v_cache):
    """ck_kv_config of cache tensors [n_blocks, block_tokens, n_kv_heads, head_dim] (any strides with
    contiguous heads, so a [n_blocks, n_kv_heads, block_tokens, head_dim] cache is passed permuted)."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError("k_cache and v_cache must be 4-dimensional, of one shape and type")
    if k_cache.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"the cache has dtype {k_cache.dtype}, expected bfloat16 or float16")
    if not k_cache.is_cuda or not v_cache.is_cuda:
        raise ValueError("the cache must be CUDA tensors")
    if k_cache.stride() != v_cache.stride() or k_cache.stride(3) != 1:
        raise ValueError("k_cache and v_cache need the same strides and contiguous heads")
    nb, bt, h, d = k_cache.shape
    sb, st, sh, _ = k_cache.stride()
    return _lib.KvConfig(h, d, bt, nb, TYPE_NUMBERS[k_cache.dtype], 0, sb, st, sh)


def append(k, v, k_cache, v_cache, slots):
    """K/V rows [ntok, n_kv_heads, head_dim] (f32, f16 or bf16) into the cache at `slots` (int64 [ntok],
    distinct; those outside the cache are skipped), rounded to the cache's type (ck_kv_append)."""
    cfg = _config(k_cache, v_cache)
    kinds = (torch.float32, torch.float16, torch.bfloat16)
    ks = _rows(k, "k", kinds, cfg.n_kv_heads, cfg.head_dim)
    vs = _rows(v, "v", k.dtype, cfg.n_kv_heads, cfg.head_dim)
    ntok = k.shape[0]
    if v.shape[0] != ntok:
        raise ValueError("k and v have different numbers of rows")
    _dev(slots, "slots", torch.int64, ntok)
    with _same_device(k, v, k_cache, v_cache, slots):
        _lib.check(_lib.load().ck_kv_append(ctypes.byref(cfg), TYPE_NUMBERS[k.dtype], _ptr(k), ks, _ptr(v), vs,
                                            _ptr(slots), ntok, _ptr(k_cache), _ptr(v_cache), _stream()), "ck_kv_append")


class PagedAttention:
    """Attention of each request's new tokens over a paged cache (ck_paged_attention), with its
    workspace.  Calls that overlap in time (other streams, graphs replayed together) need an object
    each."""

    def __init__(self, n_heads: int, n_kv_heads: int, head_dim: int, max_tokens: int, max_requests: int,
                 device="cuda"):
        self.n_heads, self.n_kv_heads, self.head_dim = n_heads, n_kv_heads, head_dim
        self.max_tokens, self.max_requests = max_tokens, max_requests
        self.ws_bytes = _lib.load().ck_paged_attention_workspace_bytes(n_heads, n_kv_heads, head_dim)
        if self.ws_bytes == 0:
            raise ValueError(f"unsupported heads: {n_heads} over {n_kv_heads} of {head_dim}")
        self.ws = torch.empty(self.ws_bytes, dtype=torch.uint8, device=device)

    def __call__(self, q, k_cache, v_cache, table, kv_len, q_start, scale: float | None = None, causal: bool = True,
                 window: int = 0, out=None, lse=None, return_lse: bool = False):
        """q [ntok, n_heads, head_dim] in the cache's type or f32 -> out of q's type (and lse fp32
        [ntok, n_heads] with return_lse).  Rows from q_start[nreq] on are not written."""
        cfg = _config(k_cache, v_cache)
        if (cfg.n_kv_heads, cfg.head_dim) != (self.n_kv_heads, self.head_dim):
            raise ValueError("the cache's heads are not those this object was made for")
        qs = _rows(q, "q", (torch.float32, k_cache.dtype), self.n_heads, self.head_dim)
        ntok = q.shape[0]
        nreq, max_blocks = table.shape
        if ntok > self.max_tokens or nreq > self.max_requests:
            raise ValueError("more rows or requests than this object was made for")
        ts = _rows(table, "table", torch.int32, max_blocks)
        _dev(kv_len, "kv_len", torch.int32, nreq)
        _dev(q_start, "q_start", torch.int32, nreq + 1)
        if out is None:
            out = torch.empty((ntok, self.n_heads, self.head_dim), dtype=q.dtype, device=q.device)
        os_ = _rows(out, "out", q.dtype, self.n_heads, self.head_dim)
        if out.shape[0] < ntok:
            raise ValueError("out has fewer rows than q")
        if return_lse and lse is None:
            lse = torch.empty((ntok, self.n_heads), dtype=torch.float32, device=q.device)
        if lse is not None:
            _dev(lse, "lse", torch.float32, ntok * self.n_heads)
        with _same_device(q, k_cache, v_cache, table, kv_len, q_start, out, lse, self.ws):
            _lib.check(_lib.load().ck_paged_attention(
                ctypes.byref(cfg), self.n_heads, TYPE_NUMBERS[q.dtype], _ptr(q), qs, _ptr(k_cache), _ptr(v_cache),
                _ptr(table), ts, max_blocks, _ptr(kv_len), _ptr(q_start), nreq, ntok,
                1.0 / math.sqrt(self.head_dim) if scale is None else scale, int(causal), window, _ptr(out), os_,
                _ptr(lse), _ptr(self.ws), self.ws_bytes, _stream()), "ck_paged_attention")
        return (out, lse) if return_lse else out

    def status(self):
        """Synchronize and raise if a device-side wait of the last call gave up."""
        _lib.check(_lib.load().ck_paged_attention_status(_ptr(self.ws), _stream()), "ck_paged_attention_status")


class PagedKV:
    """A paged KV cache with its state on the device: pages, request lengths, tables, free pages."""

    def __init__(self, n_blocks: int, block_tokens: int, n_heads: int, n_kv_heads: int, head_dim: int,
                 max_requests: int, max_blocks: int, max_tokens: int, dtype=torch.bfloat16, device="cuda"):
        shape = (n_blocks, block_tokens, n_kv_heads, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        i = lambda *n: torch.zeros(n, dtype=torch.int32, device=device)
        self.table, self.length = i(max_requests, max_blocks), i(max_requests)
        # the lowest pages on top of the stack
        self.free_blocks = torch.arange(n_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), n_blocks, dtype=torch.int32, device=device)
        self.block_tokens, self.max_requests, self.max_tokens = block_tokens, max_requests, max_tokens
        self.attention = PagedAttention(n_heads, n_kv_heads, head_dim, max_tokens, max_requests, device)

    def plan(self, new_tokens, ntok: int, out: Plan | None = None) -> Plan:
        """Advance the state by one step: request r gets new_tokens[r] rows (int32, on the device), or
        drops its last -new_tokens[r] tokens; ntok >= the step's rows.  Requests are rows 0 .. n - 1 of
        the state, n = len(new_tokens)."""
        n = new_tokens.numel()
        if n > self.max_requests or ntok > self.max_tokens:
            raise ValueError("more requests or rows than the cache was made for")
        o = out if out is not None else plan_buffers(n, ntok, self.k.device)
        o.length, o.free_count = self.length[:n], self.free_count
        return plan(self.table[:n], self.length[:n], new_tokens, self.free_blocks, self.free_count, self.block_tokens,
                    ntok, out=o)

    def append(self, k, v, plan: Plan):
        append(k, v, self.k, self.v, plan.slots)

    def attend(self, q, plan: Plan, **kw):
        return self.attention(q, self.k, self.v, self.table[:plan.kv_len.numel()], plan.kv_len, plan.q_start, **kw)
