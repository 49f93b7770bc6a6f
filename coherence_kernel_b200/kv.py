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
from .ops import _FLOATS, TYPE_NUMBERS, _call, _dev, _ptr, _stream


@dataclass
class Plan:
    """What ck_kv_plan wrote: one step's view of the cache.  Its buffers are checked when they are set."""
    length: torch.Tensor      # int32 [nreq] tokens held
    kv_len: torch.Tensor      # int32 [nreq] tokens the request's rows attend over (0: not served)
    q_start: torch.Tensor     # int32 [nreq + 1] first row of each request
    slots: torch.Tensor       # int64 [ntok] cache slot of every row, -1 for none
    positions: torch.Tensor   # int32 [ntok] position in its request, -1 for none
    free_count: torch.Tensor  # int32 [1] free pages left

    def __setattr__(self, name, value):
        old = self.__dict__.get(name)
        object.__setattr__(self, name, value)
        if old is not None:  # a buffer replaced after the first check
            try:
                self.__post_init__()
            except ValueError:
                object.__setattr__(self, name, old)
                raise

    def __post_init__(self):
        n = self.length.numel()
        for t, name, dt, k in ((self.length, "length", torch.int32, n), (self.kv_len, "kv_len", torch.int32, n),
                               (self.q_start, "q_start", torch.int32, n + 1),
                               (self.slots, "slots", torch.int64, self.slots.numel()),
                               (self.positions, "positions", torch.int32, self.slots.numel()),
                               (self.free_count, "free_count", torch.int32, 1)):
            _dev(t, name, dt, k)
            if t.device != self.length.device:
                raise ValueError("the plan's buffers must be on one device")
        # a plan of exactly n requests and ntok rows says so, so that a step into it checks one thing
        ntok = self.slots.numel()
        exact = self.kv_len.numel() == n and self.q_start.numel() == n + 1 and self.positions.numel() == ntok
        object.__setattr__(self, "_fits", (n, ntok, self.length.device) if exact else None)

    def cut(self, nreq: int, ntok: int, device) -> Plan:
        """The plan of nreq requests and ntok rows in these buffers: itself, or views of their first elements."""
        if self._fits == (nreq, ntok, device):
            return self
        if self.length.numel() < nreq or self.slots.numel() < ntok or self.length.device != device:
            raise ValueError(f"out holds less than {nreq} requests and {ntok} rows, or is not on {device}")
        return Plan(self.length[:nreq], self.kv_len[:nreq], self.q_start[:nreq + 1], self.slots[:ntok],
                    self.positions[:ntok], self.free_count)


def plan_buffers(nreq: int, ntok: int, device) -> Plan:
    """Output buffers of `plan` for steps of nreq requests and ntok rows."""
    i = lambda *n: torch.empty(n, dtype=torch.int32, device=device)
    return Plan(i(nreq), i(nreq), i(nreq + 1), torch.empty(ntok, dtype=torch.int64, device=device), i(ntok), i(1))


_I32 = torch.int32


def _ints(t, name, n, device):
    """A contiguous int32 tensor of at least n elements on the device; returns its address."""
    if t.dtype is not _I32 or t.device != device or not t.is_contiguous() or t.numel() < n:
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} elements on {device}")
    return t.data_ptr()


def _rows3(t, name, shape, kinds, device):
    """A tensor [n, heads, dim] of this shape with contiguous rows; returns the row stride."""
    if t.shape != shape or t.dtype not in kinds or t.device != device:
        raise ValueError(f"{name} must be {list(shape)} on {device}, of {' or '.join(map(str, kinds))}")
    n, h, d = shape
    row, head, one = t.stride()
    if (one != 1 and d > 1) or (head != d and h > 1) or (row < h * d and n > 1):
        raise ValueError(f"{name}'s rows must be contiguous")
    return row if n > 1 else h * d


def _table(t, device):
    row, col = t.stride()
    n, w = t.shape
    if t.dtype is not _I32 or t.device != device or (col != 1 and w > 1) or (row < w and n > 1):
        raise ValueError(f"table must be int32 [nreq, max_blocks] on {device} with contiguous rows")
    return row if n > 1 else w


def plan(table, length, new_tokens, free_blocks, free_count, block_tokens: int, ntok: int, out: Plan | None = None) -> Plan:
    """Block tables and slot maps of one step (ck_kv_plan): table int32 [nreq, max_blocks] and
    free_blocks int32 [n_blocks] are updated in place; length and free_count are read, and the new
    ones are in the returned plan (whose tensors may be these).  out may be larger than the step: the
    returned plan is then its first nreq requests and ntok rows."""
    dev, shape = table.device, table.shape
    if dev.type != "cuda" or len(shape) != 2:
        raise ValueError("table must be a CUDA tensor [nreq, max_blocks]")
    nreq, max_blocks = shape
    stride = _table(table, dev)
    if out is None:
        o = plan_buffers(nreq, ntok, dev)
    else:
        o = out.cut(nreq, ntok, dev)
    _call("ck_kv_plan", dev, _ints(length, "length", nreq, dev), _ints(new_tokens, "new_tokens", nreq, dev), nreq,
          table.data_ptr(), stride, max_blocks, _ints(free_blocks, "free_blocks", 1, dev),
          _ints(free_count, "free_count", 1, dev), free_blocks.numel(), block_tokens, ntok, o.length.data_ptr(),
          o.free_count.data_ptr(), o.kv_len.data_ptr(), o.q_start.data_ptr(), o.slots.data_ptr(),
          o.positions.data_ptr())
    return o


def _window(window):
    """A window as the C argument: none (0) or a length; one past 32 bits bounds nothing, as any past the table's."""
    if window < 0:
        raise ValueError("window must not be negative")
    return window if window < 1 << 31 else 0


def _config(k_cache, v_cache):
    """ck_kv_config of cache tensors [n_blocks, block_tokens, n_kv_heads, head_dim] (any strides with
    contiguous heads, so a [n_blocks, n_kv_heads, block_tokens, head_dim] cache is passed permuted)."""
    kt, st, shape, dev = k_cache.dtype, k_cache.stride(), k_cache.shape, k_cache.device
    if len(st) != 4 or shape != v_cache.shape or kt is not v_cache.dtype or st != v_cache.stride() or st[3] != 1:
        raise ValueError("k_cache and v_cache must be 4-dimensional, of one shape, type and strides, heads contiguous")
    if kt is not torch.bfloat16 and kt is not torch.float16:
        raise ValueError(f"the cache has dtype {kt}, expected bfloat16 or float16")
    if dev.type != "cuda" or v_cache.device != dev:
        raise ValueError("the cache must be CUDA tensors on one device")
    nb, bt, h, d = shape
    return _lib.KvConfig(h, d, bt, nb, TYPE_NUMBERS[kt], 0, st[0], st[1], st[2])


def append(k, v, k_cache, v_cache, slots):
    """K/V rows [ntok, n_kv_heads, head_dim] (f32, f16 or bf16) into the cache at `slots` (int64 [ntok],
    distinct; those outside the cache are skipped), rounded to the cache's type (ck_kv_append)."""
    cfg = _config(k_cache, v_cache)
    dev, ntok = k_cache.device, k.shape[0]
    shape = (ntok, cfg.n_kv_heads, cfg.head_dim)
    ks = _rows3(k, "k", shape, _FLOATS, dev)
    vs = _rows3(v, "v", shape, (k.dtype,), dev)
    if slots.dtype is not torch.int64 or slots.device != dev or slots.numel() < ntok or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 tensor of {ntok} elements on {dev}")
    _call("ck_kv_append", dev, ctypes.byref(cfg), TYPE_NUMBERS[k.dtype], k.data_ptr(), ks, v.data_ptr(), vs,
          slots.data_ptr(), ntok, k_cache.data_ptr(), v_cache.data_ptr())


class PagedAttention:
    """Attention of each request's new tokens over a paged cache (ck_paged_attention), with its
    workspace.  Calls that overlap in time (other streams, graphs replayed together) need an object
    each, and the object has to be kept until its calls are done."""

    def __init__(self, n_heads: int, n_kv_heads: int, head_dim: int, max_tokens: int, max_requests: int,
                 device="cuda"):
        self.n_heads, self.n_kv_heads, self.head_dim = n_heads, n_kv_heads, head_dim
        self.max_tokens, self.max_requests = max_tokens, max_requests
        self.ws_bytes = _lib.load().ck_paged_attention_workspace_bytes(n_heads, n_kv_heads, head_dim)
        if self.ws_bytes == 0:
            raise ValueError(f"unsupported heads: {n_heads} over {n_kv_heads} of {head_dim}")
        self.ws = torch.zeros(self.ws_bytes, dtype=torch.uint8, device=device)
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(self.ws.device).synchronize()  # zero before the first call on any stream

    def __call__(self, q, k_cache, v_cache, table, kv_len, q_start, scale: float | None = None, causal: bool = True,
                 window: int = 0, out=None, lse=None, return_lse: bool = False):
        """q [ntok, n_heads, head_dim] in the cache's type or f32 -> out of q's type (and lse fp32
        [ntok, n_heads] with return_lse).  Rows from q_start[nreq] on are not written."""
        cfg = _config(k_cache, v_cache)
        heads, dim, dev = self.n_heads, self.head_dim, k_cache.device
        if cfg.n_kv_heads != self.n_kv_heads or cfg.head_dim != dim or self.ws.device != dev:
            raise ValueError("the cache's heads or device are not those this object was made for")
        ntok = q.shape[0]
        nreq, max_blocks = table.shape
        if ntok > self.max_tokens or nreq > self.max_requests:
            raise ValueError("more rows or requests than this object was made for")
        shape = (ntok, heads, dim)
        qs = _rows3(q, "q", shape, (k_cache.dtype, torch.float32), dev)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            os_ = heads * dim
        else:
            os_ = _rows3(out, "out", shape, (q.dtype,), dev)
        if lse is None:
            if return_lse:
                lse = torch.empty((ntok, heads), dtype=torch.float32, device=dev)
        elif lse.device != dev:
            raise ValueError(f"lse must be on {dev}")
        else:
            _dev(lse, "lse", torch.float32, ntok * heads)
        _call("ck_paged_attention", dev, ctypes.byref(cfg), heads, TYPE_NUMBERS[q.dtype], q.data_ptr(), qs,
              k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), _table(table, dev), max_blocks,
              _ints(kv_len, "kv_len", nreq, dev), _ints(q_start, "q_start", nreq + 1, dev), nreq, ntok,
              1.0 / math.sqrt(dim) if scale is None else scale, int(causal), _window(window), out.data_ptr(), os_,
              None if lse is None else lse.data_ptr(), self.ws.data_ptr(), self.ws_bytes)
        return (out, lse) if return_lse else out

    def status(self):
        """Synchronize and raise if a device-side wait of the last call gave up."""
        with torch.cuda.device(self.ws.device):
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
        the state, n = len(new_tokens).  The step's append and attention take the returned plan, which
        holds n requests and ntok rows also where `out` has room for more."""
        n = new_tokens.numel()
        if n > self.max_requests or ntok > self.max_tokens:
            raise ValueError("more requests or rows than the cache was made for")
        if out is None:
            b = plan_buffers(n, ntok, self.k.device)
            out = Plan(self.length[:n], b.kv_len, b.q_start, b.slots, b.positions, self.free_count)
        elif out.length.data_ptr() != self.length.data_ptr() or out.free_count.data_ptr() != self.free_count.data_ptr():
            raise ValueError("out must come from this cache's step_buffers")
        return plan(self.table[:n], self.length[:n], new_tokens, self.free_blocks, self.free_count, self.block_tokens,
                    ntok, out=out)

    def step_buffers(self, nreq: int, ntok: int) -> Plan:
        """Buffers for `plan` calls of nreq requests and ntok rows, over this cache's state (for captured steps)."""
        b = plan_buffers(nreq, ntok, self.k.device)
        return Plan(self.length[:nreq], b.kv_len, b.q_start, b.slots, b.positions, self.free_count)

    def append(self, k, v, plan: Plan):
        append(k, v, self.k, self.v, plan.slots)

    def attend(self, q, plan: Plan, **kw):
        return self.attention(q, self.k, self.v, self.table[:plan.kv_len.numel()], plan.kv_len, plan.q_start, **kw)
