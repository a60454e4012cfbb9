"""Serving many requests from one paged KV cache (tlx_paged_* of libtlx_b200).

    table = PageTable(requests, width, pages, page_size)       # block tables, free pages
    cache = PagedCache.empty(pages, page_size, kv_heads, head_dim, "int8")
    attn  = PagedAttention(heads, kv_heads, head_dim)

    plan = table.plan(cached_len, new_len, Plan(requests, n_tokens))   # once per step
    cache.append(k, v, plan.slots)                                      # per layer
    out = attn(cache, table.table, plan.q_start, plan.kv_len, q, gate=gate)

Lengths, tables and slots stay on the device: a step reads nothing back and can be
captured in a CUDA graph.  Tensors are only buffers, all on one device, which has to be
the current one; every call runs on its current stream, and a workspace (the PageTable's,
the PagedAttention's) must not be used by two calls that can overlap.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, ops
from ._lib import TLX_DT_BF16, TLX_DT_F16, TLX_DT_Q8, PagedKV, TLXError, check

NO_PAGES, TABLE_FULL, BAD_LENGTH = 1, 2, 3
_CACHE_DT = {torch.float16: TLX_DT_F16, torch.bfloat16: TLX_DT_BF16, torch.uint8: TLX_DT_Q8}


def _i32(t: torch.Tensor, n: int, name: str, device: torch.device) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or t.numel() < n:
        raise TLXError(f"{name} must be a contiguous int32 tensor of at least {n} entries on {device}")
    return t


class Plan:
    """What a step's kernels read, written by PageTable.plan: q_start [requests + 1],
    kv_len and status [requests], slots and positions [tokens] (all int32)."""

    def __init__(self, requests: int, tokens: int, device="cuda"):
        self.requests, self.tokens = int(requests), int(tokens)
        buf = torch.zeros(3 * self.requests + 1 + 2 * self.tokens, dtype=torch.int32, device=device)
        r, t = self.requests, self.tokens
        self.q_start, self.kv_len, self.status, self.slots, self.positions = buf.split([r + 1, r, r, t, t])


class PageTable:
    """Block tables of up to `requests` requests, `width` pages each, over a pool of
    `pages` pages: table [requests][width] (-1: no page), held [requests], and the free
    stack free[0 .. n_free).  Existing buffers may be given instead."""

    def __init__(self, requests: int, width: int, pages: int, page_size: int, table: torch.Tensor = None,
                 held: torch.Tensor = None, free: torch.Tensor = None, n_free: torch.Tensor = None, device="cuda"):
        ops.require_device()
        self.requests, self.width, self.pages, self.page_size = int(requests), int(width), int(pages), int(page_size)
        i32 = dict(dtype=torch.int32, device=device)
        self.table = table if table is not None else torch.full((self.requests, self.width), -1, **i32)
        self.held = held if held is not None else torch.zeros(self.requests, **i32)
        # pages leave from the end: a fresh pool hands out 0, 1, 2, ...
        self.free = free if free is not None else torch.arange(self.pages - 1, -1, -1, **i32)
        self.n_free = n_free if n_free is not None else torch.full((1,), self.pages, **i32)
        if (self.table.dtype != torch.int32 or not self.table.is_cuda or
                tuple(self.table.shape) != (self.requests, self.width) or self.table.stride(1) != 1):
            raise TLXError("table must be a row-major int32 [requests, width] CUDA tensor")
        dev = self.table.device
        _i32(self.held, self.requests, "held", dev)
        _i32(self.free, self.pages, "free", dev)
        _i32(self.n_free, 1, "n_free", dev)
        self.ws = ops.Workspace(int(_lib.lib().tlx_paged_plan_workspace_bytes()), self.table.device)

    def plan(self, cached_len: torch.Tensor, new_len: torch.Tensor, plan: Plan, held_out: torch.Tensor = None,
             n_free_out: torch.Tensor = None) -> Plan:
        """Gives every request the pages that its cached and new tokens need and fills
        `plan`.  held and n_free are updated in place unless other buffers are given."""
        n = plan.requests
        if n > self.requests:
            raise TLXError(f"the plan has {n} requests, the table {self.requests}")
        dev = self.table.device
        _i32(cached_len, n, "cached_len", dev)
        _i32(new_len, n, "new_len", dev)
        held_out = self.held if held_out is None else _i32(held_out, n, "held_out", dev)
        n_free_out = self.n_free if n_free_out is None else _i32(n_free_out, 1, "n_free_out", dev)
        for t in (plan.q_start, plan.kv_len, plan.status, plan.slots, plan.positions):
            if t.device != dev:
                raise TLXError("the plan must be on the table's device")
        rc = _lib.lib().tlx_paged_plan(
            cached_len.data_ptr(), new_len.data_ptr(), n, self.page_size, self.table.data_ptr(), self.table.stride(0),
            self.width, self.held.data_ptr(), held_out.data_ptr(), self.free.data_ptr(), self.pages,
            self.n_free.data_ptr(), n_free_out.data_ptr(), plan.tokens, plan.q_start.data_ptr(),
            plan.kv_len.data_ptr(), plan.slots.data_ptr(), plan.positions.data_ptr(), plan.status.data_ptr(),
            self.ws.buf.data_ptr(), self.ws.nbytes, ops._raw_stream(self.table))
        check(rc, "paged_plan")
        return plan

    def release(self, done: torch.Tensor) -> None:
        """Returns the pages of every request with done[b] != 0 to the free stack."""
        n = done.numel()
        if n > self.requests:
            raise TLXError(f"done has {n} entries, the table {self.requests} requests")
        _i32(done, 1, "done", self.table.device)
        check(_lib.lib().tlx_paged_release(done.data_ptr(), n, self.table.data_ptr(), self.table.stride(0), self.width,
                                           self.held.data_ptr(), self.free.data_ptr(), self.pages,
                                           self.n_free.data_ptr(), ops._raw_stream(self.table)), "paged_release")


class PagedCache:
    """A pool of K / V pages: k, v [pages][kv_heads][page_size][head_dim] fp16, bf16 or
    uint8 codes with fp16 scales [pages][kv_heads][page_size][head_dim / 32].  Any strides
    with contiguous rows (a [pages][page_size][kv_heads][head_dim] pool is its permuted
    view).  The object describes these very tensors: another pool is another PagedCache."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor = None, v_scale: torch.Tensor = None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or not k.is_cuda or v.device != k.device:
            raise TLXError("k and v must be CUDA [pages, kv_heads, page_size, head_dim] tensors of one dtype")
        if k.dtype not in _CACHE_DT:
            raise TLXError(f"a cache is fp16, bf16 or uint8 codes, not {k.dtype}")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise TLXError("the rows of k and v must be contiguous")
        q8 = k.dtype == torch.uint8
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        for s in (k_scale, v_scale):
            if q8 and (s is None or s.dtype != torch.float16 or s.device != k.device or s.stride(3) != 1 or
                       tuple(s.shape) != (*k.shape[:3], self.head_dim // 32)):
                raise TLXError("uint8 codes need fp16 scales [pages, kv_heads, page_size, head_dim / 32]")
            if not q8 and s is not None:
                raise TLXError("only uint8 codes have scales")
        self.q_dtype = torch.float16 if q8 else k.dtype
        none = (0, 0, 0)
        self.c = PagedKV(k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if q8 else None,
                         v_scale.data_ptr() if q8 else None, k.stride()[:3], v.stride()[:3],
                         k_scale.stride()[:3] if q8 else none, v_scale.stride()[:3] if q8 else none, self.pages,
                         self.page_size, self.kv_heads, self.head_dim, _CACHE_DT[k.dtype])
        self._ref = ctypes.byref(self.c)

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype="int8", device="cuda"):
        """dtype: torch.float16, torch.bfloat16 or "int8"."""
        shape = (pages, kv_heads, page_size, head_dim)
        if dtype == "int8":
            k, v = (torch.full(shape, 128, dtype=torch.uint8, device=device) for _ in range(2))
            ks, vs = (torch.zeros((*shape[:3], head_dim // 32), dtype=torch.float16, device=device) for _ in range(2))
            return cls(k, v, ks, vs)
        return cls(*(torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)))

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Rows k, v [tokens][kv_heads][head_dim] into their slots (slot -1: skipped)."""
        if (k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in ops._DT or
                k.stride(2) != 1 or v.stride(2) != 1 or k.device != self.k.device or v.device != self.k.device or
                k.shape[1] != self.kv_heads or k.shape[2] != self.head_dim):
            raise TLXError("k and v must be [tokens, kv_heads, head_dim] rows of one dtype on the cache's device")
        n = k.shape[0]
        _i32(slots, n, "slots", self.k.device)
        rc = _lib.lib().tlx_paged_append(self._ref, k.data_ptr(), v.data_ptr(), ops._DT[k.dtype], k.stride(0),
                                         k.stride(1), v.stride(0), v.stride(1), slots.data_ptr(), n, ops._raw_stream(k))
        check(rc, "paged_append")


class PagedAttention:
    """Attention of each request's new tokens over its pages (tlx_paged_attention), with
    the workspace for `heads` query heads on `kv_heads` KV heads of `head_dim`."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, device="cuda"):
        ops.require_device()
        self.heads, self.kv_heads, self.head_dim = int(heads), int(kv_heads), int(head_dim)
        nb = int(_lib.lib().tlx_paged_attention_workspace_bytes(self.heads, self.kv_heads, self.head_dim))
        if nb == 0:
            raise TLXError(f"unsupported heads: {heads} query, {kv_heads} KV, dim {head_dim}")
        self.ws = ops.Workspace(nb, device)
        self.scale = self.head_dim ** -0.5

    def __call__(self, cache: PagedCache, table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
                 q: torch.Tensor, gate: torch.Tensor = None, scale: float = None, max_new: int = None,
                 out: torch.Tensor = None) -> torch.Tensor:
        """q [tokens][heads][head_dim] -> out of the same shape; row t of request b's n new
        tokens sees keys 0 .. kv_len[b] - n + t.  gate: out is multiplied by its sigmoid.
        scale defaults to head_dim ** -0.5.  max_new: the most new tokens of any request
        (default: the number of rows)."""
        shape, dt = q.shape, cache.q_dtype
        if out is None:
            out = torch.empty(shape, dtype=dt, device=q.device)
        dev = cache.k.device
        if (len(shape) != 3 or shape[1] != self.heads or shape[2] != self.head_dim or q.dtype != dt or
                q.device != dev or out.shape != shape or out.dtype != dt or out.device != dev):
            raise TLXError(f"q and out must be {dt} [tokens, {self.heads}, {self.head_dim}] rows on the cache's device")
        n, (qt, qh, q1), (ot, oh, o1) = shape[0], q.stride(), out.stride()
        gp, gt, gh, g1 = None, 0, 0, 1
        if gate is not None:
            if gate.shape != shape or gate.dtype != dt or gate.device != dev:
                raise TLXError("gate must be rows like q's")
            gp, (gt, gh, g1) = gate.data_ptr(), gate.stride()
        if q1 != 1 or o1 != 1 or g1 != 1:
            raise TLXError("the rows of q, out and gate must be contiguous")
        if cache.kv_heads != self.kv_heads or cache.head_dim != self.head_dim:
            raise TLXError("the cache has other heads than this attention")
        if table.dtype != torch.int32 or table.dim() != 2 or table.device != dev or table.stride(1) != 1:
            raise TLXError("table must be a row-major int32 [requests, width] tensor on the cache's device")
        r = kv_len.numel()
        if table.shape[0] < r:
            raise TLXError(f"the table has {table.shape[0]} rows for {r} requests")
        _i32(kv_len, 1, "kv_len", dev)
        _i32(q_start, r + 1, "q_start", dev)
        if self.ws.buf.device != dev:
            raise TLXError("the attention's workspace is on another device than the cache")
        rc = _lib.lib().tlx_paged_attention(
            cache._ref, table.data_ptr(), table.stride(0), table.shape[1], q_start.data_ptr(), kv_len.data_ptr(), r,
            q.data_ptr(), ops._DT[dt], qt, qh, self.heads, n, n if max_new is None else max_new,
            self.scale if scale is None else scale, gp, gt, gh, out.data_ptr(), ot, oh, self.ws.buf.data_ptr(), self.ws.nbytes,
            ops._raw_stream(q))
        check(rc, "paged_attention")
        return out

    def error(self) -> int:
        """The error bits of the kernels' bounded waits; synchronous."""
        return self.ws.error()
