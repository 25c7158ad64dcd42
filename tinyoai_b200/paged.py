"""Operators of a serving step over a paged KV cache held as torch tensors.

The host-side mirror of the header section "Operators over a paged KV cache
the caller holds in device memory" (include/tinyoai_cuda.h, which states the
mathematics, the types and the limits). A step over a cache:

    cache = paged.Cache(k, v)                      # [pages, KV heads, positions, head size]
    plan = paged.StepPlan(max_requests, max_tokens, cache.page_tokens, k.device)
    plan.build(held, fresh, tables, free_pages)    # block tables, positions, slots
    q = cache.append(qkv, heads, plan.positions, plan.slots, rotary=..., norm=...)
    cache.page_means(plan.slots, means)            # for attend_sparse
    out = cache.attend(q, tables, plan.starts, plan.lengths, max_fresh, prefix=prompt_pages)
    out, pages = cache.attend_sparse(q, means, tables, plan.starts, plan.lengths, max_fresh, top=64)

Every call queues its work on `stream` (a torch.cuda.Stream; None: torch's
current stream of the cache's device) and returns. Nothing synchronises, so
the calls can be captured into CUDA graphs; results and workspaces come from
torch's allocator unless `out` is given. A tensor that was made on another
stream has to be ordered with `stream` by the caller, as for any torch call.
Bad arguments raise BackendError with the library's TCU_EINVAL or TCU_EUNSUP.
"""
import ctypes as C
import math

import torch

from . import _lib
from ._lib import BackendError, check, lib

__all__ = ["Cache", "HeadNorm", "Rotary", "StepPlan"]

_CODES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_NORMS = {"none": _lib.NORM_NONE, "rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}


def _bad(message):
    return BackendError(_lib.TCU_EINVAL, message)


def _code(name, t):
    c = _CODES.get(t.dtype)
    if c is None:
        raise BackendError(_lib.TCU_EUNSUP, f"{name} is {t.dtype}: float32, float16 and bfloat16 are possible")
    return c


def _whole(name, t, dtype, device, dims=1):
    """A contiguous tensor of whole numbers (its rows may lie apart when dims is 2)."""
    if t.dtype != dtype or t.dim() != dims or t.device != device:
        raise _bad(f"{name} must be a {dims}-d {dtype} tensor on {device}, got {t.dim()}-d {t.dtype} on {t.device}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise _bad(f"{name} is not contiguous")
    return t.data_ptr()


def _stream(stream, device):
    return (torch.cuda.current_stream(device) if stream is None else stream).cuda_stream


def _on_gpu(name, t):
    if t.device.type != "cuda":
        raise _bad(f"{name} must be on a GPU, got {t.device}")
    return t.device


class Rotary:
    """Rotation of query and key heads: table [positions, pairs, 2] of
    (cos, sin), float32. Pair i is features (i, i + pairs), or (2i, 2i + 1)
    when adjacent."""

    def __init__(self, table, adjacent=False):
        _on_gpu("rotary table", table)
        if table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32 or not table.is_contiguous():
            raise _bad("the rotary table is a contiguous float32 tensor [positions, pairs, 2]")
        self.table = table
        self.struct = _lib.Rotary(table.data_ptr(), table.shape[0], table.shape[1], 1 if adjacent else 0)


class HeadNorm:
    """Norm of each query and key head: kind "rms" or "layer", float32
    weights [heads, head size] (or [1, head size], shared by all heads)."""

    def __init__(self, kind, q_weight, k_weight, eps):
        if kind not in _NORMS:
            raise _bad(f"unknown norm {kind!r}")
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            _on_gpu(name, w)
            if w.dim() != 2 or w.dtype != torch.float32 or not w.is_contiguous() or w.device != q_weight.device:
                raise _bad(f"{name} is a contiguous float32 tensor [heads or 1, head size]")
        if q_weight.shape[1] != k_weight.shape[1]:
            raise _bad("query and key weights are of one head size")
        self.q_weight, self.k_weight = q_weight, k_weight
        # One row of each is every head's; otherwise append checks that there is a row for each head.
        self.shared = q_weight.shape[0] == 1 and k_weight.shape[0] == 1
        self.struct = _lib.HeadNorm(_NORMS[kind], float(eps), q_weight.data_ptr(), k_weight.data_ptr(), 0 if self.shared else q_weight.shape[1])


class StepPlan:
    """Block tables, positions and slots of a step, built on the GPU
    (tcu_plan_step). Holds the step's buffers, so that steps allocate nothing:
    for up to max_requests requests and capacity tokens

      starts     int32 [requests + 1]   first token of each request
      lengths    int32 [requests]       positions after the step
      positions  int32 [capacity]       of each token, -1 behind the last
      slots      int64 [capacity]       page * page_tokens + offset, -1 behind the last
      counts     int32 [3]              requests planned, tokens planned, pages taken

    starts and lengths are views of the last build's requests."""

    def __init__(self, max_requests, capacity, page_tokens, device="cuda"):
        if max_requests < 0 or capacity < 0:
            raise _bad("negative capacity")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise _bad(f"a step plan lives on a GPU, not on {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.max_requests, self.capacity, self.page_tokens = max_requests, capacity, page_tokens
        self._starts = torch.zeros(max_requests + 1, dtype=torch.int32, device=self.device)
        self._lengths = torch.zeros(max_requests, dtype=torch.int32, device=self.device)
        self.starts, self.lengths = self._starts, self._lengths
        self.positions = torch.full((capacity,), -1, dtype=torch.int32, device=self.device)
        self.slots = torch.full((capacity,), -1, dtype=torch.int64, device=self.device)
        self.counts = torch.zeros(3, dtype=torch.int32, device=self.device)
        self._outs = (self._starts.data_ptr(), self._lengths.data_ptr(), self.positions.data_ptr(), self.slots.data_ptr(),
                      self.counts.data_ptr())

    def build(self, held, fresh, tables, free_pages, stream=None):
        """held, fresh: int32 [requests], positions held and tokens added;
        tables: int32 [requests, width], updated in place; free_pages: int32.
        Returns self."""
        d = self.device
        n = held.shape[0] if held.dim() == 1 else -1
        h, f = _whole("held", held, torch.int32, d), _whole("fresh", fresh, torch.int32, d)
        t, p = _whole("tables", tables, torch.int32, d, 2), _whole("free_pages", free_pages, torch.int32, d)
        if fresh.shape[0] != n or tables.shape[0] != n or n > self.max_requests:
            raise _bad(f"{n} requests held, {fresh.shape[0]} fresh, {tables.shape[0]} tables, room for {self.max_requests}")
        width = tables.shape[1]
        stride = tables.stride(0) if n > 1 else max(width, tables.stride(0))
        if self.starts.shape[0] != n + 1:
            self.starts, self.lengths = self._starts[:n + 1], self._lengths[:n]
        check(lib().tcu_plan_step(d.index, _stream(stream, d), n, h, f, self.page_tokens, t, width, stride, p, free_pages.shape[0],
                                  self.capacity, *self._outs))
        return self


class Cache:
    """A paged KV cache: k and v [pages, KV heads, positions of a page, head
    size], of one type and with the same strides (any order of the first three
    dimensions, the last one contiguous). The tensors stay the caller's."""

    def __init__(self, k, v):
        self.device = _on_gpu("k", k)
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise _bad("k and v are tensors [pages, KV heads, positions, head size] of one shape, type and device")
        if k.stride() != v.stride() or k.stride(3) != 1:
            raise _bad("k and v need the same strides and a contiguous last dimension")
        self.k, self.v, self.code = k, v, _code("the cache", k)
        self.num_pages, self.kv_heads, self.page_tokens, self.head_dim = k.shape
        self.struct = _lib.PagedKV(k.data_ptr(), v.data_ptr(), self.code, self.num_pages, self.page_tokens, self.kv_heads, self.head_dim,
                                   k.stride(0), k.stride(1), k.stride(2))
        self._ref = C.byref(self.struct)
        self._sized = (None, 0)

    def append(self, qkv, heads, positions, slots, rotary=None, norm=None, out=None, stream=None):
        """Norm and rotation of the step's rows and their append
        (tcu_paged_append). qkv: [rows, (heads + 2 KV heads) * head size];
        positions int32 and slots int64 [rows]. Returns the queries
        [rows, heads, head size]; rows that are skipped (slot -1) keep what
        `out` held."""
        d, hd = self.device, self.head_dim
        if qkv.dim() != 2 or qkv.device != d or qkv.shape[1] != (heads + 2 * self.kv_heads) * hd or qkv.stride(1) != 1:
            raise _bad(f"qkv must be rows of ({heads} + 2 * {self.kv_heads}) * {hd} values on {d}, got {tuple(qkv.shape)} on {qkv.device}")
        rows, code = qkv.shape[0], _code("qkv", qkv)
        p, s = _whole("positions", positions, torch.int32, d), _whole("slots", slots, torch.int64, d)
        if positions.shape[0] != rows or slots.shape[0] != rows:
            raise _bad(f"{rows} rows, {positions.shape[0]} positions, {slots.shape[0]} slots")
        if out is None:
            out = torch.empty((rows, heads, hd), dtype=qkv.dtype, device=d)
        elif out.shape != (rows, heads, hd) or out.dtype != qkv.dtype or out.device != d or out.stride(2) != 1 or (heads > 1 and out.stride(1) != hd):
            raise _bad(f"out must be [{rows}, {heads}, {hd}] of {qkv.dtype} on {d}, its heads contiguous")
        rot = nrm = None
        if rotary is not None:
            if rotary.table.device != d:
                raise _bad("the rotary table is on another device")
            rot = C.byref(rotary.struct)
        if norm is not None:
            if norm.q_weight.device != d or norm.q_weight.shape[1] != hd:
                raise _bad(f"norm weights of head size {norm.q_weight.shape[1]} on {norm.q_weight.device}, the cache has {hd} on {d}")
            if not norm.shared and (norm.q_weight.shape[0] != heads or norm.k_weight.shape[0] != self.kv_heads):
                raise _bad("norm weights per head must be [heads, head size] and [KV heads, head size]")
            nrm = C.byref(norm.struct)
        width = qkv.shape[1]
        check(lib().tcu_paged_append(d.index, _stream(stream, d), self._ref, code, rows, heads, qkv.data_ptr(),
                                     qkv.stride(0) if rows > 1 else max(width, qkv.stride(0)), p, s, rot, nrm, out.data_ptr(),
                                     out.stride(0) if rows > 1 else max(heads * hd, out.stride(0))))
        return out

    def page_means(self, slots, means, stream=None):
        """Mean keys of the pages that the step's slots complete
        (tcu_paged_means), into means [pages, KV heads, head size] of the
        cache's type. Returns means."""
        self._check_means(means)
        s = _whole("slots", slots, torch.int64, self.device)
        check(lib().tcu_paged_means(self.device.index, _stream(stream, self.device), self._ref, slots.shape[0], s, means.data_ptr()))
        return means

    def attend(self, q, tables, starts, lengths, max_fresh, prefix=None, scale=None, max_length=0, out=None, stream=None):
        """Attention of the step's queries (tcu_paged_attend). q: [rows,
        heads, head size]; tables int32 [requests, width]; starts int32
        [requests + 1] and lengths int32 [requests] as StepPlan gives them;
        max_fresh: the most rows of one request; prefix: int32 pages that all
        requests begin with, read once for all; scale: 1 / sqrt(head size) by
        default; max_length: a bound on lengths, where the host knows one
        (sizes the work; 0: what the tables map). Returns out [rows, heads,
        head size]; rows behind starts[-1] keep what `out` held."""
        d = self.device
        out, queries = self._queries(q, tables, starts, lengths, max_fresh, scale, out)
        pages, at = 0, None
        if prefix is not None:
            at, pages = _whole("prefix", prefix, torch.int32, d), prefix.shape[0]
        ref = C.byref(queries)
        key = (0, q.dtype, q.shape, tables.shape, max_fresh, pages, max_length)
        size = self._workspace_bytes(key, lambda n: lib().tcu_paged_attend_workspace(self._ref, ref, pages, max_length, n))
        work = torch.empty(size, dtype=torch.uint8, device=d) if stream is None else self._on(stream, size)
        check(lib().tcu_paged_attend(d.index, _stream(stream, d), self._ref, ref, at, pages, max_length, work.data_ptr(), size))
        return out

    def attend_sparse(self, q, means, tables, starts, lengths, max_fresh, top, first=1, last=1, scale=None, out=None, pages=None, stream=None):
        """Attention of each query over its first, last and `top` best pages
        (tcu_paged_attend_sparse); arguments as for attend, means as
        page_means keeps them. Returns (out, pages): pages int32 [rows, KV
        heads, first + last + top], the logical pages read, ascending, -1
        behind them."""
        d = self.device
        self._check_means(means)
        out, queries = self._queries(q, tables, starts, lengths, max_fresh, scale, out)
        shape = (q.shape[0], self.kv_heads, first + last + top)
        if min(first, top) < 0 or last < 1:
            raise _bad(f"first {first} and top {top} must not be negative, last {last} must be at least 1")
        if pages is None:
            pages = torch.empty(shape, dtype=torch.int32, device=d)
        elif pages.shape != shape or pages.dtype != torch.int32 or pages.device != d or not pages.is_contiguous():
            raise _bad(f"pages must be a contiguous int32 tensor {shape} on {d}")
        ref = C.byref(queries)
        key = (1, q.dtype, q.shape, tables.shape, max_fresh, first, last, top)
        size = self._workspace_bytes(key, lambda n: lib().tcu_paged_attend_sparse_workspace(self._ref, ref, first, last, top, n))
        work = torch.empty(size, dtype=torch.uint8, device=d) if stream is None else self._on(stream, size)
        check(lib().tcu_paged_attend_sparse(d.index, _stream(stream, d), self._ref, ref, means.data_ptr(), first, last, top, pages.data_ptr(),
                                            work.data_ptr(), size))
        return out, pages

    def _on(self, stream, size):
        """A workspace that torch's allocator hands out again only behind `stream`."""
        with torch.cuda.stream(stream):
            return torch.empty(size, dtype=torch.uint8, device=self.device)

    def _workspace_bytes(self, key, ask):
        """The size the library asks for; the last answer is kept for calls of the same shape."""
        if self._sized[0] != key:
            n = C.c_uint64()
            check(ask(C.byref(n)))
            self._sized = (key, n.value)
        return self._sized[1]

    def _check_means(self, means):
        if means.shape != (self.num_pages, self.kv_heads, self.head_dim) or means.dtype != self.k.dtype or means.device != self.device or not means.is_contiguous():
            raise _bad(f"means must be a contiguous {self.k.dtype} tensor {(self.num_pages, self.kv_heads, self.head_dim)} on {self.device}")

    def _queries(self, q, tables, starts, lengths, max_fresh, scale, out):
        d, hd = self.device, self.head_dim
        if q.dim() != 3 or q.shape[2] != hd or q.device != d or q.stride(2) != 1:
            raise _bad(f"q must be [rows, heads, {hd}] on {d}, its last dimension contiguous, got {tuple(q.shape)} on {q.device}")
        rows, heads, _ = q.shape
        st, le, tb = _whole("starts", starts, torch.int32, d), _whole("lengths", lengths, torch.int32, d), _whole("tables", tables, torch.int32, d, 2)
        n, width = tables.shape
        if lengths.shape[0] != n or starts.shape[0] != n + 1:
            raise _bad(f"{n} tables, {lengths.shape[0]} lengths, {starts.shape[0]} starts")
        if out is None:
            out = torch.empty((rows, heads, hd), dtype=q.dtype, device=d)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != d or out.stride(2) != 1:
            raise _bad(f"out must be {tuple(q.shape)} of {q.dtype} on {d}, its last dimension contiguous")
        stride = tables.stride(0) if n > 1 else max(width, tables.stride(0))
        return out, _lib.PagedQueries(_code("q", q), n, rows, heads, max_fresh, width, q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(),
                                      out.stride(0), out.stride(1), st, le, tb, stride, 1.0 / math.sqrt(hd) if scale is None else scale)
