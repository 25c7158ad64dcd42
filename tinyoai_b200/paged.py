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
torch's allocator, on that stream, unless `out` is given. A tensor that was
made on another stream has to be ordered with `stream` by the caller, as for
any torch call. The operators serve and record no gradients: where autograd is
on, floating-point inputs that require gradients are refused (use
torch.no_grad, or detach them).
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
    """The address of a contiguous tensor of whole numbers (its rows may lie apart when dims is 2)."""
    if t.dtype is dtype and t.device == device and t.dim() == dims and (t.is_contiguous() or t.stride(-1) == 1):
        return t.data_ptr()
    if t.dtype != dtype or t.dim() != dims or t.device != device:
        raise _bad(f"{name} must be a {dims}-d {dtype} tensor on {device}, got {t.dim()}-d {t.dtype} on {t.device}")
    raise _bad(f"{name} is not contiguous")


# The current stream's handle without a Stream object around it.
_current = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _stream(stream, index):
    return _current(index) if stream is None else stream.cuda_stream


def _new(like, shape, stream, dtype=None):
    """A tensor from torch's allocator, which hands its memory out again only
    to work behind this call on the stream it is used on."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _on_gpu(name, t):
    if t.device.type != "cuda":
        raise _bad(f"{name} must be on a GPU, got {t.device}")
    return t.device


def _lost_gradients():
    """Refuses a call, one of whose inputs requires gradients, where autograd is on: it would lose them without a word."""
    if torch.is_grad_enabled():
        raise BackendError(_lib.TCU_EUNSUP, "the paged operators record no gradients: call them under torch.no_grad(), or with detached tensors")


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
        self.ref = C.byref(self.struct)


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
        self.ref, self.device, self.head_dim = C.byref(self.struct), q_weight.device, q_weight.shape[1]
        self.heads = (q_weight.shape[0], k_weight.shape[0])


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
        words = torch.empty(2 * max_requests + 4 + capacity, dtype=torch.int32, device=self.device)
        self._starts, self._lengths, self.counts, self.positions = words.split([max_requests + 1, max_requests, 3, capacity])
        self.starts, self.lengths = self._starts, self._lengths
        self.slots = torch.empty(capacity, dtype=torch.int64, device=self.device)
        self.index, self._n, self._call = self.device.index, max_requests, lib().tcu_plan_step
        self._outs = tuple(t.data_ptr() for t in (self._starts, self._lengths, self.positions, self.slots, self.counts))

    def build(self, held, fresh, tables, free_pages, stream=None):
        """held, fresh: int32 [requests], positions held and tokens added (held
        may be this plan's lengths: a loop's next step); tables: int32
        [requests, width], updated in place; free_pages: int32. Returns self."""
        d, index = self.device, self.index
        h, f = _whole("held", held, torch.int32, d), _whole("fresh", fresh, torch.int32, d)
        t, p = _whole("tables", tables, torch.int32, d, 2), _whole("free_pages", free_pages, torch.int32, d)
        n, width = tables.shape
        if len(held) != n or len(fresh) != n or n > self.max_requests:
            raise _bad(f"{len(held)} requests held, {len(fresh)} fresh, {n} tables, room for {self.max_requests}")
        if self._n != n:
            self.starts, self.lengths, self._n = self._starts[:n + 1], self._lengths[:n], n
        check(self._call(index, _stream(stream, index), n, h, f, self.page_tokens, t, width, tables.stride(0) if n > 1 else width, p,
                         len(free_pages), self.capacity, *self._outs))
        return self


class Cache:
    """A paged KV cache: k and v [pages, KV heads, positions of a page, head
    size], of one type and with the same strides (any order of the first three
    dimensions, the last one contiguous). The tensors stay the caller's."""

    def __init__(self, k, v):
        self.device = _on_gpu("k", k)
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise _bad("k and v are tensors [pages, KV heads, positions, head size] of one shape, type and device")
        # A dimension of one has no stride to speak of.
        strides, other = ([t.stride(i) if t.shape[i] > 1 else t.shape[3] for i in range(3)] for t in (k, v))
        if strides != other or k.stride(3) != 1 or v.stride(3) != 1:
            raise _bad("k and v need the same strides and a contiguous last dimension")
        self.k, self.v, self.code = k, v, _code("the cache", k)
        self.num_pages, self.kv_heads, self.page_tokens, self.head_dim = k.shape
        self._means = torch.Size((self.num_pages, self.kv_heads, self.head_dim))
        self._scale = 1 / math.sqrt(self.head_dim) if self.head_dim else 0.0
        self.struct = _lib.PagedKV(k.data_ptr(), v.data_ptr(), self.code, self.num_pages, self.page_tokens, self.kv_heads, self.head_dim,
                                   *strides)
        self._ref = C.byref(self.struct)
        self._sized = (None, 0)
        self.index, self._lib = self.device.index, lib()

    def append(self, qkv, heads, positions, slots, rotary=None, norm=None, out=None, stream=None):
        """Norm and rotation of the step's rows and their append
        (tcu_paged_append). qkv: [rows, (heads + 2 KV heads) * head size];
        positions int32 and slots int64 [rows]. Returns the queries
        [rows, heads, head size]; rows that are skipped (slot -1) keep what
        `out` held."""
        d, index, hd = self.device, self.index, self.head_dim
        if qkv.requires_grad or self.k.requires_grad or self.v.requires_grad:
            _lost_gradients()
        width = (heads + 2 * self.kv_heads) * hd
        if qkv.dim() != 2 or qkv.device != d or qkv.shape[1] != width or qkv.stride(1) != 1:
            raise _bad(f"qkv must be rows of ({heads} + 2 * {self.kv_heads}) * {hd} values on {d}, got {tuple(qkv.shape)} on {qkv.device}")
        rows = qkv.shape[0]
        p, s = _whole("positions", positions, torch.int32, d), _whole("slots", slots, torch.int64, d)
        if len(positions) != rows or len(slots) != rows:
            raise _bad(f"{rows} rows, {len(positions)} positions, {len(slots)} slots")
        stride = heads * hd
        if out is None:
            out = _new(qkv, (rows, heads, hd), stream)
        else:
            if out.shape != (rows, heads, hd) or out.dtype != qkv.dtype or out.device != d or out.stride(2) != 1 or (heads > 1 and out.stride(1) != hd):
                raise _bad(f"out must be [{rows}, {heads}, {hd}] of {qkv.dtype} on {d}, its heads contiguous")
            stride = out.stride(0) if rows > 1 else stride
        rot = nrm = None
        if rotary is not None:
            if rotary.table.device != d:
                raise _bad("the rotary table is on another device")
            if rotary.table.requires_grad:
                _lost_gradients()
            rot = rotary.ref
        if norm is not None:
            if norm.device != d or norm.head_dim != hd:
                raise _bad(f"norm weights of head size {norm.head_dim} on {norm.device}, the cache has {hd} on {d}")
            if not norm.shared and norm.heads != (heads, self.kv_heads):
                raise _bad("norm weights per head must be [heads, head size] and [KV heads, head size]")
            if norm.q_weight.requires_grad or norm.k_weight.requires_grad:
                _lost_gradients()
            nrm = norm.ref
        check(self._lib.tcu_paged_append(index, _stream(stream, index), self._ref, _code("qkv", qkv), rows, heads, qkv.data_ptr(),
                                         qkv.stride(0) if rows > 1 else width, p, s, rot, nrm, out.data_ptr(), stride))
        return out

    def page_means(self, slots, means, stream=None):
        """Mean keys of the pages that the step's slots complete
        (tcu_paged_means), into means [pages, KV heads, head size] of the
        cache's type. Returns means."""
        if means.requires_grad or self.k.requires_grad:
            _lost_gradients()
        self._check_means(means)
        s = _whole("slots", slots, torch.int64, self.device)
        check(self._lib.tcu_paged_means(self.index, _stream(stream, self.index), self._ref, len(slots), s, means.data_ptr()))
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
        index = self.index
        out, ref = self._queries(q, tables, starts, lengths, max_fresh, scale, out, stream)
        pages, at = 0, None
        if prefix is not None:
            at, pages = _whole("prefix", prefix, torch.int32, self.device), len(prefix)
        key = ("attend", q.dtype, q.shape, tables.shape, max_fresh, pages, max_length)
        sized = self._sized  # one read: another thread may replace it
        size = sized[1] if sized[0] == key else self._size(key, self._lib.tcu_paged_attend_workspace, ref, pages, max_length)
        work = _new(self.k, size, stream, torch.uint8) if size else None
        check(self._lib.tcu_paged_attend(index, _stream(stream, index), self._ref, ref, at, pages, max_length, work.data_ptr() if size else None, size))
        return out

    def attend_sparse(self, q, means, tables, starts, lengths, max_fresh, top, first=1, last=1, scale=None, out=None, pages=None, stream=None):
        """Attention of each query over its first, last and `top` best pages
        (tcu_paged_attend_sparse); arguments as for attend, means as
        page_means keeps them. Returns (out, pages): pages int32 [rows, KV
        heads, first + last + top], the logical pages read, ascending, -1
        behind them."""
        d, index = self.device, self.index
        if means.requires_grad:
            _lost_gradients()
        self._check_means(means)
        out, ref = self._queries(q, tables, starts, lengths, max_fresh, scale, out, stream)
        if min(first, top) < 0 or last < 1:
            raise _bad(f"first {first} and top {top} must not be negative, last {last} must be at least 1")
        shape = (q.shape[0], self.kv_heads, first + last + top)
        if pages is None:
            pages = _new(tables, shape, stream)
        elif pages.shape != shape or pages.dtype != torch.int32 or pages.device != d or not pages.is_contiguous():
            raise _bad(f"pages must be a contiguous int32 tensor {shape} on {d}")
        key = ("sparse", q.dtype, q.shape, tables.shape, max_fresh, first, last, top)
        sized = self._sized
        size = sized[1] if sized[0] == key else self._size(key, self._lib.tcu_paged_attend_sparse_workspace, ref, first, last, top)
        work = _new(self.k, size, stream, torch.uint8)
        check(self._lib.tcu_paged_attend_sparse(index, _stream(stream, index), self._ref, ref, means.data_ptr(), first, last, top, pages.data_ptr(),
                                                work.data_ptr(), size))
        return out, pages

    def _size(self, key, ask, ref, *counts):
        """Workspace bytes of a call, kept for the next one of the same shape."""
        n = C.c_uint64()
        check(ask(self._ref, ref, *counts, C.byref(n)))
        self._sized = (key, n.value)
        return n.value

    def _check_means(self, means):
        if means.shape != self._means or means.dtype is not self.k.dtype or means.device != self.device or not means.is_contiguous():
            raise _bad(f"means must be a contiguous {self.k.dtype} tensor {tuple(self._means)} on {self.device}")

    def _queries(self, q, tables, starts, lengths, max_fresh, scale, out, stream):
        d, hd = self.device, self.head_dim
        if q.requires_grad or self.k.requires_grad or self.v.requires_grad:
            _lost_gradients()
        if q.dim() != 3 or q.shape[2] != hd or q.device != d or q.stride(2) != 1:
            raise _bad(f"q must be [rows, heads, {hd}] on {d}, its last dimension contiguous, got {tuple(q.shape)} on {q.device}")
        rows, heads, _ = q.shape
        st, le, tb = _whole("starts", starts, torch.int32, d), _whole("lengths", lengths, torch.int32, d), _whole("tables", tables, torch.int32, d, 2)
        n, width = tables.shape
        if len(lengths) != n or len(starts) != n + 1:
            raise _bad(f"{n} tables, {len(lengths)} lengths, {len(starts)} starts")
        if out is None:
            out = _new(q, (rows, heads, hd), stream)
            ots, ohs = heads * hd, hd
        else:
            if out.shape != q.shape or out.dtype != q.dtype or out.device != d or out.stride(2) != 1:
                raise _bad(f"out must be {tuple(q.shape)} of {q.dtype} on {d}, its last dimension contiguous")
            ots, ohs, _ = out.stride()
        qts, qhs, _ = q.stride()
        if rows == 1:  # the stride of a dimension of one means nothing
            qts = ots = heads * hd
        if heads == 1:
            qhs = ohs = hd
        return out, C.byref(_lib.PagedQueries(_code("q", q), n, rows, heads, max_fresh, width, q.data_ptr(), qts, qhs, out.data_ptr(), ots, ohs, st, le, tb,
                                              tables.stride(0) if n > 1 else width, self._scale if scale is None else scale))
