"""Serving over a paged key/value cache.

Requests of any length share the pages of a ``PagedCache``.  ``PageTables`` holds
on the device which pages are whose: a step's new tokens get their pages and slots
from ``page_extend`` and ``page_truncate`` gives pages back, neither with a look
from the host.  ``paged_append`` writes the tokens' keys and values (head norms and
rotation in the same launch), ``paged_attention`` attends from one token a session,
and ``sample`` takes the next tokens.  The reference has none of these: its sessions
own an f32 cache each (attention.rs:6-30) and decode greedily (generation.rs:34-42).

A call's tensors lie on the current CUDA device.  Every call only enqueues work on
``stream`` (default: the current one); the outputs it allocates belong to it.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

from . import _native as N
from .gemv import ShapeError
from .speculative import _code, _empty, _handle, _ints, _on_device, _ptr, _rows, _Torch


@dataclass
class PagedCache:
    """k, v [pages, page_size, kv_heads, head_dim] f32 or bf16: any strides that
    are the same for both and multiples of 16 bytes, the last dimension
    contiguous (heads-first pages are a transposed view)."""

    k: object
    v: object

    def __post_init__(self):
        if _Torch.module is None:
            _Torch.load()
        k, v = self.k, self.v
        if k.dim() != 4 or k.shape[3] % 16 or not 0 < k.shape[3] <= 256:
            raise ShapeError(f"pages: [pages, page_size, kv_heads, head_dim % 16 == 0 <= 256] expected, got "
                             f"{list(k.shape)}")
        self.code = _code(k)
        if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device or v.stride() != k.stride():
            raise ShapeError("pages: k and v of one shape, type, device and stride expected")
        # (the pitch of a dimension of one is never used)
        n, p, h, d = k.shape
        st = k.stride()
        if st[3] != 1:
            raise ShapeError("pages: the last dimension must be contiguous")
        self.pitches = (st[0] if n > 1 else p * h * d, st[1] if p > 1 else h * d, st[2] if h > 1 else d)
        if any(s < d or s * k.element_size() % 16 for s in self.pitches):
            raise ShapeError(f"pages: strides {list(st)} have to be multiples of 16 bytes and hold a head vector")

    @classmethod
    def zeros(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=None, device="cuda") -> "PagedCache":
        import torch
        shape = (pages, page_size, kv_heads, head_dim)
        dtype = torch.bfloat16 if dtype is None else dtype
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    @property
    def shape(self):
        return self.k.shape

    def nbytes(self) -> int:
        return 2 * self.k.numel() * self.k.element_size()


@dataclass
class PageTables:
    """Which pages of a pool are whose: table [batch, max_pages] (any row pitch),
    lengths [batch] (the tokens that each request holds), free [pages] (a stack of
    the pages that nobody holds) and free_count [1], all int32 on the device."""

    table: object
    lengths: object
    free: object
    free_count: object
    page_size: int

    def __post_init__(self):
        if _Torch.module is None:
            _Torch.load()
        t = self.table
        if t.dim() != 2 or t.dtype is not _Torch.i32 or (t.shape[1] > 1 and t.stride(1) != 1):
            raise ShapeError(f"tables: int32 [batch, max_pages], rows contiguous, expected, got {t.dtype} "
                             f"{list(t.shape)}")
        _ints(self.lengths, "lengths", t.shape[0])
        _ints(self.free, "free", self.free.numel())
        _ints(self.free_count, "free_count", 1)
        if self.page_size < 1:
            raise ShapeError(f"tables: pages of {self.page_size} tokens")

    @classmethod
    def empty(cls, batch: int, pages: int, page_size: int, max_pages: int, device="cuda") -> "PageTables":
        """No request holds a token; the pool's first pages go first."""
        import torch
        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.full((batch, max_pages), -1, **i32), torch.zeros(batch, **i32),
                   torch.arange(pages - 1, -1, -1, **i32), torch.full((1,), pages, **i32), page_size)

    @property
    def pitch(self) -> int:
        return _pitch(self.table)


@dataclass
class PageMap:
    """Where a step's new tokens lie, a row each (-1 in rows without one): slots,
    positions, requests [rows]; starts [batch + 1], each request's first row."""

    slots: object
    positions: object
    requests: object
    starts: object


def _pitch(t) -> int:
    """Elements between the rows of a matrix whose rows are contiguous."""
    return t.stride(0) if t.shape[0] > 1 else max(1, t.shape[1])


def page_extend(tables: PageTables, counts, rows: int, padded: bool = False, out: PageMap | None = None,
                stream=None) -> PageMap:
    """Takes pages for counts [batch] new tokens of each request and says where
    they lie: rows in order of request (``padded``: rows / batch of them a request).
    A request that the pool, its table or the rows cannot hold whole keeps its
    length, and its rows are -1."""
    b, width = tables.table.shape
    _ints(counts, "counts", b)
    if rows < 1 or (padded and rows % b):
        raise ShapeError(f"page_extend: {rows} rows of {b} requests")
    if out is not None:
        for t, what, n in ((out.slots, "slots", rows), (out.positions, "positions", rows),
                           (out.requests, "requests", rows), (out.starts, "starts", b + 1)):
            if t is not None or what in ("slots", "positions"):
                _ints(t, what, n)
    _on_device("page_extend", tables.table, tables.lengths, tables.free, tables.free_count, counts,
               *(() if out is None else (out.slots, out.positions, out.requests, out.starts)))
    if out is None:
        out = PageMap(*(_empty(stream, counts, _Torch.i32, n) for n in (rows, rows, rows, b + 1)))
    N.call("fpb_page_extend", tables.table.data_ptr(), tables.pitch, b, width, tables.lengths.data_ptr(),
           counts.data_ptr(), tables.free.data_ptr(), tables.free_count.data_ptr(), tables.free.shape[0],
           tables.page_size, rows, int(padded), out.slots.data_ptr(), out.positions.data_ptr(), _ptr(out.requests),
           _ptr(out.starts), _handle(stream, counts))
    return out


def page_truncate(tables: PageTables, lengths, stream=None) -> None:
    """Cuts the requests to lengths [batch] (negative, or not below the present
    one: as it was; 0: the request is done) and gives their pages back."""
    b, width = tables.table.shape
    _ints(lengths, "lengths", b)
    _on_device("page_truncate", tables.table, tables.lengths, tables.free, tables.free_count, lengths)
    N.call("fpb_page_truncate", tables.table.data_ptr(), tables.pitch, b, width, tables.lengths.data_ptr(),
           lengths.data_ptr(), tables.free.data_ptr(), tables.free_count.data_ptr(), tables.free.shape[0],
           tables.page_size, _handle(stream, lengths))


def paged_append(cache: PagedCache, slots, positions, k, v, q=None, q_gamma=None, k_gamma=None, eps: float = 1e-6,
                 rotary_dim: int = 0, theta: float = 10_000.0, q_out=None, stream=None):
    """Norms (where a gamma is given) and rotates k [rows, kv_heads, head_dim] by
    positions [rows] and writes it and v at slots [rows] (negative: no token; no two
    alike); q [rows, q_heads, head_dim] (any row and head pitch) is normed and rotated
    into q_out (allocated in q's dtype where None), which is returned."""
    _, p, hk, d = cache.shape
    if k.dim() != 3 or k.shape[1:] != (hk, d) or v.shape != k.shape or v.dtype != k.dtype:
        raise ShapeError(f"paged_append: k, v [rows, {hk}, {d}] of one dtype expected, got {list(k.shape)} {k.dtype}, "
                         f"{list(v.shape)} {v.dtype}")
    n = k.shape[0]
    _ints(slots, "slots", n)
    _ints(positions, "positions", n)
    for t, what in ((k, "k"), (v, "v")):
        if hk > 1 and t.stride(1) != d:
            raise ShapeError(f"paged_append: {what}'s heads must be contiguous")
    for g in (q_gamma, k_gamma):
        if g is not None and (g.shape != (d,) or _code(g) != N.FPB_F32 or not g.is_contiguous()):
            raise ShapeError(f"paged_append: gammas [{d}] f32 expected")
    hq, q_pitch, q_head, out_code = 0, 0, 0, N.FPB_F32
    if q is not None:
        if q.dim() != 3 or q.shape[0] != n or q.shape[2] != d or q.dtype != k.dtype:
            raise ShapeError(f"paged_append: q [{n}, q_heads, {d}] of k's dtype expected, got {list(q.shape)} {q.dtype}")
        hq, q_pitch = q.shape[1], _rows(q, "q", n, 1)
        q_head = q.stride(1) if hq > 1 else d
        if q_out is not None and (q_out.shape != (n, hq, d) or not q_out.is_contiguous()):
            raise ShapeError(f"paged_append: q_out [{n}, {hq}, {d}] contiguous expected")
        out_code = _code(q if q_out is None else q_out)
    elif q_out is not None:
        raise ShapeError("paged_append: q_out without q")
    k_code, k_pitch, v_pitch = _code(k), _rows(k, "k", n, 1), _rows(v, "v", n, 1)
    _on_device("paged_append", cache.k, slots, positions, k, v, q, q_gamma, k_gamma, q_out)
    if q is not None and q_out is None:
        q_out = _empty(stream, q, q.dtype, n, hq, d)
    if n:
        N.call("fpb_paged_append", _ptr(q), q_pitch, q_head, k.data_ptr(), k_pitch, v.data_ptr(), v_pitch, k_code,
               _ptr(q_gamma), _ptr(k_gamma), slots.data_ptr(), positions.data_ptr(), n, hq, hk, d, rotary_dim, theta,
               eps, _ptr(q_out), out_code, cache.k.data_ptr(), cache.v.data_ptr(), cache.code, cache.shape[0], p,
               *cache.pitches, _handle(stream, k))
    return q_out


def paged_attention_workspace_bytes(cache: PagedCache, batch: int, q_heads: int) -> int:
    return int(N.lib.fpb_paged_attn_workspace_bytes(batch, q_heads, cache.shape[2], cache.shape[3]))


def paged_attention(q, cache: PagedCache, table, lengths, gate=None, scale: float | None = None, out=None,
                    workspace=None, stream=None):
    """out [batch, q_heads, head_dim] (allocated in the pages' type where None;
    f32 or bf16): each session's attention over its first lengths [batch] tokens,
    those of its row of table [batch, max_pages] (int32, any row pitch), times
    sigmoid(gate) where a gate (f32, q's shape) is given; zeros for a length of 0.
    q [batch, q_heads, head_dim] f32 or bf16, any row and head pitch; scale default
    1 / sqrt(head_dim); ``workspace``: uint8 of ``paged_attention_workspace_bytes``
    (allocated where None), which calls on different streams must not share."""
    pages, p, hk, d = cache.shape
    if q.dim() != 3 or q.shape[2] != d or q.shape[1] % hk or not q.shape[1]:
        raise ShapeError(f"paged_attention: q [batch, a multiple of {hk}, {d}] expected, got {list(q.shape)}")
    b, hq = q.shape[0], q.shape[1]
    if table.dim() != 2 or table.dtype is not _Torch.i32 or table.shape[0] != b or (
            table.shape[1] > 1 and table.stride(1) != 1):
        raise ShapeError(f"paged_attention: table int32 [{b}, max_pages] expected, got {table.dtype} "
                         f"{list(table.shape)}")
    _ints(lengths, "lengths", b)
    q_code, q_pitch, gate_pitch, gate_head = _code(q), _rows(q, "q", b, 1), 0, 0
    if gate is not None:
        if gate.shape != q.shape or gate.dtype is not _Torch.f32:
            raise ShapeError(f"paged_attention: gate f32 {list(q.shape)} expected")
        gate_pitch, gate_head = _rows(gate, "gate", b, 1), gate.stride(1) if hq > 1 else d
    out_code = cache.code if out is None else _code(out)
    if out is not None and (out.shape != q.shape or not out.is_contiguous()):
        raise ShapeError("paged_attention: out of q's shape, contiguous, expected")
    if workspace is not None and (workspace.dtype is not _Torch.u8 or not workspace.is_contiguous()):
        raise ShapeError("paged_attention: workspace contiguous uint8 expected")
    _on_device("paged_attention", cache.k, q, table, lengths, gate, out, workspace)
    if out is None:
        out = _empty(stream, q, cache.k.dtype, b, hq, d)
    if workspace is None:
        workspace = _empty(stream, q, _Torch.u8, N.lib.fpb_paged_attn_workspace_bytes(b, hq, hk, d))
    N.call("fpb_paged_attn", q.data_ptr(), q_code, q_pitch, q.stride(1) if hq > 1 else d, cache.k.data_ptr(),
           cache.v.data_ptr(), cache.code, pages, p, *cache.pitches, table.data_ptr(), _pitch(table), table.shape[1],
           lengths.data_ptr(), _ptr(gate), gate_pitch, gate_head, b, hq, hk, d,
           1.0 / math.sqrt(d) if scale is None else scale, workspace.data_ptr(), workspace.numel(), out.data_ptr(),
           out_code, _handle(stream, q))
    return out


def sample(logits, temperature, noise, top_k=None, top_p=None, min_p=None, logprobs: bool = False, out=None,
           stream=None):
    """The next tokens int32 [batch] (``out``, where given) from logits [batch, vocab]
    f32 or bf16 (non-finite ones count as -inf; a row of them gives -1).  A row's tokens
    are ordered by logit, falling, ties by index; top_k keeps the first ones, top_p the
    shortest part of those whose weights exp((l - max) / temperature) reach p of their
    sum, min_p those of at least min_p of the largest weight; the token is argmax weight /
    noise over what is kept.  noise [batch, vocab] f32: exponential variates.
    temperature (0 or below: greedy), top_p, min_p [batch] f32 and top_k [batch] int32,
    on the device; None for a filter: none (top_k 0, top_p 1 and min_p 0 do nothing).
    With ``logprobs``, (tokens, logprobs [batch] f32): the log of the token's weight
    among what is kept."""
    if _Torch.module is None:
        _Torch.load()
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ShapeError(f"sample: logits [batch, vocab], rows contiguous, expected, got {list(logits.shape)}")
    b, vocab = logits.shape
    code = _code(logits)
    if noise.dtype is not _Torch.f32 or noise.shape != (b, vocab) or (vocab > 1 and noise.stride(1) != 1):
        raise ShapeError(f"sample: noise f32 [{b}, {vocab}] expected")
    for t, what in ((temperature, "temperature"), (top_p, "top_p"), (min_p, "min_p")):
        if (t is not None or what == "temperature") and (t.dtype is not _Torch.f32 or t.shape != (b,) or
                                                         not t.is_contiguous()):
            raise ShapeError(f"sample: {what} f32 [{b}] expected")
    if top_k is not None:
        _ints(top_k, "top_k", b)
    if out is not None:
        _ints(out, "out", b)
    _on_device("sample", logits, temperature, noise, top_k, top_p, min_p, out)
    tokens = _empty(stream, logits, _Torch.i32, b) if out is None else out
    logs = _empty(stream, logits, _Torch.f32, b) if logprobs else None
    N.call("fpb_sample", logits.data_ptr(), code, _pitch(logits), temperature.data_ptr(), _ptr(top_k), _ptr(top_p),
           _ptr(min_p), noise.data_ptr(), _pitch(noise), b, vocab, tokens.data_ptr(), _ptr(logs),
           _handle(stream, logits))
    return (tokens, logs) if logprobs else tokens
