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
from .speculative import _code, _empty, _ints, _Torch

# (a decode step's calls take a few microseconds each: on the current stream a call
# that is right goes by _calls; what that leaves alone is checked and made here, with
# the entry points looked up once and each property read once)
_extend, _truncate, _append = N.lib.fpb_page_extend, N.lib.fpb_page_truncate, N.lib.fpb_paged_append
_attn, _attn_bytes, _sample = N.lib.fpb_paged_attn, N.lib.fpb_paged_attn_workspace_bytes, N.lib.fpb_sample


PAGE_MAX_ROWS = 0x7ffffff0  # of a page map


def _keep(self, **values) -> None:
    """What the entry points take of an object, as they take it."""
    for name, value in values.items():
        object.__setattr__(self, name, value)


@dataclass(frozen=True)
class PagedCache:
    """k, v [pages, page_size, kv_heads, head_dim] f32 or bf16: any strides that
    are the same for both and multiples of 16 bytes, the last dimension
    contiguous (heads-first pages are a transposed view).  Their addresses, shapes and
    strides are read once, here: the tensors are written to, not given other storage."""

    k: object
    v: object

    def __post_init__(self):
        if _Torch.module is None:
            _Torch.load()
        k, v = self.k, self.v
        if k.dim() != 4 or k.shape[3] % 16 or not 0 < k.shape[3] <= 256:
            raise ShapeError(f"pages: [pages, page_size, kv_heads, head_dim % 16 == 0 <= 256] expected, got "
                             f"{list(k.shape)}")
        code = _code(k)
        if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device or v.stride() != k.stride():
            raise ShapeError("pages: k and v of one shape, type, device and stride expected")
        # (the pitch of a dimension of one is never used)
        n, p, h, d = k.shape
        st = k.stride()
        if st[3] != 1:
            raise ShapeError("pages: the last dimension must be contiguous")
        pitches = (st[0] if n > 1 else p * h * d, st[1] if p > 1 else h * d, st[2] if h > 1 else d)
        if any(s < d or s * k.element_size() % 16 for s in pitches):
            raise ShapeError(f"pages: strides {list(st)} have to be multiples of 16 bytes and hold a head vector")
        _keep(self, code=code, device=k.get_device(), dtype=k.dtype, dims=(n, p, h, d),
              address=(k.data_ptr(), v.data_ptr()), layout=(code, n, p, *pitches))

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


@dataclass(frozen=True)
class PageTables:
    """Which pages of a pool are whose: table [batch, max_pages] (any row pitch),
    lengths [batch] (the tokens that each request holds), free [pages] (a stack of
    the pages that nobody holds) and free_count [1], all int32 on the device.  As in
    ``PagedCache``, their addresses and shapes are read once."""

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
        for x in (self.lengths, self.free, self.free_count):
            if x.device != t.device:
                raise ShapeError(f"tables: tensors on {t.device} and {x.device}")
        _keep(self, device=t.get_device(), batch=t.shape[0],
              address=(t.data_ptr(), _pitch(t), t.shape[0], t.shape[1], self.lengths.data_ptr()),
              pool=(self.free.data_ptr(), self.free_count.data_ptr(), self.free.shape[0], self.page_size))

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


def _heads(t, n: int, h: int, d: int):
    """(row pitch, head pitch) of t [n, h, d], d contiguous."""
    row, head, one = t.stride()
    if one != 1 and d != 1:
        raise ShapeError(f"a head vector must be contiguous, got strides {t.stride()}")
    return row if n > 1 else h * d, head if h > 1 else d


def _elsewhere(what: str, device: int, *tensors):
    """The tensors' addresses are what the kernels get, so they lie on the current
    CUDA device: the error that says which does not."""
    for t in tensors:
        if t is not None and t.get_device() != device:
            return ShapeError(f"{what}: tensors on device {device} and on {t.device}")
    return ShapeError(f"{what}: tensors on device {device}, which is not the current CUDA device")


def _done(status: int, name: str) -> None:
    if status:
        N.check(status, name)


def _at(t, device: int):
    """The address of an optional tensor, which has to lie on the device (else -1)."""
    return None if t is None else t.data_ptr() if t.get_device() == device else -1


def page_extend(tables: PageTables, counts, rows: int, padded: bool = False, out: PageMap | None = None,
                stream=None) -> PageMap:
    """Takes pages for counts [batch] new tokens of each request (not the tables' own
    lengths) and says where they lie: rows in order of request (``padded``: rows / batch of them a request).
    A request that the pool, its table or the rows cannot hold whole keeps its
    length, and its rows are -1."""
    if stream is None and _Torch.calls is not None and (out is None or out.slots is not None):
        m = (None, None, None, None) if out is None else (out.slots, out.positions, out.requests, out.starts)
        got = _Torch.calls.page_extend(tables.table, tables.lengths, tables.free, tables.free_count, tables.page_size,
                                       counts, rows, padded, *m)
        if got is not NotImplemented:
            if type(got) is int:
                N.check(got, "fpb_page_extend")
            return PageMap(*got) if out is None else out
    b, device = tables.batch, tables.device
    _ints(counts, "counts", b)
    if not 1 <= rows <= PAGE_MAX_ROWS or (padded and rows % b):
        raise ShapeError(f"page_extend: {rows} rows of {b} requests")
    if device < 0 or device != counts.get_device() or device != _Torch.current_device():
        raise _elsewhere("page_extend", device, counts)
    if out is None:
        # one allocation: three rows of a multiple of four, and the starts
        up = (rows + 3) // 4 * 4
        flat = _empty(stream, counts, _Torch.i32, 3 * up + b + 1)
        if up == rows:
            out = PageMap(*flat.split_with_sizes((rows, rows, rows, b + 1)))
        else:
            parts = flat.split_with_sizes((rows, up - rows, rows, up - rows, rows, up - rows, b + 1))
            out = PageMap(parts[0], parts[2], parts[4], parts[6])
        first = flat.data_ptr()
        at = first, first + 4 * up, first + 8 * up, first + 12 * up
    else:
        given = (out.slots, "slots", rows), (out.positions, "positions", rows), (out.requests, "requests", rows), (
            out.starts, "starts", b + 1)
        for t, what, n in given:
            if t is not None or what in ("slots", "positions"):
                _ints(t, what, n)
        at = [_at(t, device) for t, _, _ in given]
        if -1 in at:
            raise _elsewhere("page_extend", device, out.slots, out.positions, out.requests, out.starts)
    _done(_extend(*tables.address, counts.data_ptr(), *tables.pool, rows, padded, *at,
                  _Torch.raw_stream(device) if stream is None else stream), "fpb_page_extend")
    return out


def page_truncate(tables: PageTables, lengths, stream=None) -> None:
    """Cuts the requests to lengths [batch] (negative, or not below the present
    one: as it was; 0: the request is done; not otherwise among the tables' own) and
    gives their pages back."""
    if stream is None and _Torch.calls is not None:
        got = _Torch.calls.page_truncate(tables.table, tables.lengths, tables.free, tables.free_count, tables.page_size,
                                         lengths)
        if got is not NotImplemented:
            if got is not None:
                N.check(got, "fpb_page_truncate")
            return
    device = tables.device
    _ints(lengths, "lengths", tables.batch)
    if device < 0 or device != lengths.get_device() or device != _Torch.current_device():
        raise _elsewhere("page_truncate", device, lengths)
    _done(_truncate(*tables.address, lengths.data_ptr(), *tables.pool,
                    _Torch.raw_stream(device) if stream is None else stream), "fpb_page_truncate")


def paged_append(cache: PagedCache, slots, positions, k, v, q=None, q_gamma=None, k_gamma=None, eps: float = 1e-6,
                 rotary_dim: int = 0, theta: float = 10_000.0, q_out=None, stream=None):
    """Norms (where a gamma is given) and rotates k [rows, kv_heads, head_dim] by
    positions [rows] and writes it and v at slots [rows] (negative: no token; no two
    alike); q [rows, q_heads, head_dim] (any row and head pitch) is normed and rotated
    into q_out (allocated in q's dtype where None), which is returned."""
    if stream is None and _Torch.calls is not None:
        got = _Torch.calls.paged_append(cache.k, cache.v, slots, positions, k, v, q, q_gamma, k_gamma, eps, rotary_dim,
                                        theta, q_out)
        if got is not NotImplemented:
            if type(got) is int:
                N.check(got, "fpb_paged_append")
            return got
    _, _, hk, d = cache.dims
    device, shape, dtype = cache.device, k.shape, k.dtype
    if len(shape) != 3 or shape[1] != hk or shape[2] != d or v.shape != shape or v.dtype is not dtype:
        raise ShapeError(f"paged_append: k, v [rows, {hk}, {d}] of one dtype expected, got {list(shape)} {dtype}, "
                         f"{list(v.shape)} {v.dtype}")
    n = shape[0]
    code = _code(k)
    _ints(slots, "slots", n)
    _ints(positions, "positions", n)
    k_pitch, k_head = _heads(k, n, hk, d)
    v_pitch, v_head = _heads(v, n, hk, d)
    if k_head != d or v_head != d:
        raise ShapeError("paged_append: the heads of k and v must be contiguous")
    for g in (q_gamma, k_gamma):
        if g is not None and (g.dtype is not _Torch.f32 or g.shape != (d,) or not g.is_contiguous()):
            raise ShapeError(f"paged_append: gammas [{d}] f32 expected")
    hq = q_pitch = q_head = out_code = 0
    if q is not None:
        if q.dim() != 3 or q.shape[0] != n or q.shape[2] != d or q.dtype is not dtype:
            raise ShapeError(f"paged_append: q [{n}, q_heads, {d}] of k's dtype expected, got {list(q.shape)} {q.dtype}")
        hq, out_code = q.shape[1], code
        q_pitch, q_head = _heads(q, n, hq, d)
        if q_out is not None:
            out_code = _code(q_out)
            if q_out.shape != (n, hq, d) or not q_out.is_contiguous():
                raise ShapeError(f"paged_append: q_out [{n}, {hq}, {d}] contiguous expected")
    elif q_out is not None:
        raise ShapeError("paged_append: q_out without q")
    at = [_at(t, device) for t in (q, q_gamma, k_gamma, q_out)]
    if device < 0 or not (device == k.get_device() == v.get_device() == slots.get_device() == positions.get_device() ==
                          _Torch.current_device()) or -1 in at:
        raise _elsewhere("paged_append", device, k, v, slots, positions, q, q_gamma, k_gamma, q_out)
    if q is not None and q_out is None:
        q_out = _empty(stream, q, dtype, n, hq, d)
        at[3] = q_out.data_ptr()
    if n:
        _done(_append(at[0], q_pitch, q_head, k.data_ptr(), k_pitch, v.data_ptr(), v_pitch, code, at[1], at[2],
                      slots.data_ptr(), positions.data_ptr(), n, hq, hk, d, rotary_dim, theta, eps, at[3], out_code,
                      *cache.address, *cache.layout, _Torch.raw_stream(device) if stream is None else stream),
              "fpb_paged_append")
    return q_out


def paged_attention_workspace_bytes(cache: PagedCache, batch: int, q_heads: int) -> int:
    return int(_attn_bytes(batch, q_heads, cache.shape[2], cache.shape[3]))


def paged_attention(q, cache: PagedCache, table, lengths, gate=None, scale: float | None = None, out=None,
                    workspace=None, stream=None):
    """out [batch, q_heads, head_dim] (allocated in the pages' type where None;
    f32 or bf16; q itself or apart from q and the gate): each session's attention over its first lengths [batch] tokens,
    those of its row of table [batch, max_pages] (int32, any row pitch), times
    sigmoid(gate) where a gate (f32, q's shape) is given; zeros for a length of 0.
    Infinities and NaN are as the formula has them.
    q [batch, q_heads, head_dim] f32 or bf16, any row and head pitch; scale default
    1 / sqrt(head_dim); ``workspace``: uint8 of ``paged_attention_workspace_bytes``
    (allocated where None), which calls on different streams must not share."""
    if stream is None and _Torch.calls is not None:
        got = _Torch.calls.paged_attention(q, cache.k, cache.v, table, lengths, gate, scale, out, workspace)
        if got is not NotImplemented:
            if type(got) is int:
                N.check(got, "fpb_paged_attn")
            return got
    _, _, hk, d = cache.dims
    device, shape = cache.device, q.shape
    if len(shape) != 3 or shape[2] != d or shape[1] % hk or not shape[1]:
        raise ShapeError(f"paged_attention: q [batch, a multiple of {hk}, {d}] expected, got {list(shape)}")
    b, hq, _ = shape
    width = table.shape
    if len(width) != 2 or table.dtype is not _Torch.i32 or width[0] != b or (width[1] > 1 and table.stride(1) != 1):
        raise ShapeError(f"paged_attention: table int32 [{b}, max_pages] expected, got {table.dtype} "
                         f"{list(table.shape)}")
    width = width[1]
    _ints(lengths, "lengths", b)
    q_code = _code(q)
    q_pitch, q_head = _heads(q, b, hq, d)
    gate_pitch = gate_head = 0
    if gate is not None:
        if gate.shape != shape or gate.dtype is not _Torch.f32:
            raise ShapeError(f"paged_attention: gate f32 {list(shape)} expected")
        gate_pitch, gate_head = _heads(gate, b, hq, d)
    out_code = cache.code
    if out is not None:
        out_code = _code(out)
        if out.shape != shape or not out.is_contiguous():
            raise ShapeError("paged_attention: out of q's shape, contiguous, expected")
    if workspace is not None and (workspace.dtype is not _Torch.u8 or not workspace.is_contiguous()):
        raise ShapeError("paged_attention: workspace contiguous uint8 expected")
    at = [_at(gate, device), _at(out, device), _at(workspace, device)]
    if device < 0 or not (device == q.get_device() == table.get_device() == lengths.get_device() ==
                          _Torch.current_device()) or -1 in at:
        raise _elsewhere("paged_attention", device, q, table, lengths, gate, out, workspace)
    if workspace is None:
        room = _attn_bytes(b, hq, hk, d)
        workspace = _empty(stream, q, _Torch.u8, room)
        at[2] = workspace.data_ptr()
    else:
        room = workspace.numel()
    if out is None:
        out = _empty(stream, q, cache.dtype, b, hq, d)
        at[1] = out.data_ptr()
    _done(_attn(q.data_ptr(), q_code, q_pitch, q_head, *cache.address, *cache.layout, table.data_ptr(),
                table.stride(0) if b > 1 else max(1, width), width, lengths.data_ptr(), at[0], gate_pitch, gate_head, b,
                hq, hk, d, 1.0 / math.sqrt(d) if scale is None else scale, at[2], room, at[1], out_code,
                _Torch.raw_stream(device) if stream is None else stream), "fpb_paged_attn")
    return out


def sample(logits, temperature, noise, top_k=None, top_p=None, min_p=None, logprobs: bool = False, out=None,
           stream=None):
    """The next tokens int32 [batch] (``out``, where given) from logits [batch, vocab]
    f32 or bf16 (non-finite ones count as -inf; a row of them gives -1).  A row's tokens
    are ordered by logit, falling, ties by index; top_k keeps the first ones, top_p the
    shortest part of those whose weights exp((l - max) / temperature) reach p of their
    sum, min_p those of at least min_p of the largest weight; the token is argmax weight /
    noise over what is kept.  noise [batch, vocab] f32: exponential variates.
    temperature (0 or below: greedy; None: 1), top_p, min_p [batch] f32 and top_k [batch]
    int32, on the device; None for a filter: none (top_k 0, top_p 1 and min_p 0 do nothing).
    With ``logprobs``, (tokens, logprobs [batch] f32): the log of the token's weight
    among what is kept."""
    if _Torch.module is None:
        _Torch.load()
    if stream is None and _Torch.calls is not None:
        got = _Torch.calls.sample(logits, temperature, noise, top_k, top_p, min_p, logprobs, out)
        if got is not NotImplemented:
            if type(got) is int:
                N.check(got, "fpb_sample")
            return got
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ShapeError(f"sample: logits [batch, vocab], rows contiguous, expected, got {list(logits.shape)}")
    b, vocab = shape = logits.shape
    code, f32 = _code(logits), _Torch.f32
    if noise.dtype is not f32 or noise.shape != shape or (vocab > 1 and noise.stride(1) != 1):
        raise ShapeError(f"sample: noise f32 [{b}, {vocab}] expected")
    device = logits.get_device()
    for t, what in ((temperature, "temperature"), (top_p, "top_p"), (min_p, "min_p")):
        if t is not None and (t.dtype is not f32 or t.shape != (b,) or not t.is_contiguous()):
            raise ShapeError(f"sample: {what} f32 [{b}] expected")
    if top_k is not None:
        _ints(top_k, "top_k", b)
    if out is not None:
        _ints(out, "out", b)
    at = [_at(t, device) for t in (temperature, top_k, top_p, min_p, noise, out)]
    if device < 0 or device != _Torch.current_device() or -1 in at:
        raise _elsewhere("sample", device, temperature, top_k, top_p, min_p, noise, out)
    tokens = _empty(stream, logits, _Torch.i32, b) if out is None else out
    logs = _empty(stream, logits, f32, b) if logprobs else None
    _done(_sample(logits.data_ptr(), code, logits.stride(0) if b > 1 else vocab, *at[:5],
                  noise.stride(0) if b > 1 else vocab, b, vocab, tokens.data_ptr(),
                  logs.data_ptr() if logprobs else None, _Torch.raw_stream(device) if stream is None else stream),
          "fpb_sample")
    return (tokens, logs) if logprobs else tokens
