"""Speculative decoding over an 8-bit key/value cache.

``Kv8Cache`` holds keys and values as e4m3 codes with one exponent byte a head
vector.  A step appends a tree of drafted tokens (``kv8_append``: head norms,
rotation, quantisation in one launch), attends over the cache
(``tree_attention``), verifies the drafts against the target's logits
(``tree_verify``) and moves the accepted path's rows together (``kv8_keep``).
A single token is a tree of one node; a prompt is a chain (``parents=None``).
The reference has none of these: its cache is f32 (attention.rs:6-30) and its
greedy decode takes one token a step (generation.rs:34-42).

A tree is ``parents`` [batch, nodes] int32: -1 for node 0, an earlier node for
the others, -2 for a node that is not there.  A call's tensors lie on the current
CUDA device.  Every call only enqueues work on ``stream`` (default: the current
one); the outputs it allocates belong to it.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

from . import _native as N
from .gemv import ShapeError

TREE_MAX_NODES = 64


class _Torch:
    """torch and what the calls need of it, looked up once (a decode step's
    calls take a few microseconds each)."""

    module = None

    @classmethod
    def load(cls):
        import torch
        cls.f32, cls.bf16, cls.i32, cls.u8 = torch.float32, torch.bfloat16, torch.int32, torch.uint8
        cls.codes = {torch.float32: N.FPB_F32, torch.bfloat16: N.FPB_BF16}
        cls.raw_stream = staticmethod(torch._C._cuda_getCurrentRawStream) if hasattr(
            torch._C, "_cuda_getCurrentRawStream") else staticmethod(
                lambda index: torch.cuda.current_stream(index).cuda_stream)
        cls.current_device = staticmethod(getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device))
        cls.module = torch


def _empty(stream, like, dtype, *shape):
    """Memory of the stream that will write it: torch hands memory out in the
    order of the stream it was asked for on."""
    if stream is None:
        return like.new_empty(*shape, dtype=dtype)
    torch = _Torch.module
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=like.device)):
        return like.new_empty(*shape, dtype=dtype)


def _handle(stream, like) -> int:
    return _Torch.raw_stream(like.get_device()) if stream is None else stream


def _on_device(what: str, like, *tensors) -> None:
    """A call's tensors lie on the current CUDA device: their addresses are what
    the kernels get."""
    device = like.get_device()
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise ShapeError(f"{what}: tensors on {like.device} and {t.device}")
    if device < 0 or device != _Torch.current_device():
        raise ShapeError(f"{what}: tensors on {like.device}, which is not the current CUDA device")


def _code(t) -> int:
    code = _Torch.codes.get(t.dtype)
    if code is None:
        raise ShapeError(f"expected float32 or bfloat16, got {t.dtype}")
    return code


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t, what: str, batch: int, nodes: int) -> int:
    """Elements between rows of [batch, nodes, ...]: one pitch over both, the
    trailing dimension contiguous."""
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] != 1:
        raise ShapeError(f"{what}: the last dimension must be contiguous")
    if nodes == 1:
        return st[0] if batch > 1 else t.shape[-1] * t.shape[-2]
    if batch > 1 and st[0] != nodes * st[1]:
        raise ShapeError(f"{what}: sessions must follow one another at nodes * row pitch")
    return st[1]


def _ints(t, what: str, *shape):
    if t.dtype is not _Torch.i32 or t.shape != shape or not t.is_contiguous():
        raise ShapeError(f"{what}: contiguous int32 {list(shape)} expected, got {t.dtype} {list(t.shape)}")


def _parents(parents, batch: int, nodes: int):
    if parents is not None:
        _ints(parents, "parents", batch, nodes)
        if nodes > TREE_MAX_NODES:
            raise ShapeError(f"a tree has at most {TREE_MAX_NODES} nodes, got {nodes}")


@dataclass
class Kv8Cache:
    """k, v [batch, max_seq, kv_heads, head_dim] uint8 (e4m3 codes); k_exp,
    v_exp [batch, max_seq, kv_heads] uint8: value = code * 2^(byte - 127)."""

    k: object
    v: object
    k_exp: object
    v_exp: object

    def __post_init__(self):
        if _Torch.module is None:
            _Torch.load()
        k = self.k
        if k.dim() != 4 or k.shape[3] % 16 or not 0 < k.shape[3] <= 256:
            raise ShapeError(f"cache: [batch, max_seq, kv_heads, head_dim % 16 == 0 <= 256] expected, got "
                             f"{list(k.shape)}")
        u8, full = _Torch.u8, k.shape
        for t, shape in ((k, full), (self.v, full), (self.k_exp, full[:3]), (self.v_exp, full[:3])):
            if t.dtype is not u8 or t.shape != shape or not t.is_contiguous() or t.device != k.device:
                raise ShapeError("cache: contiguous uint8 codes of one shape and exponents [batch, max_seq, kv_heads] "
                                 "on one device expected")

    @classmethod
    def zeros(cls, batch: int, max_seq: int, kv_heads: int, head_dim: int, device="cuda") -> "Kv8Cache":
        import torch
        u8 = dict(dtype=torch.uint8, device=device)
        return cls(torch.zeros(batch, max_seq, kv_heads, head_dim, **u8),
                   torch.zeros(batch, max_seq, kv_heads, head_dim, **u8),
                   torch.full((batch, max_seq, kv_heads), 119, **u8), torch.full((batch, max_seq, kv_heads), 119, **u8))

    @property
    def shape(self):
        return self.k.shape

    def nbytes(self) -> int:
        return 2 * (self.k.numel() + self.k_exp.numel())

    def zero_(self) -> None:
        for t, fill in ((self.k, 0), (self.v, 0), (self.k_exp, 119), (self.v_exp, 119)):
            t.fill_(fill)


def kv8_append(cache: Kv8Cache, positions, k, v, q=None, parents=None, q_gamma=None, k_gamma=None, eps: float = 1e-6,
               rotary_dim: int = 0, theta: float = 10_000.0, q_out=None, stream=None):
    """Norms (where a gamma is given), rotates and quantises k, v [batch, nodes,
    kv_heads, head_dim] into rows position + node of the cache; q [batch, nodes,
    q_heads, head_dim] (any row and head pitch) is normed and rotated into
    q_out (allocated in q's dtype where None), which is returned."""
    b, s, hk, d = cache.shape
    if k.dim() != 4 or k.shape[0] != b or k.shape[2:] != (hk, d) or v.shape != k.shape or v.dtype != k.dtype:
        raise ShapeError(f"kv8_append: k, v [{b}, nodes, {hk}, {d}] of one dtype expected, got {list(k.shape)} "
                         f"{k.dtype}, {list(v.shape)} {v.dtype}")
    n = k.shape[1]
    _parents(parents, b, n)
    _ints(positions, "positions", b)
    for t, what in ((k, "k"), (v, "v")):
        if hk > 1 and t.stride(2) != d:
            raise ShapeError(f"kv8_append: {what}'s heads must be contiguous")
    for g in (q_gamma, k_gamma):
        if g is not None and (g.shape != (d,) or _code(g) != N.FPB_F32 or not g.is_contiguous()):
            raise ShapeError(f"kv8_append: gammas [{d}] f32 expected")
    hq, q_pitch, q_head, out_code = 0, 0, 0, N.FPB_F32
    if q is not None:
        if q.dim() != 4 or q.shape[:2] != (b, n) or q.shape[3] != d or q.dtype != k.dtype:
            raise ShapeError(f"kv8_append: q [{b}, {n}, q_heads, {d}] of k's dtype expected, got {list(q.shape)} "
                             f"{q.dtype}")
        hq, q_pitch = q.shape[2], _rows(q, "q", b, n)
        q_head = q.stride(2) if hq > 1 else d
        if q_out is not None and (q_out.shape != (b, n, hq, d) or not q_out.is_contiguous()):
            raise ShapeError(f"kv8_append: q_out [{b}, {n}, {hq}, {d}] contiguous expected")
        out_code = _code(q if q_out is None else q_out)
    elif q_out is not None:
        raise ShapeError("kv8_append: q_out without q")
    _on_device("kv8_append", cache.k, positions, k, v, q, parents, q_gamma, k_gamma, q_out)
    if q is not None and q_out is None:
        q_out = _empty(stream, q, q.dtype, b, n, hq, d)
    N.call("fpb_kv8_append", _ptr(q), q_pitch, q_head, k.data_ptr(), _rows(k, "k", b, n), v.data_ptr(),
           _rows(v, "v", b, n), _code(k), _ptr(q_gamma), _ptr(k_gamma), positions.data_ptr(), _ptr(parents), b, n, hq,
           hk, d, rotary_dim, theta, eps, s, _ptr(q_out), out_code, cache.k.data_ptr(), cache.v.data_ptr(),
           cache.k_exp.data_ptr(), cache.v_exp.data_ptr(), _handle(stream, k))
    return q_out


def kv8_read(cache: Kv8Cache, begin, count: int, dtype=None, stream=None):
    """(k, v) [batch, count, kv_heads, head_dim] as the values that rows
    [begin, begin + count) stand for; begin: an int, or int32 [batch]."""
    b, s, hk, d = cache.shape
    dtype = _Torch.f32 if dtype is None else dtype
    begins = where = None
    if not isinstance(begin, int):
        _ints(begin, "begin", b)
        where, begins, begin = begin, begin.data_ptr(), 0
    if count < 1 or begin < 0:
        raise ShapeError(f"kv8_read: rows [{begin}, +{count})")
    _on_device("kv8_read", cache.k, where)
    k, v = _empty(stream, cache.k, dtype, b, count, hk, d), _empty(stream, cache.k, dtype, b, count, hk, d)
    N.call("fpb_kv8_read", cache.k.data_ptr(), cache.v.data_ptr(), cache.k_exp.data_ptr(), cache.v_exp.data_ptr(), b,
           s, hk, d, begins, begin, count, k.data_ptr(), v.data_ptr(), _code(k), _handle(stream, cache.k))
    return k, v


def kv8_keep(cache: Kv8Cache, positions, path, stream=None) -> None:
    """Row position + d becomes row position + path[d] of each session: path
    [batch, nodes] ascending, -1 after its end (``tree_verify``'s)."""
    b, s, hk, d = cache.shape
    _ints(positions, "positions", b)
    _ints(path, "path", b, path.shape[-1])
    _on_device("kv8_keep", cache.k, positions, path)
    N.call("fpb_kv8_keep", cache.k.data_ptr(), cache.v.data_ptr(), cache.k_exp.data_ptr(), cache.v_exp.data_ptr(), b, s,
           hk, d, positions.data_ptr(), path.data_ptr(), path.shape[1], _handle(stream, cache.k))


def tree_attention_workspace_bytes(cache: Kv8Cache, nodes: int, q_heads: int) -> int:
    b, s, hk, d = cache.shape
    return int(N.lib.fpb_tree_attn_workspace_bytes(b, nodes, q_heads, hk, d, s))


def tree_attention(q, cache: Kv8Cache, positions, parents=None, gate=None, scale: float | None = None, out=None,
                   workspace=None, stream=None):
    """out [batch, nodes, q_heads, head_dim] bf16: each node's attention over
    the rows before its session's position, its ancestors and itself (already
    appended), times sigmoid(gate) where a gate (f32, q's shape) is given.
    q f32 or bf16, any row and head pitch, rounded to f16 for the products (each
    row scaled by a power of two), as the weights are; scale default 1 /
    sqrt(head_dim);
    ``workspace``: uint8 of ``tree_attention_workspace_bytes`` (allocated where
    None)."""
    b, s, hk, d = cache.shape
    if q.dim() != 4 or q.shape[0] != b or q.shape[3] != d or q.shape[2] % hk:
        raise ShapeError(f"tree_attention: q [{b}, nodes, a multiple of {hk}, {d}] expected, got {list(q.shape)}")
    n, hq = q.shape[1], q.shape[2]
    _parents(parents, b, n)
    _ints(positions, "positions", b)
    gate_pitch = gate_head = 0
    if gate is not None:
        if gate.shape != q.shape or gate.dtype is not _Torch.f32:
            raise ShapeError(f"tree_attention: gate f32 {list(q.shape)} expected")
        gate_pitch, gate_head = _rows(gate, "gate", b, n), gate.stride(2) if hq > 1 else d
    if out is not None and (out.shape != q.shape or out.dtype is not _Torch.bf16 or not out.is_contiguous()):
        raise ShapeError("tree_attention: out bf16 of q's shape, contiguous, expected")
    if workspace is not None and (workspace.dtype is not _Torch.u8 or not workspace.is_contiguous()):
        raise ShapeError("tree_attention: workspace contiguous uint8 expected")
    _on_device("tree_attention", cache.k, q, positions, parents, gate, out, workspace)
    if out is None:
        out = _empty(stream, q, _Torch.bf16, b, n, hq, d)
    if workspace is None:
        workspace = _empty(stream, q, _Torch.u8, N.lib.fpb_tree_attn_workspace_bytes(b, n, hq, hk, d, s))
    N.call("fpb_tree_attn", q.data_ptr(), _code(q), _rows(q, "q", b, n), q.stride(2) if hq > 1 else d,
           cache.k.data_ptr(), cache.v.data_ptr(), cache.k_exp.data_ptr(), cache.v_exp.data_ptr(), positions.data_ptr(),
           _ptr(parents), _ptr(gate), gate_pitch, gate_head, b, n, hq, hk, d, s,
           1.0 / math.sqrt(d) if scale is None else scale, workspace.data_ptr(), workspace.numel(), out.data_ptr(),
           _handle(stream, q))
    return out


def tree_verify(logits, tokens, parents=None, temperature: float = 0.0, accept=None, noise=None, draft=None,
                stream=None):
    """(path, count, next): the drafted tokens [batch, nodes] that the target
    accepts, walking down from node 0, and the token after them.  logits [batch,
    nodes, vocab] f32 or bf16; temperature 0 takes the target's argmax; above
    it, accept [batch, nodes] uniform and noise [batch, vocab] exponential
    variates decide, and draft [batch, nodes, vocab] f32 (None: certain drafts)
    holds the probabilities that each node's children were drawn from.  Emitted
    tokens are then distributed as the target's."""
    if _Torch.module is None:
        _Torch.load()
    if logits.dim() != 3:
        raise ShapeError(f"tree_verify: logits [batch, nodes, vocab] expected, got {list(logits.shape)}")
    b, n, vocab = logits.shape
    _ints(tokens, "tokens", b, n)
    _parents(parents, b, n)
    if n > TREE_MAX_NODES:
        raise ShapeError(f"a tree has at most {TREE_MAX_NODES} nodes, got {n}")
    noise_pitch = draft_pitch = 0
    if temperature != 0.0:
        if accept is None or noise is None:
            raise ShapeError("tree_verify: a temperature above 0 needs accept and noise")
        if accept.dtype is not _Torch.f32 or accept.shape != (b, n) or not accept.is_contiguous():
            raise ShapeError(f"tree_verify: accept f32 [{b}, {n}] expected")
        if noise.dtype is not _Torch.f32 or noise.shape != (b, vocab) or (vocab > 1 and noise.stride(1) != 1):
            raise ShapeError(f"tree_verify: noise f32 [{b}, {vocab}] expected")
        noise_pitch = noise.stride(0) if b > 1 else vocab
        if draft is not None:
            if draft.dtype is not _Torch.f32 or draft.shape != logits.shape:
                raise ShapeError(f"tree_verify: draft f32 {list(logits.shape)} expected")
            draft_pitch = _pitch(draft, "draft")
    else:
        accept = noise = draft = None
    _on_device("tree_verify", logits, tokens, parents, accept, noise, draft)
    path = _empty(stream, logits, _Torch.i32, b, n)
    count, nxt = _empty(stream, logits, _Torch.i32, b), _empty(stream, logits, _Torch.i32, b)
    N.call("fpb_tree_verify", logits.data_ptr(), _code(logits), _pitch(logits, "logits"), _ptr(draft), draft_pitch,
           tokens.data_ptr(), _ptr(parents), _ptr(accept), _ptr(noise), noise_pitch, b, n, vocab, temperature,
           path.data_ptr(), count.data_ptr(), nxt.data_ptr(), _handle(stream, logits))
    return path, count, nxt


def _pitch(t, what: str) -> int:
    """Elements between the rows of [batch, nodes, vocab]."""
    b, n, vocab = t.shape
    st = t.stride()
    if vocab > 1 and st[2] != 1:
        raise ShapeError(f"{what}: the vocabulary must be contiguous")
    if n == 1:
        return st[0] if b > 1 else vocab
    if b > 1 and st[0] != n * st[1]:
        raise ShapeError(f"{what}: sessions must follow one another at nodes * row pitch")
    return st[1]
