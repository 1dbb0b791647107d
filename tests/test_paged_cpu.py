"""Argument checks of the paged cache's entry points and wrappers (no GPU), and
the oracle's stack against its definition."""
import ctypes as C

import numpy as np
import pytest

import firepit_b200 as F
from firepit_b200 import _native as N
from oracle import paged as R

f = (C.c_float * 8)()  # never read: every call is refused before a launch
i = (C.c_int32 * 8)()
f, i = (C.addressof(x) // 16 * 16 + 16 for x in (f, i))
bad, shape = N.FPB_ERR_INVALID_ARGUMENT, N.FPB_ERR_SHAPE


def test_page_entry_points_check_arguments():
    def extend(table=i, pitch=4, batch=2, width=4, lengths=i, counts=i, free=i, free_count=i, pages=8, p=16, rows=4,
               padded=0, slots=i, positions=i):
        return N.lib.fpb_page_extend(table, pitch, batch, width, lengths, counts, free, free_count, pages, p, rows, padded,
                                     slots, positions, None, None, None)

    for name in ("table", "lengths", "counts", "free", "free_count", "slots", "positions"):
        assert extend(**{name: None}) == bad, name
    for kw in (dict(batch=0), dict(batch=16385), dict(width=0), dict(pitch=3), dict(pages=0), dict(p=0), dict(rows=0),
               dict(rows=3, padded=1), dict(pages=1 << 28), dict(width=1 << 28, pitch=1 << 28), dict(rows=1 << 31),
               dict(pitch=1 << 40)):
        assert extend(**kw) == shape, kw

    for counts in (i, i + 4, i - 4):  # two requests' counts among their lengths
        assert extend(counts=counts) == bad

    def cut(table=i, lengths=i, to=i, free=i, free_count=i, batch=2, pages=8):
        return N.lib.fpb_page_truncate(table, 4, batch, 4, lengths, to, free, free_count, pages, 16, None)

    for name in ("table", "lengths", "to", "free", "free_count"):
        assert cut(**{name: None}) == bad, name
    assert cut(batch=0) == shape and cut(pages=0) == shape


def test_page_maps_of_too_many_rows_are_refused_before_memory_is_asked_for():
    torch = pytest.importorskip("torch")
    tables = F.PageTables.empty(3, 6, 16, 4, device="cpu")
    for rows in (0x7ffffff1, 1 << 40, 1 << 62):
        with pytest.raises(F.ShapeError, match="rows"):
            F.page_extend(tables, torch.zeros(3, dtype=torch.int32), rows)


def test_page_truncate_takes_no_lengths_among_the_lengths():
    """New lengths that are read again behind the writes of others' lengths."""
    def cut(lengths, to):
        return N.lib.fpb_page_truncate(i, 4, 2, 4, lengths, to, i, i, 8, 16, None)

    assert cut(i, i + 4) == bad and cut(i + 4, i) == bad


def test_paged_append_checks_arguments():
    def append(q=f, q_pitch=64, q_head=32, k=f, k_pitch=64, v=f, v_pitch=64, dtype=0, qg=f, kg=f, slots=i, pos=i, rows=2,
               hq=2, hk=2, d=32, rot=32, theta=1e4, eps=1e-6, q_out=f, q_out_dtype=0, kp=f, vp=f, page_dtype=1, pages=4,
               p=16, page_pitch=1024, row_pitch=64, head_pitch=32):
        return N.lib.fpb_paged_append(q, q_pitch, q_head, k, k_pitch, v, v_pitch, dtype, qg, kg, slots, pos, rows, hq, hk,
                                      d, rot, theta, eps, q_out, q_out_dtype, kp, vp, page_dtype, pages, p, page_pitch,
                                      row_pitch, head_pitch, None)

    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(pos=None), dict(q=None), dict(q_out=None), dict(hq=0),
               dict(kp=None), dict(vp=None), dict(dtype=2), dict(page_dtype=2), dict(q_out_dtype=5), dict(kp=f + 8),
               dict(vp=f + 2), dict(q=f + 1), dict(k=f + 2), dict(q_out=f + 8), dict(qg=f + 4), dict(kg=f + 4),
               dict(row_pitch=68), dict(head_pitch=33), dict(page_pitch=1028)):
        assert append(**kw) == bad, kw
    for kw in (dict(rows=0), dict(rows=1 << 31), dict(hq=65536), dict(hk=0), dict(hk=4097), dict(d=24), dict(d=272), dict(d=0),
               dict(rot=3), dict(rot=34), dict(theta=0.5), dict(theta=float("nan")), dict(k_pitch=63), dict(v_pitch=63),
               dict(q_head=31), dict(pages=0), dict(p=0), dict(pages=1 << 28), dict(row_pitch=16), dict(head_pitch=16),
               dict(page_pitch=16), dict(page_pitch=1 << 40)):
        assert append(**kw) == shape, kw


def test_paged_attention_checks_arguments():
    def attn(q=f, q_dtype=0, q_pitch=64, q_head=32, kp=f, vp=f, page_dtype=1, pages=4, p=16, page_pitch=1024, row_pitch=64,
             head_pitch=32, table=i, table_pitch=4, width=4, lengths=i, gate=None, gate_pitch=64, gate_head=32, batch=2, hq=2,
             hk=2, d=32, scale=0.1, ws=f, ws_bytes=1 << 30, out=f, out_dtype=1):
        return N.lib.fpb_paged_attn(q, q_dtype, q_pitch, q_head, kp, vp, page_dtype, pages, p, page_pitch, row_pitch,
                                    head_pitch, table, table_pitch, width, lengths, gate, gate_pitch, gate_head, batch, hq, hk,
                                    d, scale, ws, ws_bytes, out, out_dtype, None)

    for kw in (dict(q=None), dict(kp=None), dict(vp=None), dict(table=None), dict(lengths=None), dict(ws=None), dict(out=None),
               dict(q_dtype=2), dict(page_dtype=2), dict(out_dtype=2), dict(q=f + 1), dict(ws=f + 8), dict(out=f + 8),
               dict(gate=f + 2), dict(kp=f + 8), dict(row_pitch=68)):
        assert attn(**kw) == bad, kw
    for kw in (dict(batch=0), dict(batch=16385), dict(hq=3), dict(hq=0), dict(hq=65536 * 2), dict(hk=0), dict(d=24), dict(d=272),
               dict(width=0), dict(table_pitch=3), dict(width=1 << 28, table_pitch=1 << 28), dict(q_head=31),
               dict(gate=f, gate_head=31), dict(scale=float("nan")), dict(scale=float("inf")), dict(pages=0), dict(p=0)):
        assert attn(**kw) == shape, kw
    assert attn(ws_bytes=0) == N.FPB_ERR_WORKSPACE


def test_paged_attention_checks_where_its_output_lies():
    """Over the gate, which blocks read behind one another's outputs, or over other rows'
    queries: refused."""
    buf = (C.c_float * 4096)()
    p = C.addressof(buf) // 16 * 16 + 16

    def attn(q, out, out_dtype=0, q_pitch=64, q_head=32, gate=None, gate_pitch=64, gate_head=32):
        return N.lib.fpb_paged_attn(q, 0, q_pitch, q_head, f, f, 1, 4, 16, 1024, 64, 32, i, 4, 4, i, gate, gate_pitch,
                                    gate_head, 2, 2, 2, 32, 0.1, f, 1 << 30, out, out_dtype, None)

    for kw in (dict(q=p, out=p, out_dtype=1), dict(q=p, out=p + 16), dict(q=p + 16, out=p), dict(q=p, out=p, q_pitch=128),
               dict(q=p, out=p, q_head=64, q_pitch=128), dict(q=p + 4096, out=p, gate=p),
               dict(q=p + 4096, out=p, gate=p + 508), dict(q=p + 4096, out=p + 256, gate=p, gate_pitch=128, gate_head=64)):
        assert attn(**kw) == bad, kw


def test_sample_checks_arguments():
    def sample(logits=f, dtype=0, pitch=100, t=f, noise=f, noise_pitch=100, batch=2, vocab=100, tokens=i):
        return N.lib.fpb_sample(logits, dtype, pitch, t, None, None, None, noise, noise_pitch, batch, vocab, tokens, None,
                                None)

    for kw in (dict(logits=None), dict(noise=None), dict(tokens=None), dict(dtype=2), dict(logits=f + 2), dict(noise=f + 2),
               dict(logits=f + 1, dtype=1)):
        assert sample(**kw) == bad, kw
    for kw in (dict(batch=0), dict(batch=65536), dict(vocab=0), dict(pitch=99), dict(noise_pitch=99),
               dict(vocab=393217, pitch=393217, noise_pitch=393217), dict(pitch=1 << 40)):
        assert sample(**kw) == shape, kw


def test_paged_wrappers_check_tensors():
    torch = pytest.importorskip("torch")
    cache = F.PagedCache.zeros(6, 16, 2, 64, device="cpu")
    assert cache.nbytes() == 2 * 6 * 16 * 2 * 64 * 2
    tables = F.PageTables.empty(3, 6, 16, 4, device="cpu")
    i32 = dict(dtype=torch.int32)
    n3, rows = torch.zeros(3, **i32), torch.zeros(5, **i32)
    kv, q = torch.zeros(5, 2, 64), torch.zeros(5, 4, 64)
    q3 = torch.zeros(3, 4, 64)
    logits, noise = torch.zeros(3, 10), torch.ones(3, 10)
    calls = [
        lambda: F.PagedCache(cache.k[..., :40], cache.v[..., :40]),
        lambda: F.PagedCache(cache.k, cache.v[:, :, :1]),
        lambda: F.PagedCache(cache.k.half(), cache.v.half()),
        lambda: F.PagedCache(cache.k, cache.v.float()),
        lambda: F.PagedCache(cache.k, cache.v.transpose(1, 2).contiguous().transpose(1, 2)),
        lambda: F.PagedCache(cache.k[:1].expand(6, 16, 2, 64), cache.v[:1].expand(6, 16, 2, 64)),
        lambda: F.PagedCache(cache.k.transpose(2, 3), cache.v.transpose(2, 3)),
        lambda: F.PagedCache(torch.zeros(2, 16, 2, 36)[..., :32], torch.zeros(2, 16, 2, 36)[..., :32].bfloat16()),
        lambda: F.PageTables(tables.table.long(), tables.lengths, tables.free, tables.free_count, 16),
        lambda: F.PageTables(tables.table, tables.lengths[:2], tables.free, tables.free_count, 16),
        lambda: F.PageTables(tables.table, tables.lengths, tables.free, tables.free_count, 0),
        lambda: F.PageTables(tables.table.t(), tables.lengths, tables.free, tables.free_count, 16),
        lambda: F.page_extend(tables, n3[:2], 5),
        lambda: F.page_extend(tables, n3.long(), 5),
        lambda: F.page_extend(tables, n3, 0),
        lambda: F.page_extend(tables, n3, 5, padded=True),
        lambda: F.page_extend(tables, n3, 5, out=F.PageMap(rows, rows[:4], None, None)),
        lambda: F.page_truncate(tables, n3.float()),
        lambda: F.paged_append(cache, rows, rows, kv[:, :1], kv[:, :1]),
        lambda: F.paged_append(cache, rows, rows, kv, kv.bfloat16()),
        lambda: F.paged_append(cache, rows.long(), rows, kv, kv),
        lambda: F.paged_append(cache, rows, rows[:4], kv, kv),
        lambda: F.paged_append(cache, rows, rows, kv, kv, q=q.bfloat16()),
        lambda: F.paged_append(cache, rows, rows, kv, kv, q_out=q),
        lambda: F.paged_append(cache, rows, rows, kv, kv, q=q, q_gamma=torch.zeros(32)),
        lambda: F.paged_append(cache, rows, rows, kv, kv, q=q, q_out=q[:, :2]),
        lambda: F.paged_append(cache, rows, rows, kv.half(), kv.half()),
        lambda: F.paged_append(cache, rows, rows, torch.zeros(5, 2, 128)[..., ::2], kv),
        lambda: F.paged_attention(q3[:, :3], cache, tables.table, n3),
        lambda: F.paged_attention(q3[..., :32], cache, tables.table, n3),
        lambda: F.paged_attention(q3.half(), cache, tables.table, n3),
        lambda: F.paged_attention(q3, cache, tables.table[:2], n3),
        lambda: F.paged_attention(q3, cache, tables.table.long(), n3),
        lambda: F.paged_attention(q3, cache, tables.table, n3[:2]),
        lambda: F.paged_attention(q3, cache, tables.table, n3, gate=q3.bfloat16()),
        lambda: F.paged_attention(q3, cache, tables.table, n3, out=q3.half()),
        lambda: F.paged_attention(q3, cache, tables.table, n3, workspace=q3),
        lambda: F.sample(logits[0], n3.float(), noise),
        lambda: F.sample(logits.half(), n3.float(), noise),
        lambda: F.sample(logits, n3, noise),
        lambda: F.sample(logits, n3.float(), noise[:, :9]),
        lambda: F.sample(logits, n3.float(), noise.bfloat16()),
        lambda: F.sample(logits, n3.float(), noise, top_k=n3.float()),
        lambda: F.sample(logits, n3.float(), noise, top_p=n3),
        lambda: F.sample(logits, n3.float(), noise, min_p=n3.float()[:2]),
        lambda: F.sample(logits, n3.float(), noise, out=n3.long()),
        lambda: F.sample(logits.t(), torch.zeros(10), noise.t()),
    ]
    for at, call in enumerate(calls):
        with pytest.raises(F.ShapeError):
            call()
            pytest.fail(f"call {at} was taken")


def test_paged_wrappers_check_devices():
    """Tensors that are right in every other way, but not on a CUDA device: no
    address of theirs reaches a kernel."""
    torch = pytest.importorskip("torch")
    cache = F.PagedCache.zeros(6, 16, 2, 64, device="cpu")
    tables = F.PageTables.empty(3, 6, 16, 4, device="cpu")
    i32 = dict(dtype=torch.int32)
    n3, kv, q = torch.zeros(3, **i32), torch.zeros(3, 2, 64), torch.zeros(3, 4, 64)
    out = F.PageMap(torch.zeros(3, **i32), torch.zeros(3, **i32), torch.zeros(3, **i32), torch.zeros(4, **i32))
    for call in (lambda: F.page_extend(tables, n3, 3), lambda: F.page_extend(tables, n3, 3, True, out),
                 lambda: F.page_truncate(tables, n3), lambda: F.paged_append(cache, n3, n3, kv, kv, q=q),
                 lambda: F.paged_attention(q, cache, tables.table, n3, gate=q),
                 lambda: F.sample(torch.zeros(3, 10), torch.zeros(3), torch.ones(3, 10))):
        with pytest.raises(F.ShapeError, match="device"):
            call()


def test_oracle_pool_and_filters():
    pool = R.Pool(3, 10, 4, 4)
    slots, pos, req, starts = pool.extend([5, 0, 9], 20)
    assert slots[:14].tolist() == [0, 1, 2, 3, 4, 8, 9, 10, 11, 12, 13, 14, 15, 16] and (slots[14:] == -1).all()
    assert pos[:6].tolist() == [0, 1, 2, 3, 4, 0] and req[4:6].tolist() == [0, 2] and starts.tolist() == [0, 5, 5, 14]
    free = list(pool.free)
    pool.extend([4, 4, 4], 20)
    pool.truncate([5, 0, 9])
    assert pool.free == free and pool.lengths.tolist() == [5, 0, 9]
    assert pool.extend([0, 17, 1], 30)[0].tolist()[17] != -1 and pool.lengths.tolist() == [5, 0, 10]  # 17 > 4 pages
    x = np.array([1.0, 3.0, 3.0, -np.inf, 2.0])
    assert R.kept(x, top_k=2)[0].tolist() == [1, 2] and R.kept(x, top_k=1)[0].tolist() == [1]
    assert R.kept(x, temperature=0.0)[0].tolist() == [1] and R.kept(x)[0].tolist() == [1, 2, 4, 0]
    assert R.kept(x, top_p=0.5)[0].tolist() == [1, 2] and R.kept(x, top_p=0.0)[0].tolist() == [1]
    assert R.kept(x, min_p=0.3)[0].tolist() == [1, 2, 4] and R.kept(x, min_p=5.0)[0].tolist() == [1, 2]
    assert R.sample(np.full(3, -np.inf), np.ones(3))[0] == -1
