"""Serving over a paged cache: page tables, append, attention of one token and
sampling against the oracle's restatement in 64 bits (oracle/paged.py).

Bars, derived from the arithmetic:
 - page tables: whole numbers, equal.
 - append: as in the 8-bit cache's tests: 3e-6 of the head's largest value for
   norms and rotation in f32, and half a step of the type that it is kept in
   (bf16 2^-8, f32 2^-24); v that fits its type is equal.
 - attention: f32 pages, products and sums in f32: a score is off by at most
   ds = (d + 4) 2^-24 scale * sum |q_i k_i|, so a weight by 2 ds + 2^-21 (its
   power) of itself, the sums over n tokens by (n + 64) 2^-24, and the output by
   (2 ds + 2^-20 + (n + 64) 2^-23) * sum p |v|.  Products of factors in two parts
   of 11 bits stay within that: a product is off by 2^-20 (what the cut factor's two
   parts leave), 2^-21 (the parts' own product, left out) and 2^-22, 1.75 * 2^-20 in
   all, so the output by (3 * 2^-20 of the scores, twice, and 1.75 * 2^-20) * sum p
   |v|, below 8 * 2^-20 where the bar's (64) 2^-23 alone is as much.  bf16 pages: q and the weights are
   split in two parts of 8 bits each (2^-16 with the sign), products exact in
   f32: 2^-16 more in ds and 2^-15 more of sum p |v|.  Then half a step of the
   output's type and 2^-21 for the gate.
 - sampling: a weight's logarithm is off by up to 4 * 2^-24 of |l - max l| / T
   (three roundings), 6e-5 for the distances of up to 256 that matter beside f32's
   smallest weight; the tests' own stay below 80 (2e-5), its power by 2^-21, sums by
   2^-17 of themselves at most: a token is right if it is the oracle's for top_p
   within 3e-5 of the given one, or if its weight / noise is within 6e-5 of the
   winner's there.  logprobs: 4e-5 + 2^-22 of itself.
"""
import math

import numpy as np
import pytest

from oracle import paged as R
from oracle.speculative import norm_rotate

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


@pytest.fixture(scope="module")
def F(torch):
    import firepit_b200
    return firepit_b200


@pytest.fixture(autouse=True)
def _no_device_error(F):
    yield
    assert F.device_error(reset=True) == 0


def _dev(torch, x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


def _host(t):
    return t.float().cpu().numpy().astype(np.float64)


def _type(torch, name):
    return torch.float32 if name == "f32" else torch.bfloat16


# ---- page tables ---------------------------------------------------------------------------------------------------
def _same(tables, pool):
    n = int(tables.free_count.cpu()[0])
    assert n == len(pool.free)
    assert (tables.free.cpu().numpy()[:n] == pool.free).all()
    assert (tables.lengths.cpu().numpy() == pool.lengths).all()
    assert (tables.table.cpu().numpy() == pool.table).all()


def _maps(m, want):
    for got, w in zip((m.slots, m.positions, m.requests, m.starts), want):
        assert (got.cpu().numpy() == w).all()


@pytest.mark.parametrize("batch,pages,p,width,rows,padded", [
    (1, 3, 1, 3, 4, False), (5, 40, 16, 9, 64, False), (7, 30, 3, 11, 35, True), (64, 900, 16, 20, 64, True),
    (1030, 4000, 8, 6, 9001, False), (3, 2000, 24, 700, 30000, False), (300, 60, 4, 5, 800, False), (700, 9000, 1, 30, 9001, False),
    (40, 70000, 2, 2000, 4000, False)])
def test_page_tables_follow_the_stack(F, torch, batch, pages, p, width, rows, padded):
    """Steps of extensions and truncations, among them more than the pool, the
    tables and the rows can hold."""
    rng = np.random.default_rng(batch * 7 + pages)
    tables, pool = F.PageTables.empty(batch, pages, p, width), R.Pool(batch, pages, p, width)
    for step in range(8):
        most = rows // batch if padded else max(1, 2 * rows // batch)
        counts = rng.integers(0, most + 2, batch) if step % 2 else np.minimum(1, rng.integers(0, 3, batch))
        if step == 4:
            counts[:] = 0
        m = F.page_extend(tables, _dev(torch, counts.astype(np.int32)), rows, padded)
        _maps(m, pool.extend(counts, rows, padded))
        _same(tables, pool)
        cut = np.where(rng.random(batch) < 0.5, -1, rng.integers(0, width * p + 1, batch))
        cut[rng.random(batch) < 0.2] = 0
        F.page_truncate(tables, _dev(torch, cut.astype(np.int32)))
        pool.truncate(cut)
        _same(tables, pool)


@pytest.mark.parametrize("batch,pages,p,width,rows", [
    (16384, 40000, 4, 4, 20000), (16384, 16384, 1, 1, 16384), (64, 65536, 2, 1100, 6144), (64, 65537, 2, 1100, 6145),
    (9, 65536, 1, 7300, 20000), (9, 70000, 1, 7281, 20000)])
def test_page_tables_at_the_limits_of_their_ways(F, torch, batch, pages, p, width, rows):
    """The most requests, and pages and rows on both sides of where one block, a cluster
    and many blocks take a step."""
    rng = np.random.default_rng(batch + pages)
    tables, pool = F.PageTables.empty(batch, pages, p, width), R.Pool(batch, pages, p, width)
    for step in range(6):
        counts = rng.integers(0, 2 * rows // batch + 2, batch)
        m = F.page_extend(tables, _dev(torch, counts.astype(np.int32)), rows)
        _maps(m, pool.extend(counts, rows))
        _same(tables, pool)
        if step % 3 == 2:  # everything goes back at once
            cut = np.zeros(batch, np.int64)
        else:
            cut = np.where(rng.random(batch) < 0.7, -1, rng.integers(0, width * p + 1, batch))
        F.page_truncate(tables, _dev(torch, cut.astype(np.int32)))
        pool.truncate(cut)
        _same(tables, pool)
    assert len(pool.free) == pages


def test_page_tables_what_a_step_took_goes_back(F, torch):
    tables = F.PageTables.empty(6, 50, 4, 8)
    F.page_extend(tables, _dev(torch, np.array([3, 9, 0, 4, 5, 1], np.int32)), 22)
    before = [t.clone() for t in (tables.table, tables.lengths, tables.free, tables.free_count)]
    lengths = tables.lengths.clone()
    F.page_extend(tables, _dev(torch, np.array([1, 7, 8, 4, 0, 12], np.int32)), 40)
    F.page_truncate(tables, lengths)
    for t, w in zip((tables.table, tables.lengths, tables.free, tables.free_count), before):
        assert torch.equal(t, w)


def test_page_tables_ranges_of_the_state(F, torch):
    """Lengths, counts and entries that cannot be are recorded, and the requests
    beside them are served."""
    tables = F.PageTables.empty(4, 20, 4, 5)
    tables.lengths.copy_(_dev(torch, np.array([-3, 0, 21, 0], np.int32)))
    m = F.page_extend(tables, _dev(torch, np.array([1, 2, 1, -5], np.int32)), 8)
    assert F.device_error(reset=True) == 507
    assert m.slots.cpu().tolist() == [-1, 0, 1, -1, -1, -1, -1, -1]
    assert tables.lengths.cpu().tolist() == [-3, 2, 21, 0] and int(tables.free_count) == 19
    F.page_truncate(tables, _dev(torch, np.zeros(4, np.int32)))
    assert F.device_error(reset=True) == 507 and tables.lengths.cpu().tolist() == [-3, 0, 21, 0]
    tables = F.PageTables.empty(2, 20, 4, 5)
    tables.free[19] = 20  # the first page that goes
    m = F.page_extend(tables, _dev(torch, np.array([4, 4], np.int32)), 8)
    assert F.device_error(reset=True) == 506
    assert m.slots.cpu().tolist() == [-1] * 4 + [4, 5, 6, 7]
    tables = F.PageTables.empty(2, 20, 4, 5)
    tables.free_count.fill_(21)
    m = F.page_extend(tables, _dev(torch, np.array([4, 0], np.int32)), 8)
    assert F.device_error(reset=True) == 507 and m.slots.cpu().tolist() == [-1] * 8
    tables.free_count.fill_(20)
    tables.lengths.fill_(4)  # pages that nobody took cannot come back
    F.page_truncate(tables, _dev(torch, np.zeros(2, np.int32)))
    assert F.device_error(reset=True) == 507 and tables.lengths.cpu().tolist() == [4, 4]


def test_page_tables_rows_up_to_2_31(F, torch):
    """As many rows as there may be, all but five without a token, into vectors of
    the caller's."""
    tables, rows = F.PageTables.empty(1, 6, 2, 6), 0x7ffffff0
    out = F.PageMap(*(torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(2)), None, None)
    assert F.page_extend(tables, _dev(torch, np.array([5], np.int32)), rows, True, out) is out
    for t, want in ((out.slots, [0, 1, 2, 3, 4]), (out.positions, [0, 1, 2, 3, 4])):
        assert t[:5].tolist() == want and all(bool((x == -1).all()) for x in t[5:].split(1 << 28))
    assert tables.lengths.tolist() == [5] and tables.free_count.tolist() == [3]


def test_page_tables_in_a_graph(F, torch):
    """One captured step, replayed: the state moves on; a pitched table."""
    wide = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
    t = F.PageTables.empty(3, 64, 8, 16)
    tables, pool = F.PageTables(wide[:, 4:20], t.lengths, t.free, t.free_count, 8), R.Pool(3, 64, 8, 16)
    counts = torch.ones(3, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=side):
        m = F.page_extend(tables, counts, 3, True)
    for step in range(20):
        counts[1] = step % 2
        g.replay()
        _maps(m, pool.extend([1, step % 2, 1], 3, True))
    _same(tables, pool)
    assert (wide[:, :4] == -1).all() and (wide[:, 20:] == -1).all()


# ---- append --------------------------------------------------------------------------------------------------------
def _pages(torch, pages, p, hk, d, dtype, layout, fill=None):
    """k and v pages; heads first, or both in one allocation, as views."""
    shape = (pages, p, hk, d)
    if layout == "heads":
        k, v = (torch.zeros(pages, hk, p, d, dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2))
    elif layout == "one":
        both = torch.zeros(pages, 2, p, hk, d, dtype=dtype, device="cuda")
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = (torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(2))
    for t in (k, v):
        t.copy_(torch.randn(shape, device="cuda") if fill is None else torch.full(shape, fill, device="cuda"))
    return k, v


@pytest.mark.parametrize("n,hq,hk,d,rot,p,layout,dtype,pages", [
    (1, 2, 1, 16, 16, 1, "plain", "f32", "bf16"), (8, 16, 2, 256, 64, 16, "heads", "f32", "f32"),
    (37, 6, 3, 80, 20, 24, "one", "bf16", "bf16"), (3000, 4, 4, 64, 64, 7, "plain", "f32", "bf16"),
    (130, 5, 1, 96, 0, 16, "heads", "bf16", "f32"), (11, 3, 3, 240, 238, 32, "one", "f32", "f32")])
def test_paged_append_matches_the_formulas(F, torch, n, hq, hk, d, rot, p, layout, dtype, pages):
    rng = np.random.default_rng(n * 10 + d)
    td, tp = _type(torch, dtype), _type(torch, pages)
    count = n // p + 5
    qg = _dev(torch, rng.standard_normal((n, hq, 2, d)).astype(np.float32) * 3, td)
    kv = _dev(torch, rng.standard_normal((n, 2, hk, d)).astype(np.float32), td)
    q, k, v = qg[:, :, 0], kv[:, 0], kv[:, 1]  # pitched views of wider rows
    qga, kga = (_dev(torch, (1 + 0.1 * rng.standard_normal(d)).astype(np.float32)) for _ in range(2))
    kp, vp = _pages(torch, count, p, hk, d, tp, layout)
    cache = F.PagedCache(kp, vp)
    kb, vb = _host(kp), _host(vp)
    slots = rng.permutation(count * p)[:n].astype(np.int32)
    slots[rng.random(n) < 0.1] = -1
    slots[0] = count * p - 1 if count * p - 1 not in slots else slots[0]
    pos = rng.integers(0, 70000, n).astype(np.int32)
    pos[slots < 0] = -1
    got = F.paged_append(cache, _dev(torch, slots), _dev(torch, pos), k, v, q=q, q_gamma=qga, k_gamma=kga, eps=1e-6,
                         rotary_dim=rot, theta=1e4)
    assert got.dtype == td
    got, ka, va, q, k, v = (_host(x) for x in (got, kp, vp, q, k, v))
    half = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}
    rest = np.ones(count * p, bool)
    for i, s in enumerate(slots):
        if s < 0:
            assert not got[i].any()
            continue
        rest[s] = False
        for h in range(hq):
            w = norm_rotate(q[i, h], qga.cpu().numpy(), 1e-6, int(pos[i]), rot, 1e4)
            assert np.abs(got[i, h] - w).max() <= 3e-6 * np.abs(w).max() + half[dtype] * np.abs(w).max()
        for h in range(hk):
            w = norm_rotate(k[i, h], kga.cpu().numpy(), 1e-6, int(pos[i]), rot, 1e4)
            assert np.abs(ka[s // p, s % p, h] - w).max() <= 3e-6 * np.abs(w).max() + half[pages] * np.abs(w).max()
            want = _host(_dev(torch, v[i, h].astype(np.float32)).to(tp))
            assert (va[s // p, s % p, h] == want).all()
    for a, b in ((ka, kb), (va, vb)):  # rows without a token are as they were
        assert (a.reshape(count * p, hk, d)[rest] == b.reshape(count * p, hk, d)[rest]).all()


def test_paged_append_keeps_out_of_other_rows(F, torch):
    """Slots and positions that cannot be are recorded, and nothing is written for
    them; without gammas and q the values are as they were given."""
    kp, vp = _pages(torch, 3, 4, 2, 32, torch.float32, "plain", 7.0)
    cache = F.PagedCache(kp, vp)
    k = torch.randn(4, 2, 32, device="cuda")
    v = torch.randn(4, 2, 32, device="cuda")
    for slots, pos, code in (([12, 0, -7, 2 ** 31 - 1], [1, 2, 3, 4], 506), ([1, 2, 3, -1], [0, -1, 5, -1], 502)):
        kp.fill_(7.0)
        vp.fill_(7.0)
        assert F.paged_append(cache, _dev(torch, np.array(slots, np.int32)), _dev(torch, np.array(pos, np.int32)), k,
                              v) is None
        assert F.device_error(reset=True) == code
        good = [i for i in range(4) if 0 <= slots[i] < 12 and pos[i] >= 0]
        for pages, x in ((kp, k), (vp, v)):
            flat = pages.view(12, 2, 32)
            for i in good:
                assert torch.equal(flat[slots[i]], x[i])
            others = [s for s in range(12) if s not in [slots[i] for i in good]]
            assert (flat[others] == 7.0).all()


# ---- attention -----------------------------------------------------------------------------------------------------
def _attention_case(F, torch, rng, lengths, hq, hk, d, p, dtype, pages, layout="plain", poison=math.nan, spare=3,
                    table_extra=2):
    """(q, gate, cache, table, lengths): pages in no order; what no session holds,
    and what lies behind its last token, is `poison`."""
    lengths = np.asarray(lengths, np.int32)
    b = len(lengths)
    held = [-(-int(n) // p) for n in lengths]
    count = sum(held) + spare
    order = rng.permutation(count)
    table = np.full((b, max(held) + table_extra), -1, np.int32)
    kp, vp = _pages(torch, count, p, hk, d, _type(torch, pages), layout, poison)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
        for t in (kp, vp):
            t[torch.from_numpy(table[i, :n].astype(np.int64)).cuda()] = torch.randn(
                n, p, hk, d, device="cuda").to(t.dtype)
        if lengths[i] % p:
            for t in (kp, vp):
                t[int(table[i, n - 1]), int(lengths[i]) % p:] = poison
    qg = torch.randn(b, hq, 2, d, device="cuda")
    q = (qg[:, :, 0] * 1.5).to(_type(torch, dtype))
    return q, qg[:, :, 1], F.PagedCache(kp, vp), _dev(torch, table), _dev(torch, lengths)


def _check_attention(got, q, gate, cache, table, lengths, scale, sessions=None, heads=None):
    bf16 = str(cache.k.dtype).endswith("bfloat16")
    out16 = str(got.dtype).endswith("bfloat16")
    b, hq, d = q.shape
    hk, p = cache.shape[2], cache.shape[1]
    q, got = _host(q), _host(got)
    table, lengths = table.cpu().numpy(), lengths.cpu().numpy()
    g = None if gate is None else 1.0 / (1.0 + np.exp(-_host(gate)))
    for i in range(b) if sessions is None else sessions:
        n = int(lengths[i])
        if n == 0:
            assert not got[i].any()
            continue
        pages = table[i, :-(-n // p)].astype(np.int64)
        k, v = (_host(t[pages.tolist()]).reshape(-1, hk, d)[:n] for t in (cache.k, cache.v))
        for h in range(hq) if heads is None else heads:
            kh = h // (hq // hk)
            want, pv, most = R.attend(q[i, h], k[:, kh], v[:, kh], scale)
            ds = most * ((d + 4) * 2.0 ** -24 + (2.0 ** -16 if bf16 else 0.0))
            bar = (2 * ds + 2.0 ** -20 + (n + 64) * 2.0 ** -23 + (2.0 ** -15 if bf16 else 0.0)) * pv
            if g is not None:
                want, bar = want * g[i, h], bar * g[i, h]
            bar = bar + np.abs(want) * ((2.0 ** -8 if out16 else 2.0 ** -24) + 2.0 ** -21)
            assert (np.abs(got[i, h] - want) <= bar).all(), (i, h, float((np.abs(got[i, h] - want) / bar).max()))


CASES = [
    # lengths, q heads, kv heads, head_dim, page size, q, pages, layout
    ([1], 2, 1, 64, 16, "f32", "bf16", "plain"),
    ([0, 5, 16, 17], 8, 2, 128, 16, "f32", "bf16", "heads"),
    ([777], 16, 2, 256, 16, "f32", "bf16", "plain"),
    ([33, 0, 1000, 64, 15], 12, 3, 80, 24, "bf16", "bf16", "one"),
    ([2304, 100, 2049], 16, 2, 256, 16, "f32", "f32", "plain"),
    ([40, 3, 0, 129], 4, 4, 64, 8, "bf16", "f32", "heads"),
    ([500, 31], 32, 1, 128, 32, "bf16", "bf16", "plain"),
    ([129, 70], 34, 2, 96, 48, "f32", "bf16", "one"),
    ([19, 40, 7], 5, 5, 48, 7, "f32", "bf16", "plain"),
    ([19, 40, 7], 6, 2, 16, 1, "f32", "f32", "plain"),
    ([5000, 1, 1, 1, 16, 0, 900], 16, 4, 128, 64, "bf16", "bf16", "heads"),
    ([300, 299], 9, 3, 240, 128, "bf16", "f32", "one"),
    ([127, 128, 129, 130], 20, 2, 192, 2, "bf16", "bf16", "plain"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[1]}-{c[2]}-{c[3]}-p{c[4]}-{c[5]}-{c[6]}-{c[7]}")
@pytest.mark.parametrize("gated", [True, False])
def test_paged_attention_matches_the_formula(F, torch, case, gated):
    lengths, hq, hk, d, p, dtype, pages, layout = case
    torch.manual_seed(sum(lengths) + d)
    rng = np.random.default_rng(sum(lengths) + hq)
    q, gate, cache, table, n = _attention_case(F, torch, rng, lengths, hq, hk, d, p, dtype, pages, layout)
    scale = 1.0 / math.sqrt(d) if gated else 0.3
    out = F.paged_attention(q, cache, table, n, gate=gate if gated else None, scale=None if gated else scale)
    assert out.dtype == cache.k.dtype
    _check_attention(out, q, gate if gated else None, cache, table, n, scale)


@pytest.mark.parametrize("pages", ["f32", "bf16"])
def test_paged_attention_many_sessions(F, torch, pages):
    """More key/value heads than the GPU has room for at once, lengths from none to
    long; out in the other type."""
    torch.manual_seed(3)
    rng = np.random.default_rng(3)
    lengths = np.where(rng.random(301) < 0.1, 0, np.exp(rng.uniform(0, 7, 301))).astype(int)
    lengths[7] = 9001
    q, gate, cache, table, n = _attention_case(F, torch, rng, lengths, 8, 4, 64, 16, "f32", pages)
    other = torch.empty(q.shape, dtype=torch.bfloat16 if pages == "f32" else torch.float32, device="cuda")
    out = F.paged_attention(q, cache, table, n, gate=gate, out=other)
    assert out is other
    _check_attention(out, q, gate, cache, table, n, 0.125, sessions=[0, 7, 100, 300] + rng.integers(0, 301, 30).tolist(),
                     heads=[0, 3, 7])
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("pages", ["f32", "bf16"])
def test_paged_attention_of_the_most_sessions(F, torch, pages):
    torch.manual_seed(41)
    rng = np.random.default_rng(41)
    lengths = rng.integers(0, 40, 4096)
    lengths[4095], lengths[17] = 3000, 0
    q, gate, cache, table, n = _attention_case(F, torch, rng, lengths, 4, 2, 64, 16, "f32", pages)
    out = F.paged_attention(q, cache, table, n, gate=gate)
    _check_attention(out, q, gate, cache, table, n, 0.125, sessions=[0, 17, 4095, *rng.integers(0, 4096, 40).tolist()])
    assert torch.isfinite(out).all() and not out[n == 0].any()
    with pytest.raises(F.FpbError):
        more = torch.zeros(4097, 4, 64, device="cuda")
        F.paged_attention(more, cache, table[:1].expand(4097, -1).contiguous(), torch.zeros(4097, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("pages", ["f32", "bf16"])
@pytest.mark.parametrize("b,hq,hk,d,most", [(70, 4, 1, 64, 900), (41, 12, 1, 256, 60), (20, 16, 8, 128, 700),
                                            (32, 8, 4, 80, 300), (33, 8, 4, 80, 300), (1, 64, 64, 32, 2000), (30, 16, 8, 64, 4000),
                                            (40, 8, 8, 64, 2500)])
def test_paged_attention_ways_to_cut(F, torch, pages, b, hq, hk, d, most):
    """Few and many sessions, in one wave of blocks and in several, some without
    tokens and one whose length cannot be."""
    torch.manual_seed(b)
    rng = np.random.default_rng(b + hk)
    lengths = rng.integers(1, most, b)
    lengths[rng.random(b) < 0.2] = 0
    lengths[-1] = most
    q, gate, cache, table, n = _attention_case(F, torch, rng, lengths, hq, hk, d, 16, "f32", pages)
    out = F.paged_attention(q, cache, table, n, gate=gate)
    _check_attention(out, q, gate, cache, table, n, d ** -0.5, heads=[0, hq - 1])
    assert torch.equal(out, F.paged_attention(q, cache, table, n, gate=gate))
    if b > 1:
        n[0] = -7
        out = F.paged_attention(q, cache, table, n, gate=gate)
        assert F.device_error(reset=True) == 507
        n[0] = 0
        _check_attention(out, q, gate, cache, table, n, d ** -0.5, sessions=[0, b // 2, b - 1], heads=[hq // 2])


def test_paged_attention_two_at_once(F, torch):
    """Calls on two streams with a workspace each, and two graphs that share one and
    are replayed in turn, the workspace written to in between."""
    torch.manual_seed(21)
    rng = np.random.default_rng(21)
    cases = [_attention_case(F, torch, rng, lengths, 16, 2, 128, 16, "f32", "bf16")
             for lengths in ([4000, 3, 700], [50, 9000, 0])]
    want = [F.paged_attention(q, cache, table, n, gate=gate) for q, gate, cache, table, n in cases]
    for w, (q, gate, cache, table, n) in zip(want, cases):
        _check_attention(w, q, gate, cache, table, n, 128 ** -0.5, heads=[0, 15])
    size = F.paged_attention_workspace_bytes(cases[0][2], 3, 16)
    outs = [torch.empty_like(w) for w in want]
    sides = [torch.cuda.Stream() for _ in cases]
    spaces = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for side, ws, out, (q, gate, cache, table, n) in zip(sides, spaces, outs, cases):
            F.paged_attention(q, cache, table, n, gate=gate, out=out, workspace=ws, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    graphs = []
    for out, (q, gate, cache, table, n) in zip(outs, cases):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=sides[0]):
            F.paged_attention(q, cache, table, n, gate=gate, out=out, workspace=spaces[0])
        graphs.append(g)
    for fill in (0, 255, 17):
        for g, out, w in zip(graphs, outs, want):
            out.zero_()
            g.replay()
            assert torch.equal(out, w)
            g.replay()
            assert torch.equal(out, w)
            spaces[0].fill_(fill)


@pytest.mark.parametrize("pages", ["f32", "bf16"])
def test_paged_attention_same_bits_in_every_call(F, torch, pages):
    torch.manual_seed(4)
    rng = np.random.default_rng(4)
    q, gate, cache, table, n = _attention_case(F, torch, rng, [700, 4000, 90], 16, 2, 128, 16, "f32", pages)
    first = F.paged_attention(q, cache, table, n, gate=gate)
    for _ in range(5):
        assert torch.equal(first, F.paged_attention(q, cache, table, n, gate=gate))


@pytest.mark.parametrize("pages", ["f32", "bf16"])
def test_paged_attention_scores_of_any_size(F, torch, pages):
    """Scores that differ by thousands, a maximum that comes last, equal scores, and
    values of any size."""
    torch.manual_seed(5)
    rng = np.random.default_rng(5)
    q, _, cache, table, n = _attention_case(F, torch, rng, [400, 400, 400, 400], 4, 2, 64, 16, "f32", pages)
    t = table.cpu().long()
    cache.k[t[0, :25]] *= 30.0
    cache.k[t[1, 24]] *= 200.0
    cache.k[t[2, :25]] = 0.0
    cache.v[t[3, :25]] *= 1e30
    out = F.paged_attention(q, cache, table, n)
    # (errors of a score grow with it: ds is taken at the largest; in the first two
    # sessions the winner takes all, by more than any error)
    _check_attention(out, q, None, cache, table, n, 0.125, sessions=[2, 3])
    qh, got = _host(q), _host(out)
    for i in (0, 1):
        pages_i = t[i, :25].tolist()
        k, v = (_host(x[pages_i]).reshape(-1, 2, 64) for x in (cache.k, cache.v))
        for h in range(4):
            want, _, most = R.attend(qh[i, h], k[:, h // 2], v[:, h // 2], 0.125)
            s = np.sort((k[:, h // 2] @ qh[i, h]) * 0.125)
            if s[-1] - s[-2] > 20 + 2 * most * 2.0 ** -15:  # a weight of e^-20 elsewhere at most
                assert np.abs(got[i, h] - want).max() <= 2.0 ** -7 * np.abs(v[:, h // 2]).max()
            else:
                assert np.isfinite(got[i, h]).all()


@pytest.mark.parametrize("pages", ["f32", "bf16"])
def test_paged_attention_nan_stays_where_it_is_seen(F, torch, pages):
    """A NaN among the values of a token that is seen makes its column NaN, one
    among the keys the whole head; other sessions and heads have none."""
    torch.manual_seed(6)
    rng = np.random.default_rng(6)
    q, _, cache, table, n = _attention_case(F, torch, rng, [50, 50, 50], 4, 2, 64, 16, "f32", pages)
    t = table.cpu()
    cache.v[int(t[0, 1]), 3, 1, 5] = math.nan
    cache.k[int(t[1, 3]), 1, 0, 9] = math.nan
    out = F.paged_attention(q, cache, table, n).float().isnan().cpu()
    want = torch.zeros(3, 4, 64, dtype=torch.bool)
    want[0, 2:, 5] = True
    want[1, :2] = True
    assert torch.equal(out, want)


def test_paged_attention_bad_tables_are_recorded(F, torch):
    """A token whose page is outside the pool is not there; a length past the table,
    or a negative one, is a session without tokens."""
    torch.manual_seed(7)
    rng = np.random.default_rng(7)
    for pages in ("f32", "bf16"):
        q, gate, cache, table, n = _attention_case(F, torch, rng, [100, 60, 20], 4, 2, 64, 16, "f32", pages)
        bad = table.clone()
        bad[0, 2], bad[1, 0] = cache.shape[0], -1
        out = F.paged_attention(q, cache, bad, n, gate=gate)
        assert F.device_error(reset=True) == 506
        # the same sessions without those tokens
        keep0 = [int(x) for i, x in enumerate(table.cpu()[0, :7]) if i != 2]
        short = table.clone()
        short[0, :6] = torch.tensor(keep0, dtype=torch.int32)
        short[1, :3] = table[1, 1:4]
        _check_attention(out, q, gate, cache, short, _dev(torch, np.array([84, 44, 20], np.int32)), 0.125)
        out = F.paged_attention(q, cache, table, _dev(torch, np.array([-1, 10 ** 9, 20], np.int32)), gate=gate)
        assert F.device_error(reset=True) == 507
        assert not out[:2].any()
        _check_attention(out, q, gate, cache, table, _dev(torch, np.array([0, 0, 20], np.int32)), 0.125)
        # every token's page outside: nothing is left
        out = F.paged_attention(q, cache, torch.full_like(table, 10 ** 6), n)
        assert F.device_error(reset=True) == 506 and not out.any()


def test_paged_attention_in_a_graph_on_another_stream(F, torch):
    """Lengths and tables that change between replays; a workspace of its own."""
    torch.manual_seed(8)
    rng = np.random.default_rng(8)
    q, gate, cache, table, n = _attention_case(F, torch, rng, [3000, 64, 500, 1], 16, 2, 128, 16, "f32", "bf16")
    ws = torch.empty(F.paged_attention_workspace_bytes(cache, 4, 16), dtype=torch.uint8, device="cuda")
    out = torch.empty(q.shape, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    F.paged_attention(q, cache, table, n, gate=gate, out=out, workspace=ws, stream=side.cuda_stream)
    side.synchronize()
    _check_attention(out, q, gate, cache, table, n, 128 ** -0.5)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        F.paged_attention(q, cache, table, n, gate=gate, out=out, workspace=ws)
    for lengths in ([3000, 64, 500, 1], [1, 0, 499, 1], [2999, 1, 33, 0]):
        n.copy_(_dev(torch, np.array(lengths, np.int32)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        _check_attention(out, q, gate, cache, table, n, 128 ** -0.5)


@pytest.mark.parametrize("pages", ["f32", "bf16"])
def test_paged_attention_past_32_bits(F, torch, pages):
    """Pages whose elements lie past 2^32."""
    torch.manual_seed(9)
    d, hk, p = 128, 2, 16
    count = 2 ** 32 // (d * hk * p) + 40
    td = _type(torch, pages)
    k = torch.empty(count, p, hk, d, dtype=td, device="cuda")
    v = torch.empty(count, p, hk, d, dtype=td, device="cuda")
    cache = F.PagedCache(k, v)
    table = torch.arange(count - 20, count, dtype=torch.int32, device="cuda").view(1, 20)
    lengths = _dev(torch, np.array([300], np.int32))
    x = torch.randn(300, 2, hk, d, device="cuda")
    slots = table[0].long().repeat_interleave(p)[:300] * p + torch.arange(300, device="cuda") % p
    F.paged_append(cache, slots.int(), torch.zeros(300, dtype=torch.int32, device="cuda"), x[:, 0], x[:, 1])
    assert torch.equal(k.view(-1, hk, d)[slots], x[:, 0].to(td)) and torch.equal(v.view(-1, hk, d)[slots], x[:, 1].to(td))
    q = torch.randn(1, 4, d, device="cuda")
    _check_attention(F.paged_attention(q, cache, table, lengths), q, None, cache, table, lengths, d ** -0.5)


# ---- sampling ------------------------------------------------------------------------------------------------------
def _check_sample(torch, tokens, logprobs, logits, noise, temperature, top_k, top_p, min_p):
    logits, noise = _host(logits), _host(noise)
    for i in range(len(logits)):
        f = dict(temperature=float(temperature[i]), top_k=int(top_k[i]), min_p=float(min_p[i]))
        p = float(np.float32(top_p[i]))
        right = False
        for q in ({p} if p >= 1 or p <= 0 else {p, p * (1 - 3e-5), min(p * (1 + 3e-5), 1 - 1e-12)}):
            want, log, race = R.sample(logits[i], noise[i], top_p=q, **f)
            got = int(tokens[i])
            if got == want or (got in race and race[got] >= race[want] - 6e-5):
                order, d = R.kept(logits[i], top_p=q, **f)
                if got >= 0:
                    log = float(d[list(order).index(got)] - np.log(np.exp(d).sum()))
                close = log == float(logprobs[i]) or abs(float(logprobs[i]) - log) <= 4e-5 + abs(log) * 2.0 ** -22
                right = right or close
        assert right, (i, int(tokens[i]), want, float(logprobs[i]), log, f, p)


def _sample_inputs(torch, b, vocab, dtype, seed, spread=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    spread = torch.rand(b, 1, generator=g, device="cuda") * 5 + 0.2 if spread is None else spread
    logits = (torch.randn(b, vocab, generator=g, device="cuda") * spread + 3.0).to(_type(torch, dtype))
    noise = torch.empty(b, vocab, device="cuda").exponential_(generator=g).clamp_(min=1e-20)
    rng = np.random.default_rng(seed)
    temperature = np.where(rng.random(b) < 0.15, 0.0, rng.uniform(0.3, 2.0, b)).astype(np.float32)
    top_k = np.where(rng.random(b) < 0.5, 0, np.exp(rng.uniform(0, math.log(vocab + 20), b))).astype(np.int32)
    top_p = np.where(rng.random(b) < 0.4, 1.0, rng.uniform(0.02, 0.999, b)).astype(np.float32)
    min_p = np.where(rng.random(b) < 0.6, 0.0, np.exp(rng.uniform(-7, 0, b))).astype(np.float32)
    return logits, noise, temperature, top_k, top_p, min_p


def _run_sample(F, torch, logits, noise, *filters, **kw):
    t, k, p, m = (_dev(torch, x) for x in filters)
    return F.sample(logits, t, noise, top_k=k, top_p=p, min_p=m, logprobs=True, **kw)


@pytest.mark.parametrize("b,vocab,dtype", [(1, 1, "f32"), (3, 2, "bf16"), (40, 33, "f32"), (64, 1000, "bf16"),
                                           (48, 4099, "f32"), (24, 32000, "bf16"), (40, 50257, "f32"),
                                           (12, 151936, "f32"), (30, 151936, "bf16"), (3, 393216, "bf16"),
                                           (94, 151936, "bf16"), (47, 50257, "f32"), (93, 32000, "bf16"), (100, 4099, "f32")])
def test_sample_matches_the_definition(F, torch, b, vocab, dtype):
    args = _sample_inputs(torch, b, vocab, dtype, b * 3 + vocab)
    tokens, logprobs = _run_sample(F, torch, *args)
    _check_sample(torch, tokens.cpu(), logprobs.cpu(), *args)


@pytest.mark.parametrize("b,vocab,dtype", [
    (93, 196608, "bf16"), (93, 196609, "bf16"), (93, 202048, "bf16"), (100, 204800, "bf16"), (93, 204801, "bf16"),
    (92, 204800, "bf16"), (93, 102400, "f32"), (93, 102401, "f32"), (93, 393216, "bf16"), (93, 393216, "f32"),
    (93, 32768, "f32"), (93, 32769, "bf16"), (47, 65536, "bf16"), (47, 65537, "f32")])
def test_sample_at_the_limits_of_its_ways(F, torch, b, vocab, dtype):
    """Rows and vocabularies on both sides of where a row takes two, four and eight CTAs."""
    args = _sample_inputs(torch, b, vocab, dtype, b + vocab)
    tokens, logprobs = _run_sample(F, torch, *args)
    rows = [0, 1, b // 2, b - 1]
    _check_sample(torch, tokens[rows].cpu(), logprobs[rows].cpu(), *(x[rows] for x in args))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_equal_logits_go_by_index(F, torch, dtype):
    """Ties at the border of each filter: rows of one value, of a few values, and
    steps; every filter alone."""
    vocab, rows = 20011, []
    g = torch.Generator(device="cuda").manual_seed(1)
    rows.append(torch.zeros(vocab, device="cuda"))
    rows.append(torch.randint(0, 3, (vocab,), generator=g, device="cuda").float())
    rows.append(-(torch.arange(vocab, device="cuda") // 1000).float())
    rows.append(torch.where(torch.arange(vocab, device="cuda") % 7 == 3, 2.0, -5.0))
    logits, filters = [], []
    for r in rows:
        for k, p, m in ((1, 1.0, 0.0), (300, 1.0, 0.0), (5003, 1.0, 0.0), (0, 1e-9, 0.0), (0, 0.25, 0.0), (0, 0.9, 0.0),
                        (0, 1.0, 0.3), (0, 1.0, 1.0), (3000, 0.5, 0.0), (3000, 0.5, 1.0), (vocab, 1.0, 0.0), (0, 0.0, 0.0),
                        (-1, 2.0, -1.0), (0, 1.0, 7.0)):
            logits.append(r)
            filters.append((1.0, k, p, m))
    b = len(filters)
    noise = torch.empty(b, vocab, device="cuda").exponential_(generator=g).clamp_(min=1e-20)
    t, k, p, m = (np.array(x) for x in zip(*filters))
    args = (torch.stack(logits).to(_type(torch, dtype)), noise, t.astype(np.float32), k.astype(np.int32),
            p.astype(np.float32), m.astype(np.float32))
    tokens, logprobs = _run_sample(F, torch, *args)
    _check_sample(torch, tokens.cpu(), logprobs.cpu(), *args)
    # a small noise on each token in turn finds exactly those that are kept
    for row in (1 * 14 + 1, 2 * 14 + 4, 0 * 14 + 8):
        order, _ = R.kept(_host(args[0][row]), temperature=1.0, top_k=int(k[row]), top_p=float(np.float32(p[row])),
                          min_p=float(m[row]))
        last = [int(order[0]), int(order[-1])]
        out = [x for x in range(vocab) if x not in set(order.tolist())][:1] + [vocab - 1]
        for x in last + [o for o in out if o not in set(order.tolist())]:
            few = torch.ones(1, vocab, device="cuda")
            few[0, x] = 1e-20
            one = [a[row:row + 1] for a in args[:1]] + [few] + [a[row:row + 1] for a in args[2:]]
            got = int(_run_sample(F, torch, *one)[0])
            # (a shortest part's last token is one that rounding may take or leave)
            if x in last[:1] or int(k[row]) > 0 and p[row] >= 1:
                assert (got == x) == (x in set(order.tolist()))


def test_sample_of_rows_that_are_not_finite(F, torch):
    """Infinities, NaN and the type's lowest value among the logits."""
    vocab = 5000
    low = torch.finfo(torch.float32).min
    logits = torch.randn(9, vocab, generator=torch.Generator().manual_seed(2)).cuda()
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, 1:] = -math.inf
    logits[3, ::2] = math.nan
    logits[4, 17] = math.inf
    logits[5] = low
    logits[6, 10:] = low
    logits[7, :4000] = -math.inf
    logits[8] = math.inf
    noise = torch.empty(9, vocab).exponential_(generator=torch.Generator().manual_seed(3)).clamp_(min=1e-20).cuda()
    for t in (0.0, 0.7, 1e-30, 1e30):
        for k, p, m in ((0, 1.0, 0.0), (20, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05), (50, 0.8, 0.01)):
            f = [np.full(9, x, y) for x, y in ((t, np.float32), (k, np.int32), (p, np.float32), (m, np.float32))]
            tokens, logprobs = _run_sample(F, torch, logits, noise, *f)
            _check_sample(torch, tokens.cpu(), logprobs.cpu(), logits, noise, *f)
            assert tokens.cpu().tolist()[:3] == [-1, -1, 0] and tokens[8] == -1


def test_sample_of_numbers_that_are_none(F, torch):
    """Numbers of zero, where a weight of 0 over one is no number, and NaN: the token is
    one of those that are kept, in every way to find it, and none that a NaN stands for
    where there is another."""
    vocab = 5000
    g = torch.Generator(device="cuda").manual_seed(31)
    ways = ((5, 1.0, 0.0), (40, 0.9, 0.0), (0, 0.7, 0.0), (2000, 1.0, 0.0), (0, 1.0, 0.0), (0, 0.999, 0.0), (0, 1.0, 1e-3))
    t, k, p, m = (np.array(x) for x in zip(*((1.0, *w) for w in ways)))
    f = t.astype(np.float32), k.astype(np.int32), p.astype(np.float32), m.astype(np.float32)
    b = len(ways)
    steep = -200.0 * torch.arange(vocab, device="cuda").float().expand(b, vocab).contiguous()
    tokens, logprobs = _run_sample(F, torch, steep, torch.zeros(b, vocab, device="cuda"), *f)
    assert tokens.tolist() == [0] * b and logprobs.abs().max() < 1e-6  # every other weight is 0
    logits = torch.randn(b, vocab, generator=g, device="cuda") * 3
    noise = torch.empty(b, vocab, device="cuda").exponential_(generator=g).clamp_(min=1e-20)
    first = logits.argmax(1)
    noise[torch.arange(b), first] = math.nan
    tokens, logprobs = _run_sample(F, torch, logits, noise, *f)
    less = noise.clone()
    less[torch.arange(b), first] = 1e30  # (never drawn)
    want, same = _run_sample(F, torch, logits, less, *f)
    assert torch.equal(tokens, want) and torch.equal(logprobs, same)
    tokens, _ = _run_sample(F, torch, logits, torch.full_like(noise, math.nan), *f)
    for i in range(b):
        order, _ = R.kept(_host(logits[i]), temperature=1.0, top_k=int(k[i]), top_p=float(p[i]), min_p=float(m[i]))
        assert int(tokens[i]) in order


def test_sample_draws_from_the_distribution(F, torch):
    """Frequencies of 40000 draws from one row, each within five standard
    deviations (a chance of 6e-7 each)."""
    n, vocab = 40000, 12
    g = torch.Generator(device="cuda").manual_seed(11)
    row = torch.randn(vocab, generator=g, device="cuda")
    noise = torch.empty(n, vocab, device="cuda").exponential_(generator=g).clamp_(min=1e-20)
    full = lambda x, d: torch.full((n,), x, dtype=d, device="cuda")  # noqa: E731
    tokens = F.sample(row.expand(n, vocab).contiguous(), full(0.8, torch.float32), noise, top_k=full(9, torch.int32))
    order, d = R.kept(_host(row), temperature=0.8, top_k=9)
    p = np.exp(d) / np.exp(d).sum()
    seen = np.bincount(tokens.cpu().numpy(), minlength=vocab)
    assert seen.sum() == seen[order].sum() == n
    assert (np.abs(seen[order] - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all()


def test_sample_strides_streams_and_graphs(F, torch):
    """Pitched rows at odd addresses; out; a captured call whose parameters change."""
    vocab, b = 3001, 6
    wide = _sample_inputs(torch, b, vocab + 7, "f32", 5)
    logits, noise, filters = wide[0][:, 3:3 + vocab], wide[1][:, 5:5 + vocab], wide[2:]
    tokens, logprobs = _run_sample(F, torch, logits, noise, *filters)
    _check_sample(torch, tokens.cpu(), logprobs.cpu(), logits, noise, *filters)
    t, k, p, m = (_dev(torch, x) for x in filters)
    out = torch.zeros(b, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        _, logprobs = F.sample(logits, t, noise, top_k=k, top_p=p, min_p=m, logprobs=True, out=out)
    for seed in range(3):
        again = _sample_inputs(torch, b, vocab + 7, "f32", 50 + seed)
        for dst, src in ((wide[0], again[0]), (wide[1], again[1])):
            dst.copy_(src)
        for dst, src in zip((t, k, p, m), again[2:]):
            dst.copy_(_dev(torch, src))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        _check_sample(torch, out.cpu(), logprobs.cpu(), logits, noise, *again[2:])
    assert torch.equal(F.sample(logits, None, noise), F.sample(logits, torch.ones_like(t), noise))
    plain = F.sample(logits, t, noise)
    ones = [np.float32([float(x) for x in t.cpu()]), np.zeros(b, np.int32), np.ones(b, np.float32), np.zeros(b, np.float32)]
    _, logs = F.sample(logits, t, noise, logprobs=True)
    _check_sample(torch, plain.cpu(), logs.cpu(), logits, noise, *ones)


# ---- the wrappers ---------------------------------------------------------------------------------------------------
def _a_step(F, torch, seed):
    """Every operator once, with everything that it can be given; what they wrote."""
    torch.manual_seed(seed)
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = F.PagedCache.zeros(40, 16, 2, 64)
    tables = F.PageTables.empty(3, 40, 16, 12)
    counts = torch.tensor([20, 0, 33], **i32)
    m = F.page_extend(tables, counts, 53)
    padded = F.page_extend(tables, torch.tensor([1, 2, 0], **i32), 6, True)
    mine = F.PageMap(torch.zeros(3, **i32), torch.zeros(3, **i32), None, torch.zeros(4, **i32))
    assert F.page_extend(tables, torch.ones(3, **i32), 3, out=mine) is mine
    F.page_truncate(tables, torch.tensor([21, -1, 33], **i32))
    x = torch.randn(53, 8, 64, device="cuda")
    gamma = torch.rand(64, device="cuda") + 0.5
    q = F.paged_append(cache, m.slots, m.positions, x[:, 4:6], x[:, 6:], q=x[:, :4], q_gamma=gamma, k_gamma=gamma, eps=1e-5,
                       rotary_dim=32, theta=1e6)
    q16 = torch.empty(53, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert F.paged_append(cache, m.slots, m.positions, x[:, 4:6], x[:, 6:], q=x[:, :4], q_out=q16) is q16
    assert F.paged_append(cache, m.slots, m.positions, x[:, 4:6], x[:, 6:]) is None
    rows = torch.tensor([19, 0, 52], device="cuda")
    gate = torch.randn(3, 4, 2, 64, device="cuda")[:, :, 1]
    att = F.paged_attention(q[rows], cache, tables.table, tables.lengths, gate=gate)
    out = torch.empty(3, 4, 64, device="cuda")
    ws = torch.empty(F.paged_attention_workspace_bytes(cache, 3, 4), dtype=torch.uint8, device="cuda")
    assert F.paged_attention(q16[rows], cache, tables.table, tables.lengths, scale=0.1, out=out, workspace=ws) is out
    logits = torch.randn(3, 1000, device="cuda")
    noise = torch.empty_like(logits).exponential_()
    t = torch.ones(3, device="cuda")
    k, p = torch.tensor([5, 0, 0], **i32), torch.tensor([1.0, 0.9, 1.0], device="cuda")
    tokens, logs = F.sample(logits, t, noise, top_k=k, top_p=p, min_p=p * 0.01, logprobs=True)
    plain = F.sample(logits.bfloat16(), t, noise)
    given = torch.zeros(3, **i32)
    assert F.sample(logits, None, noise, out=given) is given
    return [m.slots, m.positions, m.requests, m.starts, padded.slots, padded.positions, padded.requests, padded.starts,
            mine.slots, mine.positions, mine.starts, tables.table, tables.lengths, tables.free, tables.free_count, q, q16,
            cache.k, cache.v, att, out, tokens, logs, plain, given]


def test_calls_by_both_ways(F, torch, monkeypatch):
    """The module of calls is there, and what it makes is what the long way makes."""
    from firepit_b200.speculative import _Torch
    first = _a_step(F, torch, 3)
    assert _Torch.calls is not None
    seen = []
    for name in ("page_extend", "page_truncate", "paged_append", "paged_attention", "sample"):
        call = getattr(_Torch.calls, name)
        monkeypatch.setattr(_Torch.calls, name, lambda *a, call=call, name=name: seen.append((name, call(*a))) or seen[-1][1])
    for x, y in zip(first, _a_step(F, torch, 3)):
        assert torch.equal(x, y)
    assert len(seen) == 12 and not any(got is NotImplemented or type(got) is int for _, got in seen)
    monkeypatch.setattr(_Torch, "calls", None)
    for x, y in zip(first, _a_step(F, torch, 3)):
        assert x.dtype == y.dtype and x.stride() == y.stride() and torch.equal(x, y)


def test_calls_that_are_refused(F, torch):
    """On the device, each by one fault: an error and no launch."""
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = F.PagedCache.zeros(6, 16, 2, 64)
    tables = F.PageTables.empty(3, 6, 16, 4)
    n3, rows, f3 = torch.zeros(3, **i32), torch.zeros(5, **i32), torch.ones(3, device="cuda")
    kv, q, q3 = (torch.zeros(*s, device="cuda") for s in ((5, 2, 64), (5, 4, 64), (3, 4, 64)))
    logits, noise = torch.zeros(3, 10, device="cuda"), torch.ones(3, 10, device="cuda")
    host = lambda x: x.cpu()  # noqa: E731
    calls = [
        lambda: F.page_extend(tables, n3[:2], 5), lambda: F.page_extend(tables, n3.long(), 5),
        lambda: F.page_extend(tables, n3, 0), lambda: F.page_extend(tables, n3, 5, padded=True),
        lambda: F.page_extend(tables, host(n3), 5), lambda: F.page_extend(tables, tables.lengths, 5),
        lambda: F.page_extend(tables, n3, 5, out=F.PageMap(rows, rows[:4], None, None)),
        lambda: F.page_extend(tables, n3, 5, out=F.PageMap(rows, host(rows), None, None)),
        lambda: F.page_truncate(tables, n3.float()), lambda: F.page_truncate(tables, host(n3)),
        lambda: F.page_truncate(tables, torch.zeros(6, **i32)[::2]),
        lambda: F.paged_append(cache, rows, rows, kv[:, :1], kv[:, :1]),
        lambda: F.paged_append(cache, rows, rows, kv, kv.bfloat16()),
        lambda: F.paged_append(cache, rows.long(), rows, kv, kv), lambda: F.paged_append(cache, rows, rows[:4], kv, kv),
        lambda: F.paged_append(cache, rows, host(rows), kv, kv), lambda: F.paged_append(cache, rows, rows, kv, host(kv)),
        lambda: F.paged_append(cache, rows, rows, kv, kv, q=q.bfloat16()),
        lambda: F.paged_append(cache, rows, rows, kv, kv, q_out=q),
        lambda: F.paged_append(cache, rows, rows, kv, kv, q=q, q_gamma=torch.zeros(32, device="cuda")),
        lambda: F.paged_append(cache, rows, rows, kv, kv, q=q, q_gamma=torch.zeros(64)),
        lambda: F.paged_append(cache, rows, rows, kv, kv, q=q, q_out=q[:, :2]),
        lambda: F.paged_append(cache, rows, rows, kv, kv, q=q, rotary_dim=65),
        lambda: F.paged_append(cache, rows, rows, kv, kv, q=q, rotary_dim=32, theta=math.nan),
        lambda: F.paged_append(cache, rows, rows, kv.half(), kv.half()),
        lambda: F.paged_append(cache, rows, rows, torch.zeros(5, 2, 128, device="cuda")[..., ::2], kv),
        lambda: F.paged_append(cache, rows, rows, torch.zeros(5, 2, 80, device="cuda")[..., :64], kv),
        lambda: F.paged_attention(q3[:, :3], cache, tables.table, n3), lambda: F.paged_attention(q3[..., :32], cache, tables.table, n3),
        lambda: F.paged_attention(q3.half(), cache, tables.table, n3), lambda: F.paged_attention(q3, cache, tables.table[:2], n3),
        lambda: F.paged_attention(q3, cache, tables.table.long(), n3), lambda: F.paged_attention(q3, cache, tables.table, n3[:2]),
        lambda: F.paged_attention(q3, cache, host(tables.table), n3),
        lambda: F.paged_attention(q3, cache, tables.table[:, :0], n3),
        lambda: F.paged_attention(q3, cache, tables.table, n3, gate=q3.bfloat16()),
        lambda: F.paged_attention(q3, cache, tables.table, n3, gate=host(q3)),
        lambda: F.paged_attention(q3, cache, tables.table, n3, out=q3.half()),
        lambda: F.paged_attention(q3, cache, tables.table, n3, workspace=q3),
        lambda: F.paged_attention(q3, cache, tables.table, n3, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda")),
        lambda: F.paged_attention(q3, cache, tables.table, n3, scale=math.inf),
        lambda: F.paged_attention(q3[:0], cache, tables.table[:0], n3[:0]),
        lambda: F.sample(logits[0], f3, noise), lambda: F.sample(logits.half(), f3, noise), lambda: F.sample(logits, n3, noise),
        lambda: F.sample(logits, f3, noise[:, :9]), lambda: F.sample(logits, f3, noise.bfloat16()),
        lambda: F.sample(logits, f3, host(noise)), lambda: F.sample(logits, f3, noise, top_k=f3),
        lambda: F.sample(logits, f3, noise, top_p=n3), lambda: F.sample(logits, f3, noise, min_p=f3[:2]),
        lambda: F.sample(logits, f3, noise, out=n3.long()), lambda: F.sample(logits, host(f3), noise),
        lambda: F.sample(logits[:0], f3[:0], noise[:0]), lambda: F.sample(logits[:1].expand(3, 10), f3, noise),
        lambda: F.sample(logits.t(), torch.ones(10, device="cuda"), noise.t()),
    ]
    before = F.launch_count()
    for at, call in enumerate(calls):
        with pytest.raises((F.ShapeError, F.FpbError)):
            call()
            pytest.fail(f"call {at} was taken")
    assert F.launch_count() == before
