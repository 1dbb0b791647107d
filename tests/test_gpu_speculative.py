"""Speculative decoding over the 8-bit cache: append, read, keep, tree
attention and verification against the oracle's restatement in 64 bits
(oracle/speculative.py).

Bars, derived from the arithmetic:
 - q (f32): the sum of squares, its root and the gain are about 20 f32
   roundings of which half count, the angle is known to pi * 2^-25 and its
   sine to 2 ulp: 3e-6 of the head's largest value; bf16: 2^-8 more of each.
 - values in the cache: half a step of e4m3 (2^-4 relative, 2^-10 of the
   exponent's unit below the normal range) on top of k's own f32 error.
 - v's codes, the read-back and the kept rows: equal.
 - attention: products of f16 with f32 sums.  A score is off by at most
   2^-11 * scale * sum |q_i k_i| = ds, so a weight by 2 ds + 2^-11 of itself,
   and the output by (2 ds + 2^-11 + 2^-16) * sum p |v| + 2^-8 |out| (bf16
   rounding, with the gate's f32 error).
 - verification: whole numbers, equal.
"""
import math

import numpy as np
import pytest

from oracle import speculative as R

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


def _tree(rng, batch, nodes, absent=True):
    out = np.full((batch, nodes), -2, np.int32)
    for b in range(batch):
        count = nodes if b == 0 or not absent else rng.integers(1, nodes + 1)
        for i in range(count):
            out[b, i] = -1 if i == 0 else i - 1 if rng.random() < 0.5 else rng.integers(max(0, i - 6), i)
    return out


def _lines(parents, batch, nodes):
    return [R.ancestors(range(-1, nodes - 1) if parents is None else parents[b]) for b in range(batch)]


def _cache(F, torch, rng, b, s, hk, d, garbage=False):
    """A filled cache and its values; `garbage`: every byte that is not
    written later is as likely a NaN as anything."""
    if garbage:
        c = [_dev(torch, rng.integers(0, 256, (b, s, hk, d), dtype=np.uint8)) for _ in range(2)]
        e = [_dev(torch, rng.integers(0, 256, (b, s, hk), dtype=np.uint8)) for _ in range(2)]
        return F.Kv8Cache(c[0], c[1], e[0], e[1])
    k = rng.standard_normal((b, s, hk, d)) * 1.3
    v = rng.standard_normal((b, s, hk, d)) * np.exp(rng.standard_normal((b, s, hk, 1)))
    (kc, ke), (vc, ve) = R.quantise(k), R.quantise(v)
    return F.Kv8Cache(*(_dev(torch, x) for x in (kc, vc, ke, ve)))


def _host(t):
    return t.float().cpu().numpy().astype(np.float64)


# ---- append and read ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("b,n,hq,hk,d,rot,tree,dtype", [
    (1, 1, 2, 1, 16, 16, False, "f32"), (3, 1, 16, 2, 256, 64, False, "f32"), (2, 7, 6, 3, 80, 20, True, "bf16"),
    (2, 64, 4, 4, 64, 64, True, "f32"), (1, 130, 5, 1, 96, 0, False, "bf16"), (2, 5, 8, 2, 128, 128, True, "bf16"),
    (1, 3, 3, 3, 240, 238, True, "f32"), (1, 2, 1, 1, 48, 2, False, "f32")])
def test_append_matches_the_formulas(F, torch, b, n, hq, hk, d, rot, tree, dtype):
    rng = np.random.default_rng(b * 1000 + n * 10 + d)
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    s = 70000 if n == 1 else n + 40
    pos = np.array([s - n - 3 * i for i in range(b)], np.int32)
    parents = _tree(rng, b, n) if tree else None
    qg = _dev(torch, rng.standard_normal((b, n, hq, 2, d)).astype(np.float32) * 3, td)
    kv = _dev(torch, rng.standard_normal((b, n, 2, hk, d)).astype(np.float32), td)
    q, k, v = qg[..., 0, :], kv[:, :, 0], kv[:, :, 1]  # pitched views of wider rows
    qga, kga = (_dev(torch, (1 + 0.1 * rng.standard_normal(d)).astype(np.float32)) for _ in range(2))
    cache = F.Kv8Cache.zeros(b, s, hk, d)
    got = F.kv8_append(cache, _dev(torch, pos), k, v, q=q, parents=None if parents is None else _dev(torch, parents),
                       q_gamma=qga, k_gamma=kga, eps=1e-6, rotary_dim=rot, theta=1e4)
    rk, rv = F.kv8_read(cache, _dev(torch, pos), n)
    got, rk, rv, q, k, v = (_host(x) for x in (got, rk, rv, q, k, v))
    codes = {x: getattr(cache, x).cpu().numpy() for x in ("k", "v", "k_exp", "v_exp")}
    lines = _lines(parents, b, n)
    for i in range(b):
        rest = np.ones(s, bool)
        for j in range(n):
            if lines[i][j] is None:
                assert not got[i, j].any() and not rk[i, j].any() and not rv[i, j].any()
                continue
            rest[pos[i] + j] = False
            at = int(pos[i]) + len(lines[i][j]) - 1
            want = R.norm_rotate(q[i, j], qga.cpu().numpy(), 1e-6, at, rot, 1e4)
            big = np.abs(want).max(-1, keepdims=True)
            assert (np.abs(got[i, j] - want) <= 3e-6 * big + (0 if dtype == "f32" else 2.0 ** -8 * np.abs(want))).all()
            want = R.norm_rotate(k[i, j], kga.cpu().numpy(), 1e-6, at, rot, 1e4)
            big = np.abs(want).max(-1, keepdims=True)
            unit = 2.0 ** R.exponent(big * (1 + 3e-6))
            assert (np.abs(rk[i, j] - want) <= 3e-6 * big + np.maximum(2.0 ** -4 * np.abs(want) * (1 + 3e-6),
                                                                        2.0 ** -10 * unit)).all()
            vc, ve = R.quantise(v[i, j])
            assert np.array_equal(codes["v"][i, pos[i] + j], vc) and np.array_equal(codes["v_exp"][i, pos[i] + j], ve)
            assert np.array_equal(rv[i, j], R.values(vc, ve))
        assert not codes["k"][i, rest].any() and (codes["k_exp"][i, rest] == 119).all()


def test_append_holds_extreme_vectors(F, torch):
    """Zeros, subnormals, the largest f32, infinities, NaN, ties and the
    exponent's boundary at 448 * 2^e."""
    d = 32
    x = np.zeros((1, 10, 1, d), np.float32)
    x[0, 1, 0, 3] = 1e-44
    x[0, 2, 0] = 3e38
    x[0, 3, 0, :4] = [np.inf, 5.0, -np.inf, 0.0]
    x[0, 4, 0, :3] = [np.nan, 1.0, -2.0]
    x[0, 5, 0, :4] = [448.0, 9.0 * 2, 17.0, 1.0625]  # ties to even: 17 between 16 and 18
    x[0, 6, 0, :2] = [np.nextafter(np.float32(448), np.float32(500)), 100.0]
    x[0, 7, 0, :3] = [448.0, 2.0 ** -9, 2.0 ** -10]
    x[0, 8, 0, :2] = [1e-30, -1e-31]
    x[0, 9, 0, :2] = [-0.0, 1.5]
    cache = F.Kv8Cache.zeros(1, 10, 1, d)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    t = _dev(torch, x)
    assert F.kv8_append(cache, pos, t, t) is None
    codes, exps = cache.v.cpu().numpy()[0, :, 0], cache.v_exp.cpu().numpy()[0, :, 0]
    assert np.array_equal(cache.k.cpu().numpy(), cache.v.cpu().numpy())
    for i in (0, 1, 2, 5, 6, 7, 8, 9):
        wc, we = R.quantise(x[0, i, 0])
        assert np.array_equal(codes[i], wc) and exps[i] == we, i
    assert exps[0] == 119 and exps[5] == 127 and exps[6] == 128
    k, _ = F.kv8_read(cache, 0, 10)
    k = k.cpu().numpy()[0, :, 0]
    assert exps[3] == 247 and np.isinf(k[3, 0]) and np.isinf(k[3, 2]) and k[3, 1] == 0
    assert np.isnan(k[4, 0]) and k[4, 1] == 1.0 and k[4, 2] == -2.0


@pytest.mark.parametrize("b,s,hk,d,count", [(1, 1, 1, 16, 1), (3, 70, 3, 80, 33), (2, 500, 2, 256, 499)])
def test_read_gives_the_values(F, torch, b, s, hk, d, count):
    rng = np.random.default_rng(s)
    cache = _cache(F, torch, rng, b, s, hk, d)
    begin = rng.integers(0, s - count + 1, b).astype(np.int32)
    want = [R.values(getattr(cache, x).cpu().numpy(), getattr(cache, x + "_exp").cpu().numpy()) for x in "kv"]
    for dtype in (torch.float32, torch.bfloat16):
        for w, g in zip(want, F.kv8_read(cache, _dev(torch, begin), count, dtype)):
            assert g.dtype == dtype
            assert np.array_equal(_host(g), np.stack([w[i, begin[i]:begin[i] + count] for i in range(b)]))
        for w, g in zip(want, F.kv8_read(cache, s - count, count, dtype)):
            assert np.array_equal(_host(g), w[:, s - count:])


def test_keep_moves_the_path(F, torch):
    rng = np.random.default_rng(4)
    b, s, hk, d, n = 4, 40, 2, 48, 9
    cache = _cache(F, torch, rng, b, s, hk, d)
    pos = np.array([0, 31, 17, 5], np.int32)
    path = np.full((b, n), -1, np.int32)
    path[0, :4], path[1, :9], path[2, :1] = [0, 2, 3, 8], range(9), [0]  # session 3: nothing kept
    before = {x: getattr(cache, x).cpu().numpy() for x in ("k", "v", "k_exp", "v_exp")}
    F.kv8_keep(cache, _dev(torch, pos), _dev(torch, path))
    for x, old in before.items():
        want = old.copy()
        for i in range(b):
            for j, src in enumerate(p for p in path[i] if p >= 0):
                want[i, pos[i] + j] = old[i, pos[i] + src]
        assert np.array_equal(getattr(cache, x).cpu().numpy(), want), x


# ---- attention ------------------------------------------------------------------------------------------------------
def _check_attention(F, torch, rng, cache, pos, parents, n, hq, q_dtype="f32", gate=True, scale=None, amp=1.5,
                     stream=None):
    b, s, hk, d = cache.shape
    td = torch.float32 if q_dtype == "f32" else torch.bfloat16
    wide = _dev(torch, (rng.standard_normal((b, n, hq, 2, d)) * amp).astype(np.float32), td)
    q = wide[..., 0, :]
    gates = _dev(torch, rng.standard_normal((b, n, hq, 2 * d)).astype(np.float32))[..., d:] if gate else None
    out = F.tree_attention(q, cache, _dev(torch, np.asarray(pos, np.int32)),
                           None if parents is None else _dev(torch, parents), gate=gates, scale=scale)
    torch.cuda.synchronize()
    assert out.dtype == torch.bfloat16
    got, q = _host(out), _host(q)
    scale = 1 / math.sqrt(d) if scale is None else scale
    k, v = (R.values(getattr(cache, x).cpu().numpy(), getattr(cache, x + "_exp").cpu().numpy()) for x in "kv")
    lines = _lines(parents, b, n)
    for i in range(b):
        for j in range(n):
            if lines[i][j] is None:
                assert not got[i, j].any()
                continue
            rows = list(range(pos[i])) + [pos[i] + a for a in lines[i][j]]
            for h in range(hq):
                kh = h // (hq // hk)
                o, pv, sabs = R.attend(q[i, j, h], k[i, rows, kh], v[i, rows, kh], scale)
                bound = (2 * 2.0 ** -11 * sabs + 2.0 ** -11 + 2.0 ** -16) * pv
                if gate:
                    g = 1 / (1 + np.exp(-_host(gates[i, j, h])))
                    o, bound = o * g, bound * g
                err = np.abs(got[i, j, h] - o)
                assert (err <= bound + 2.0 ** -8 * np.abs(o)).all(), (i, j, h, float((err / (bound + 1e-30)).max()))
    return got


@pytest.mark.parametrize("b,n,hq,hk,d,s,pos,q_dtype", [
    (1, 1, 1, 1, 16, 1, [0], "f32"),             # the first token of a session: itself alone
    (2, 1, 8, 2, 64, 130, [0, 129], "f32"),
    (1, 1, 16, 2, 256, 700, [650], "bf16"),
    (3, 1, 3, 3, 80, 300, [127, 128, 255], "f32"),  # contexts that end on either side of a tile
    (2, 5, 8, 2, 128, 400, [63, 390], "bf16"),
    (2, 16, 16, 2, 256, 520, [500, 7], "f32"),
    (1, 64, 4, 1, 96, 200, [100], "f32"),
    (2, 33, 12, 2, 192, 150, [64, 1], "bf16"),
    (1, 61, 16, 1, 128, 4200, [4100], "f32"),
    (1, 2, 48, 2, 112, 333, [300], "f32"),       # 24 heads a group
    (1, 3, 130, 1, 32, 70, [66], "f32"),         # one key head for 130 query heads
])
def test_tree_attention(F, torch, b, n, hq, hk, d, s, pos, q_dtype):
    rng = np.random.default_rng(n * 100 + d + s)
    cache = _cache(F, torch, rng, b, s, hk, d)
    _check_attention(F, torch, rng, cache, pos, _tree(rng, b, n), n, hq, q_dtype)


@pytest.mark.parametrize("tree", [False, True])
def test_many_sessions_of_any_length_share_the_gpu(F, torch, tree):
    """More sessions than a warp has lanes, from one token to some hundreds;
    with trees, fifty are not there, the first forty among them."""
    rng = np.random.default_rng(14)
    b, n, s = 75, 20, 640
    cache = _cache(F, torch, rng, b, s, 1, 32)
    pos = rng.integers(0, s - n + 1, b).astype(np.int32)
    pos[::7] = 0
    par = _tree(rng, b, n) if tree else None
    if tree:
        par[:40, 0] = par[50:60, 0] = -2
    _check_attention(F, torch, rng, cache, pos.tolist(), par, n, 2)
    assert F.device_error(reset=True) == 0


@pytest.mark.parametrize("tree,d,gate", [(False, 32, True), (True, 128, False), (True, 208, True)])
def test_more_heads_and_sessions_than_blocks(F, torch, tree, d, gate):
    """Three hundred key heads with a tile or two of tokens each: a block
    takes several of them whole."""
    rng = np.random.default_rng(15)
    b, n, hk, s = 75, 5, 4, 150
    cache = _cache(F, torch, rng, b, s, hk, d)
    pos = rng.integers(0, s - n + 1, b)
    par = _tree(rng, b, n) if tree else None
    if tree:
        par[20:30, 0] = -2
    _check_attention(F, torch, rng, cache, pos.tolist(), par, n, 16, gate=gate)


@pytest.mark.parametrize("n", [3, 20])
def test_attention_of_positions_outside_the_cache(F, torch, n):
    rng = np.random.default_rng(16)
    cache = _cache(F, torch, rng, 5, 90, 1, 32)
    q = _dev(torch, rng.standard_normal((5, n, 2, 32)).astype(np.float32))
    out = F.tree_attention(q, cache, _dev(torch, np.array([-1, 90, 1 << 30, 88, 0], np.int32)), None)
    live = (out != 0).any(-1).any(-1).cpu().numpy()
    assert not live[:3].any() and live[3].tolist() == [True] * 2 + [False] * (n - 2) and live[4].all()
    assert F.device_error(reset=True) == 502


@pytest.mark.parametrize("n,pos", [(1, 0), (70, 0), (200, 57)])
def test_chain_attention_is_causal(F, torch, n, pos):
    """parents None: a prompt's chunk, longer than a tree may be."""
    rng = np.random.default_rng(n)
    cache = _cache(F, torch, rng, 1, n + pos, 2, 64)
    _check_attention(F, torch, rng, cache, [pos], None, n, 4, gate=False)


def test_attention_scale_and_large_scores(F, torch):
    """Scores of some hundreds: one weight takes all; a negative scale; queries
    far outside f16's range."""
    rng = np.random.default_rng(5)
    cache = _cache(F, torch, rng, 1, 300, 2, 64)
    par = _tree(rng, 1, 4)
    _check_attention(F, torch, rng, cache, [290], par, 4, 4, scale=-0.5)
    _check_attention(F, torch, rng, cache, [290], par, 4, 4, amp=1e6, scale=1e-6)
    _check_attention(F, torch, rng, cache, [290], par, 4, 4, amp=1e-7, scale=1e6)
    _check_attention(F, torch, rng, cache, [290], par, 4, 4, amp=0.0)


def test_attention_of_values_of_very_different_size(F, torch):
    """Value vectors 2^-40 to 2^40 in size, and zeros among them: each row's
    own exponent weighs it."""
    rng = np.random.default_rng(6)
    b, s, hk, d = 1, 200, 1, 64
    k = rng.standard_normal((b, s, hk, d))
    v = rng.standard_normal((b, s, hk, d)) * 2.0 ** rng.integers(-40, 41, (b, s, hk, 1))
    v[0, 50:60] = 0.0
    (kc, ke), (vc, ve) = R.quantise(k), R.quantise(v)
    cache = F.Kv8Cache(*(_dev(torch, x) for x in (kc, vc, ke, ve)))
    _check_attention(F, torch, rng, cache, [190], _tree(rng, 1, 3), 3, 2)


def test_rows_that_are_not_seen_never_matter(F, torch):
    """Everything past the tree, every node that is not there and every
    sibling may hold NaN codes and any exponent."""
    rng = np.random.default_rng(7)
    b, n, s, hk, d, hq = 3, 12, 300, 2, 64, 4
    pos = np.array([100, 0, 257], np.int32)
    par = _tree(rng, b, n)
    clean, dirty = _cache(F, torch, rng, b, s, hk, d), _cache(F, torch, rng, b, s, hk, d, garbage=True)
    lines = _lines(par, b, n)
    node = n - 1
    for i in range(b):  # only what session i's last node that is there sees is filled
        node = max(j for j in range(n) if lines[i][j] is not None)
        rows = list(range(pos[i])) + [int(pos[i]) + a for a in lines[i][node]]
        for x in ("k", "v", "k_exp", "v_exp"):
            getattr(dirty, x)[i, rows] = getattr(clean, x)[i, rows]
    q = _dev(torch, rng.standard_normal((b, n, hq, d)).astype(np.float32))
    want, got = (F.tree_attention(q, c, _dev(torch, pos), _dev(torch, par)) for c in (clean, dirty))
    for i in range(b):
        node = max(j for j in range(n) if lines[i][j] is not None)
        assert torch.equal(want[i, node], got[i, node])
        for j in range(n):
            if lines[i][j] is None:
                assert not got[i, j].any()


def test_nan_reaches_those_who_see_it(F, torch):
    rng = np.random.default_rng(8)
    cache = _cache(F, torch, rng, 1, 40, 1, 32)
    par = np.array([[-1, 0, 0, 1]], np.int32)
    q = _dev(torch, rng.standard_normal((1, 4, 2, 32)).astype(np.float32))
    cache.v[0, 31, 0, 5] = 0x7f  # node 1's value: seen by nodes 1 and 3
    out = F.tree_attention(q, cache, _dev(torch, np.array([30], np.int32)), _dev(torch, par))
    nan = torch.isnan(out).any(-1).any(-1).cpu().numpy()[0]
    assert nan.tolist() == [False, True, False, True]
    cache.v[0, 31, 0, 5] = 0
    q[0, 2, 1, 7] = math.nan
    out = F.tree_attention(q, cache, _dev(torch, np.array([30], np.int32)), _dev(torch, par))
    nan = torch.isnan(out).any(-1).cpu().numpy()[0]
    assert nan.tolist() == [[False, False], [False, False], [False, True], [False, False]]


def test_sessions_without_a_tree_and_faulty_trees(F, torch):
    rng = np.random.default_rng(9)
    cache = _cache(F, torch, rng, 4, 50, 2, 64)
    par = np.array([[-1, 0, 1], [-2, 0, 1], [-1, 1, 0], [-1, 0, 1]], np.int32)  # 2: node 1 is its own parent
    pos = np.array([10, 10, 10, 48], np.int32)  # 3: node 2 would lie past the cache
    q = _dev(torch, rng.standard_normal((4, 3, 4, 64)).astype(np.float32))
    out = F.tree_attention(q, cache, _dev(torch, pos), _dev(torch, par))
    live = (out != 0).any(-1).any(-1).cpu().numpy()
    assert live.tolist() == [[True] * 3, [False] * 3, [True, False, True], [True, True, False]]
    assert F.device_error(reset=True) in (502, 504)
    kv = _dev(torch, rng.standard_normal((4, 3, 2, 64)).astype(np.float32))
    old = cache.k.clone()
    F.kv8_append(cache, _dev(torch, pos), kv, kv, parents=_dev(torch, par))
    changed = (cache.k != old).any(-1).any(-1).cpu().numpy()
    assert [np.flatnonzero(c).tolist() for c in changed] == [[10, 11, 12], [], [10, 12], [48, 49]]
    assert F.device_error(reset=True) in (502, 504)
    out = F.tree_attention(q, cache, _dev(torch, np.array([-1, 50, 1 << 30, 0], np.int32)), None)
    assert not out[:3].any() and out[3].any()
    assert F.device_error(reset=True) == 502
    F.kv8_read(cache, _dev(torch, np.array([-1, 0, 0, 0], np.int32)), 3)
    assert F.device_error(reset=True) == 502


def test_attention_agrees_with_itself_over_splits_and_streams(F, torch):
    """The same tree in a short cache and in one with room for a million rows
    (another split of the work), on another stream, twice: no dependence on
    what ran before, the same bits from one run to the next."""
    rng = np.random.default_rng(10)
    b, n, hq, hk, d = 2, 9, 8, 2, 64
    short = _cache(F, torch, rng, b, 3000, hk, d)
    pos, par = _dev(torch, np.array([2900, 1234], np.int32)), _dev(torch, _tree(rng, b, n))
    q = _dev(torch, rng.standard_normal((b, n, hq, d)).astype(np.float32))
    long_ = F.Kv8Cache.zeros(b, 1 << 20, hk, d)
    for x in ("k", "v", "k_exp", "v_exp"):
        getattr(long_, x)[:, :3000] = getattr(short, x)
    one, two = (F.tree_attention(q, c, pos, par).float() for c in (short, long_))
    assert float((one - two).abs().max()) <= 2.0 ** -7 * float(one.abs().max())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [F.tree_attention(q, short, pos, par, stream=side.cuda_stream) for _ in range(3)]
    side.synchronize()
    for o in outs:
        assert torch.equal(o.float(), one)


def test_long_cache_offsets_pass_32_bits(F, torch):
    """A cache of over 2^32 codes: the last session's rows lie past any 32-bit
    offset."""
    b, s, hk, d = 5, 1 << 21, 2, 256
    cache = F.Kv8Cache.zeros(b, s, hk, d)
    rng = np.random.default_rng(11)
    pos = np.array([3, 0, 0, 0, s - 300], np.int32)
    kv = _dev(torch, rng.standard_normal((b, 2, hk, d)).astype(np.float32))
    q = _dev(torch, rng.standard_normal((b, 2, 4, d)).astype(np.float32))
    F.kv8_append(cache, _dev(torch, pos), kv, kv)
    k, v = F.kv8_read(cache, _dev(torch, pos), 2)
    for g in (k, v):
        assert float((g - kv).abs().max()) <= 2.0 ** -4 * float(kv.abs().max())
    assert int((cache.k[4, s - 300:s - 298] != 0).sum()) > 900 and not cache.k[3, 2:4000].any()
    out = F.tree_attention(q * 50, cache, _dev(torch, pos), None)
    # zero keys score 0 against a large score: where the node's own score is positive it takes every weight
    sc = (q * 50 * k.repeat_interleave(2, 2)).sum(-1) / 16
    for h in range(4):
        if float(sc[4, 0, h]) > 60:
            assert float((out[4, 0, h].float() - v[4, 0, h // 2]).abs().max()) <= 0.01 * float(v.abs().max())
    F.kv8_keep(cache, _dev(torch, pos), _dev(torch, np.array([[0, 1]] * b, np.int32)))
    del cache


# ---- verification ---------------------------------------------------------------------------------------------------
def _softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def _verify_case(rng, b, n, vocab, temperature, drawn, tree, dtype, torch):
    logits = (rng.standard_normal((b, n, vocab)) * 2).astype(np.float32)
    if dtype == "bf16":
        logits = torch.from_numpy(logits).to(torch.bfloat16).float().numpy()
    parents = _tree(rng, b, n) if tree else np.tile(np.arange(-1, n - 1, dtype=np.int32), (b, 1))
    draft = _softmax(logits / max(temperature, 0.5) + 0.5 * rng.standard_normal(logits.shape)).astype(np.float32)
    tokens = np.zeros((b, n), np.int32)
    for i in range(b):
        for j in range(n):
            up = max(0, parents[i, j])
            if drawn:
                tokens[i, j] = rng.choice(vocab, p=draft[i, up].astype(np.float64) / draft[i, up].sum(dtype=np.float64))
            else:
                tokens[i, j] = rng.choice(np.argsort(-logits[i, up])[:3])
    accept = rng.random((b, n)).astype(np.float32)
    noise = np.maximum(rng.exponential(size=(b, vocab)), 1e-20).astype(np.float32)
    return logits, tokens, parents, draft if drawn else None, accept, noise


@pytest.mark.parametrize("b,n,vocab,temperature,drawn,tree,dtype", [
    (1, 1, 1, 0.0, False, False, "f32"), (1, 1, 7, 1.0, False, False, "f32"), (3, 5, 1000, 0.0, False, False, "f32"),
    (4, 64, 333, 0.7, False, True, "f32"), (4, 17, 4096, 1.0, True, True, "bf16"), (2, 9, 50001, 1.0, True, False, "f32"),
    (6, 12, 151936, 0.8, False, True, "bf16"), (2, 8, 151936, 1.3, True, True, "f32"), (5, 30, 77, 0.0, False, True, "bf16"),
    (1, 3, 442368, 1.0, False, True, "bf16"), (6, 12, 151936, 0.2, False, True, "f32")])
def test_verify_takes_the_walk(F, torch, b, n, vocab, temperature, drawn, tree, dtype):
    rng = np.random.default_rng(n * 7 + vocab)
    lengths = set()
    for rep in range(3):
        logits, tokens, parents, draft, accept, noise = _verify_case(rng, b, n, vocab, temperature, drawn, tree, dtype,
                                                                     torch)
        td = torch.float32 if dtype == "f32" else torch.bfloat16
        wide = torch.zeros(b, n, vocab + 5, dtype=td, device="cuda")  # rows of a wider buffer
        wide[..., :vocab] = _dev(torch, logits)
        lg = wide[..., :vocab] if rep else wide[..., :vocab].contiguous()
        path, count, nxt = F.tree_verify(lg, _dev(torch, tokens), _dev(torch, parents) if tree else None, temperature,
                                         *((_dev(torch, x) for x in (accept, noise)) if temperature else (None, None)),
                                         draft=None if draft is None else _dev(torch, draft))
        path, count, nxt = (x.cpu().numpy() for x in (path, count, nxt))
        for i in range(b):
            want, token = R.verify(logits[i], tokens[i], parents[i], temperature, accept[i], noise[i],
                                   None if draft is None else draft[i])
            assert path[i].tolist() == want + [-1] * (n - len(want)) and count[i] == len(want) and nxt[i] == token
            lengths.add(len(want))
    # a certain draft is taken with the target's own probability: hardly ever where it is spread over a large vocabulary
    assert n < 5 or len(lengths) > 1 or (vocab > 5000 and not drawn and temperature > 0.5)


def test_verify_corners(F, torch):
    """Ties, banned and non-finite logits, repeated and faulty tokens, a draft
    equal to the target, a session with no tree."""
    inf, nan = np.inf, np.nan
    V = 16
    lg = np.full((8, 3, V), -1.0, np.float32)
    lg[0, 0, [3, 9]] = 5.0                       # greedy tie: the lower index
    lg[1, 0, [2, 4, 5]] = [inf, nan, 7.0]        # only finite logits count
    lg[2] = -inf                                 # nothing left: token 0
    lg[4, 0] = -inf
    lg[4, 0, 6] = 3.0
    tokens = np.array([[0, 9, 3], [0, 2, 5], [0, 1, 2], [0, 1, 2], [0, 6, 6], [0, 16, -1], [0, 3, 3], [0, 1, 1]], np.int32)
    par = np.array([[-1, 0, 0], [-1, 0, 0], [-1, 0, 0], [-2, 0, 0], [-1, 0, 0], [-1, 0, 0], [-1, 0, 0], [-1, 0, -2]],
                   np.int32)
    dev = lambda x: _dev(torch, x)  # noqa: E731
    path, count, nxt = F.tree_verify(dev(lg), dev(tokens), dev(par))
    want = [R.verify(lg[i], tokens[i], par[i], 0) for i in range(8)]
    assert path.cpu().tolist() == [p + [-1] * (3 - len(p)) for p, _ in want]
    assert nxt.cpu().tolist() == [t if t >= 0 else -1 for _, t in want] and count.cpu().tolist()[3] == 0
    assert path.cpu().tolist()[0] == [0, 2, -1] and nxt.cpu().tolist()[2] == 0
    assert F.device_error(reset=True) == 505
    accept = np.full((8, 3), 0.999, np.float32)
    noise = np.linspace(0.5, 1.5, 8 * V).astype(np.float32).reshape(8, V)
    lg[2] = 0.0
    path, count, nxt = F.tree_verify(dev(lg), dev(tokens), dev(par), 1.0, dev(accept), dev(noise))
    for i in range(8):
        p, t = R.verify(lg[i], tokens[i], par[i], 1.0, accept[i], noise[i])
        assert path.cpu().tolist()[i] == p + [-1] * (3 - len(p)) and nxt.cpu().tolist()[i] == t, i
    assert F.device_error(reset=True) == 505
    flat = np.zeros((1, 2, V), np.float32)  # the draft covers the target: a refusal leaves all of it
    draft = np.full((1, 2, V), 1.0 / V, np.float32)
    one = np.array([[0, 3]], np.int32)
    path, count, nxt = F.tree_verify(dev(flat), dev(one), None, 1.0, dev(np.ones((1, 2), np.float32)), dev(noise[:1]),
                                     draft=dev(draft))
    assert count.item() == 1 and nxt.item() == int(np.argmax(1 / noise[0]))


@pytest.mark.parametrize("drawn", [False, True])
def test_verified_tokens_are_distributed_as_the_target(F, torch, drawn):
    """The first emitted token of 60000 sessions with one tree of three drafts:
    its frequencies are the target's within five standard deviations."""
    rng = np.random.default_rng(12)
    b, V = 60000, 6
    logits = np.array([1.0, 0.2, -0.5, 0.9, -2.0, 0.0], np.float32)
    p = _softmax(logits.astype(np.float64))
    q = _softmax(np.array([0.1, 1.0, 0.3, -0.4, 0.5, 0.2])).astype(np.float32)
    par = np.tile(np.array([-1, 0, 0, 0], np.int32), (b, 1))
    tokens = rng.choice(V, size=(b, 4), p=q.astype(np.float64) / q.sum(dtype=np.float64)).astype(np.int32)
    if not drawn:
        tokens[:, 1:] = [1, 3, 1]
    dev = lambda x: _dev(torch, x)  # noqa: E731
    lg = dev(np.tile(logits, (b, 4, 1)))
    path, count, nxt = F.tree_verify(lg, dev(tokens), dev(par), 1.0, dev(rng.random((b, 4)).astype(np.float32)),
                                     dev(rng.exponential(size=(b, V)).astype(np.float32) + 1e-12),
                                     draft=dev(np.tile(q, (b, 4, 1))) if drawn else None)
    path, nxt = path.cpu().numpy(), nxt.cpu().numpy()
    first = np.where(path[:, 1] > 0, tokens[np.arange(b), np.maximum(path[:, 1], 0)], nxt)
    freq = np.bincount(first, minlength=V) / b
    assert (np.abs(freq - p) <= 5 * np.sqrt(p * (1 - p) / b)).all(), (freq, p)
    assert (path[:, 1] > 0).mean() > 0.3


# ---- chains of several row tiles ----------------------------------------------------------------------------------
@pytest.mark.parametrize("b,n,hq,hk,d,s,pos", [
    (2, 300, 8, 8, 256, 600, [0, 0]), (3, 260, 15, 5, 192, 500, [0, 77, 200]), (2, 333, 8, 4, 256, 700, [1, 300])])
def test_chains_whose_blocks_hold_segments_without_tiles(F, torch, b, n, hq, hk, d, s, pos):
    """Row tiles that end before their session's last tile of tokens, cut so that
    blocks hold segments without any tile before others: in the first and third
    sixteen blocks have two of them in a row, in the second seven."""
    rng = np.random.default_rng(n)
    cache = _cache(F, torch, rng, b, s, hk, d)
    _check_attention(F, torch, rng, cache, pos, None, n, hq, gate=False)


# ---- the softmax's sum apart from the values' exponents ---------------------------------------------------------
@pytest.mark.parametrize("hq", [2, 24])  # both kernels
@pytest.mark.parametrize("e0,e1", [(66, -83), (-83, 66), (125, -98), (-98, 125), (-98, -98), (125, 125)])
def test_a_weight_counts_whatever_its_value_s_size(F, torch, hq, e0, e1):
    """Equal scores: the output is the mean of the values, though one of them is
    2^149 or 2^223 times the other."""
    rng = np.random.default_rng(21)
    d = 64
    v = rng.standard_normal((1, 4, 1, d))
    v *= (2.0 ** np.array([e0, e1, e1, e0]))[None, :, None, None]
    (kc, ke), (vc, ve) = R.quantise(np.zeros((1, 4, 1, d))), R.quantise(v)
    cache = F.Kv8Cache(*(_dev(torch, x) for x in (kc, vc, ke, ve)))
    _check_attention(F, torch, rng, cache, [1], np.array([[-1, 0, 1]], np.int32), 3, hq, gate=False)


@pytest.mark.parametrize("n,hq", [(3, 2), (3, 24)])
def test_attention_over_the_whole_range_of_exponents(F, torch, n, hq):
    """Value vectors 2^-105 to 2^124 in size over several tiles, in descending,
    ascending and random order."""
    rng = np.random.default_rng(22)
    s, d = 700, 64
    size = rng.integers(-105, 125, s)
    for order in (np.sort(size), np.sort(size)[::-1], size):
        k = rng.standard_normal((1, s, 1, d)) * 0.5
        v = rng.standard_normal((1, s, 1, d)) * (2.0 ** order)[None, :, None, None]
        (kc, ke), (vc, ve) = R.quantise(k), R.quantise(v)
        cache = F.Kv8Cache(*(_dev(torch, x) for x in (kc, vc, ke, ve)))
        _check_attention(F, torch, rng, cache, [s - n], _tree(rng, 1, n), n, hq, gate=False)


@pytest.mark.parametrize("hq", [2, 24])  # both kernels
@pytest.mark.parametrize("size", [120, -100])
def test_keys_of_any_size_against_queries_of_the_other(F, torch, hq, size):
    """Keys of about 2^120 and queries of about 2^-100, and the other way round:
    the scores are ordinary numbers, what they are made of is not."""
    rng = np.random.default_rng(28)
    s, d, n = 200, 64, 3
    k = rng.standard_normal((1, s, 1, d)) * 2.0 ** size
    v = rng.standard_normal((1, s, 1, d))
    (kc, ke), (vc, ve) = R.quantise(k), R.quantise(v)
    cache = F.Kv8Cache(*(_dev(torch, x) for x in (kc, vc, ke, ve)))
    other = -100 if size == 120 else 110
    _check_attention(F, torch, rng, cache, [s - n], _tree(rng, 1, n), n, hq, amp=2.0 ** other,
                     scale=2.0 ** -(size + other) / 8)


# ---- zero value vectors ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hq", [1, 4, 24])  # eight and sixteen rows a tile, the tcgen05 kernel
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("size", [1.0, 1e-7, 1e-20])
@pytest.mark.parametrize("zeros", [(0,), (3, 150, 151, 399), (401, 402), (70, 401), tuple(range(400))])
def test_zero_values_with_the_largest_scores(F, torch, hq, d, size, zeros):
    """Rows whose value is zero take nearly all of the weight: what the others
    give keeps its bits.  Scores: queries of ones and keys of a constant, so that
    a zero row's is 24 and another's within [0, 1].  Bars as above, the weights'
    relative to the sum that the exact weights have."""
    rng = np.random.default_rng(23)
    s, pos, n = 404, 400, 4
    a = rng.random(s)
    a[list(zeros)] = 24.0
    k = np.repeat(a[:, None], d, 1) / math.sqrt(d)
    v = rng.standard_normal((s, d)) * size
    v[list(zeros)] = rng.choice([0.0, -0.0], (len(zeros), d))
    (kc, ke), (vc, ve) = R.quantise(k), R.quantise(v)
    cache = F.Kv8Cache(*(_dev(torch, x[None, :, None]) for x in (kc, vc, ke, ve)))
    q = torch.ones(1, n, hq, d, device="cuda")
    par = np.array([[-1, 0, 1, 1]], np.int32)
    outs = [F.tree_attention(q, cache, _dev(torch, np.array([pos], np.int32)), _dev(torch, par)) for _ in range(3)]
    assert all(torch.equal(o, outs[0]) for o in outs)
    got = _host(outs[0])
    k, v = R.values(kc, ke), R.values(vc, ve)
    for j, line in enumerate(R.ancestors(par[0])):
        rows = list(range(pos)) + [pos + i for i in line]
        o, pv, sabs = R.attend(np.ones(d), k[rows], v[rows], 1 / math.sqrt(d))
        bound = (2 * 2.0 ** -11 * sabs + 2.0 ** -11 + 2.0 ** -16) * pv
        assert (np.abs(got[0, j] - o) <= bound + 2.0 ** -8 * np.abs(o)).all(), (j, got[0, j, 0, :4], o[:4])


# ---- NaN among the values -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hq", [2, 8, 48])  # both kernels
@pytest.mark.parametrize("d", [48, 64, 128, 256])
@pytest.mark.parametrize("tree", [True, False])
def test_a_nan_code_reaches_its_column_alone(F, torch, hq, d, tree):
    """A NaN among the codes of a value makes that column NaN for the nodes that
    see its row, in the context as in the tree, and nothing else."""
    rng = np.random.default_rng(24)
    s, pos, n, hk = 300, 290, 4, 2
    clean = _cache(F, torch, rng, 1, s, hk, d)
    dirty = F.Kv8Cache(*(getattr(clean, x).clone() for x in ("k", "v", "k_exp", "v_exp")))
    par = np.array([[-1, 0, 0, 1]], np.int32) if tree else None
    lines = _lines(par, 1, n)[0]
    at = [(7, 3), (7, 17), (289, 0), (pos + 1, 5), (pos + 1, d - 1), (pos + 2, 31), (pos + 3, 14)]
    want = np.zeros((n, d), bool)
    for row, col in at:
        dirty.v[0, row, 1, col] = 0x7f if col % 2 else 0xff
        for j in range(n):
            want[j, col] |= row < pos or row - pos in lines[j]
    q = _dev(torch, rng.standard_normal((1, n, hq, d)).astype(np.float32))
    where, par = _dev(torch, np.array([pos], np.int32)), None if par is None else _dev(torch, par)
    a, b = (F.tree_attention(q, c, where, par)[0] for c in (clean, dirty))
    nan = torch.isnan(b).cpu().numpy()
    assert not nan[:, :hq // 2].any() and torch.equal(a[:, :hq // 2], b[:, :hq // 2])
    for h in range(hq // 2, hq):
        assert np.array_equal(nan[:, h], want), h
    # elsewhere the outputs are the clean ones, but for the codes that a NaN has replaced
    assert torch.equal(torch.where(torch.isnan(b), 0.0, b), torch.where(torch.isnan(b), 0.0, a))


# ---- absent nodes ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_append_of_absent_nodes_gives_zeros_at_any_eps(F, torch, eps):
    rng = np.random.default_rng(25)
    d = 64
    q, k = (_dev(torch, rng.standard_normal((1, 4, 2, d)).astype(np.float32)) for _ in range(2))
    ones = torch.ones(d, device="cuda")
    cache = F.Kv8Cache.zeros(1, 8, 2, d)
    got = F.kv8_append(cache, torch.zeros(1, dtype=torch.int32, device="cuda"), k, k, q=q,
                       parents=_dev(torch, np.array([[-1, -2, 0, 1]], np.int32)), q_gamma=ones, k_gamma=ones, eps=eps,
                       rotary_dim=32)
    assert not got[0, [1, 3]].any() and torch.isfinite(got).all() and (got[0, [0, 2]] != 0).any(-1).all()
    assert not cache.k[0, [1, 3]].any() and cache.k[0, [0, 2]].any()


@pytest.mark.parametrize("hq", [2, 24])  # both kernels
def test_absent_nodes_past_the_cache_are_no_error(F, torch, hq):
    """Only a node that is there can lie outside the cache: the slots that a tree
    leaves empty at the end of its cache, and a session without a tree at any
    position, record nothing."""
    rng = np.random.default_rng(26)
    s, n, d = 40, 4, 32
    cache = _cache(F, torch, rng, 3, s, 1, d)
    par = np.array([[-1, 0, -2, -2], [-2, -2, -2, -2], [-1, 0, 1, 2]], np.int32)
    got = _check_attention(F, torch, rng, cache, [s - 2, 7, s - n], par, n, hq)
    assert got[0, :2].any(-1).all() and F.device_error(reset=True) == 0
    q = _dev(torch, rng.standard_normal((3, n, hq, d)).astype(np.float32))
    out = F.tree_attention(q, cache, _dev(torch, np.array([s - 2, -5, s - n], np.int32)), _dev(torch, par))
    assert not out[1].any() and F.device_error(reset=True) == 0
    par[0, 2] = 0  # node 2 is there now, and outside
    out = F.tree_attention(q, cache, _dev(torch, np.array([s - 2, 7, s - n], np.int32)), _dev(torch, par))
    assert out[0, :2].any() and not out[0, 2:].any() and F.device_error(reset=True) == 502


def test_wrappers_refuse_tensors_of_another_device(F, torch):
    """One argument at a time on the host, the others on the GPU: refused before
    anything is launched."""
    cache = F.Kv8Cache.zeros(2, 32, 2, 64)
    z = dict(device="cuda")
    pos, par = torch.zeros(2, dtype=torch.int32, **z), torch.zeros(2, 4, dtype=torch.int32, **z)
    q, kv, ones = torch.zeros(2, 4, 6, 64, **z), torch.zeros(2, 4, 2, 64, **z), torch.ones(64, **z)
    lg, unit = torch.zeros(2, 4, 10, **z), torch.ones(2, 10, **z)
    ws = torch.zeros(F.tree_attention_workspace_bytes(cache, 4, 6), dtype=torch.uint8, **z)
    calls = [
        (F.kv8_append, dict(positions=pos, k=kv, v=kv, q=q, parents=par, q_gamma=ones, k_gamma=ones, q_out=q.clone())),
        (F.kv8_read, dict(begin=pos, count=4)),
        (F.kv8_keep, dict(positions=pos, path=par)),
        (F.tree_attention, dict(q=q, positions=pos, parents=par, gate=q, out=q.bfloat16(), workspace=ws)),
        (F.tree_verify, dict(logits=lg, tokens=par, parents=par, accept=lg[..., 0].contiguous(), noise=unit, draft=lg)),
    ]
    launches = F.launch_count()
    for call, args in calls:
        own = dict(temperature=1.0) if call is F.tree_verify else dict(cache=cache)
        for name, t in args.items():
            if torch.is_tensor(t):
                with pytest.raises(F.ShapeError, match="cpu"):
                    call(**own, **dict(args, **{name: t.cpu()}))
                    pytest.fail(f"{call.__name__}: {name} was taken")
    assert F.launch_count() == launches


# ---- offsets past 32 bits -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hq", [4, 40])  # both kernels
def test_attention_and_moves_past_32_bits(F, torch, hq):
    """The last session of a cache of over 2^32 codes, its rows at the end: the
    own row's score is large and positive, so that the output is that row's value;
    then a path that moves rows there."""
    b, s, hk, d = 5, 1 << 21, 2, 256
    cache = F.Kv8Cache.zeros(b, s, hk, d)
    rng = np.random.default_rng(27)
    pos = np.array([3, 0, 0, 0, s - 300], np.int32)
    kv = _dev(torch, rng.standard_normal((b, 3, 2, hk, d)).astype(np.float32))
    k, v = kv[:, :, 0], kv[:, :, 1]
    par = _dev(torch, np.array([[-1, 0, 0]] * b, np.int32))
    where = _dev(torch, pos)
    F.kv8_append(cache, where, k, v, parents=par)
    held_k, held_v = F.kv8_read(cache, where, 3)
    # zero keys score 0, the own one 20 |k|^2 / 16 of about 300, another node's some 80 at most beside it
    q = 20.0 * k.repeat_interleave(hq // hk, 2)
    score = torch.einsum("bihd,bjhd->bhij", q, held_k.repeat_interleave(hq // hk, 2)) / 16
    own = score.diagonal(dim1=2, dim2=3)
    assert float(own.min()) > 60 + float((score - torch.diag_embed(own)).max())
    out = F.tree_attention(q, cache, where, par).float()
    want = held_v.repeat_interleave(hq // hk, 2)
    # the other weights are below 2^21 e^-60, the own one is 1 but for its own f16's 2^-11 and bf16's 2^-8
    assert bool(((out - want).abs() <= (2.0 ** -11 + 2.0 ** -8) * want.abs() + 1e-12).all())
    before = {x: getattr(cache, x)[4, s - 300:s - 296].clone() for x in ("k", "v", "k_exp", "v_exp")}
    F.kv8_keep(cache, where, _dev(torch, np.array([[0, 2, -1]] * b, np.int32)))
    for x, old in before.items():
        now = getattr(cache, x)[4, s - 300:s - 296]
        assert torch.equal(now[[0, 2, 3]], old[[0, 2, 3]]) and torch.equal(now[1], old[2]), x
        assert x.endswith("exp") or not torch.equal(old[1], old[2])
    del cache
