"""Attention over the paged cache where numbers leave the usual range: infinite keys,
values and queries, values from the smallest normal number to the largest, against the
formula in 64 bits.

NaN stays where it is seen.  What the formula gives for infinities: a score of -inf a
weight of 0 (with no other, zeros, as without tokens), one of +inf NaN in the whole
head, an infinite value its column (NaN where both signs meet), however small its
token's weight.  Finite numbers have test_gpu_paged.py's bars, taken over the finite
terms, and n * 2^-148 for sums and products below the normal range (each is off by
2^-149 at most).
"""
import math

import numpy as np
import pytest

from test_gpu_paged import F, _attention_case, _dev, _host, _no_device_error, torch  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu

KINDS = ("key -inf", "key +inf", "value", "query", "hopeless", "nan", "masked", "plain", "columns", "small", "large", "sparse")


def _special(torch, kind, rng, i, n, q, k, v, scale):
    """What is out of the ordinary in session i; k, v [n, heads, d] and q [heads, d] are
    f32 copies on the host, in place."""
    d = q.shape[1]
    if kind == "key -inf":
        q[:, 3], q[:, d - 1] = np.abs(q[:, 3]) + 0.125, -np.abs(q[:, d - 1]) - 0.37
        for t in {0, n // 2, n - 1}:
            if n > 1 and t != 1:
                k[t, :, 3] = -math.inf
        if n > 6:
            k[5, :, d - 1] = math.inf
    elif kind == "key +inf":
        q[:, 2] = np.abs(q[:, 2]) + 0.125
        k[n // 3, 0, 2] = math.inf
    elif kind == "value":
        v[n // 2, 0, 5], v[0, 0, 7], v[n - 1, 0, 7] = math.inf, -math.inf, -math.inf
        v[n // 2, 0, 9] = math.inf
        v[(n // 2 + 1) % n, 0, 9] = -math.inf if n > 1 else math.inf
    elif kind == "query":
        q[1, 4] = math.inf
        k[n // 2, :, 4] = np.abs(k[n // 2, :, 4]) + 0.1
    elif kind == "hopeless":
        q[:, 6] = 8.0
        k[:, :, 6] = 0.0
        k[n // 2, :, 6] = -200.0 / (8.0 * scale) if n > 1 else 0.0
        v[n // 2, :, 1] = -math.inf
    elif kind == "nan":
        v[0, 0, 5], v[n // 2, 0, 6], q[1, 2] = math.nan, math.inf, math.nan
    elif kind == "masked":
        q[:, 1] = np.abs(q[:, 1]) + 0.125
        k[:, :, 1] = -math.inf
    elif kind == "columns":
        v *= 2.0 ** np.linspace(-120, 120, d).round().astype(np.float32)
    elif kind == "small":
        v *= np.float32(2.0 ** -118)
    elif kind == "sparse":  # columns of a few tokens each, most of them of next to no weight
        at = np.arange(n)
        q[:, 6] = 2.0
        k[:, :, 6] = -(37.5 / scale * (at % d) / d)[:, None]
        v *= (at[:, None] % d == np.arange(d))[:, None, :]
    elif kind == "large":
        v *= np.float32(2.0 ** 122)


def _want(q, k, v, scale):
    """(output, sum of p |v| over finite values, largest sum of |q k| scale of a finite score)."""
    with np.errstate(invalid="ignore", over="ignore"):
        s = (k @ q) * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out = np.array([(p * col)[(p != 0) | ~np.isfinite(col) | np.isnan(p)].sum() for col in v.T])
        fine = np.isfinite(s)
        most = float((np.abs(k[fine]) @ np.abs(q)).max() * scale) if fine.any() else 0.0
        return out, np.nan_to_num(p) @ np.where(np.isfinite(v), np.abs(v), 0.0), most


@pytest.mark.parametrize("pages", ["f32", "bf16"])
@pytest.mark.parametrize("n,hq,hk,d,p,times,dtype", [
    (40, 8, 2, 64, 16, 1, "f32"), (1, 4, 2, 64, 8, 1, "f32"), (3001, 4, 2, 128, 16, 1, "f32"),
    (1500, 32, 2, 128, 32, 1, "f32"), (700, 4, 1, 256, 16, 1, "bf16"), (333, 16, 1, 256, 64, 1, "f32"),
    (90, 6, 2, 80, 24, 1, "f32"), (450, 8, 8, 64, 7, 5, "f32"), (130, 20, 2, 192, 16, 9, "bf16")])
def test_paged_attention_values_out_of_the_ordinary(F, torch, n, hq, hk, d, p, times, dtype, pages):
    """Sessions of each kind beside one another, whole and in shares, in one wave of
    blocks and (many sessions) in several."""
    torch.manual_seed(n + d)
    rng = np.random.default_rng(n + d)
    b = len(KINDS) * times
    lengths = [max(1, n - 3 * (i % 4)) for i in range(b)]
    q, gate, cache, table, lens = _attention_case(F, torch, rng, lengths, hq, hk, d, p, dtype, pages)
    scale = d ** -0.5
    host, tab = [], table.cpu().long()
    for i, m in enumerate(lengths):
        ids = tab[i, :-(-m // p)].cuda()
        qi = q[i].float().cpu().numpy()
        ki, vi = (t[ids].float().cpu().numpy().reshape(-1, hk, d)[:m] for t in (cache.k, cache.v))
        _special(torch, KINDS[i % len(KINDS)], rng, i, m, qi, ki, vi, scale)
        rows = torch.arange(m, device="cuda")
        for t, x in ((cache.k, ki), (cache.v, vi)):
            t.view(-1, hk, d)[ids[rows // p] * p + rows % p] = _dev(torch, x).to(t.dtype)
        q[i] = _dev(torch, qi).to(q.dtype)
        host.append((_host(q[i]), *(_host(t[ids]).reshape(-1, hk, d)[:m] for t in (cache.k, cache.v))))
    out = torch.full(q.shape, 7.0, device="cuda")
    assert F.paged_attention(q, cache, table, lens, gate=gate, out=out) is out
    if dtype == "f32":  # in the queries' place
        mine = q.clone()
        assert F.paged_attention(mine, cache, table, lens, gate=gate, out=mine) is mine
        assert torch.equal(torch.nan_to_num(mine), torch.nan_to_num(out))
    again = F.paged_attention(q, cache, table, lens, gate=gate)
    assert torch.equal(torch.nan_to_num(again), torch.nan_to_num(out.to(again.dtype)))
    got, g = _host(out), 1.0 / (1.0 + np.exp(-_host(gate)))
    two = 2.0 ** -16 if pages == "bf16" else 0.0
    for i, (qi, ki, vi) in enumerate(host):
        kind = KINDS[i % len(KINDS)]
        if kind == "masked":
            assert not got[i].any()
            continue
        for h in range(hq):
            want, pv, most = _want(qi[h], ki[:, h // (hq // hk)], vi[:, h // (hq // hk)], scale)
            where = (kind, i, h)
            with np.errstate(invalid="ignore"):
                ds = most * ((d + 4) * 2.0 ** -24 + two)
                bar = (2 * ds + 2.0 ** -20 + (lengths[i] + 64) * 2.0 ** -23 + 2 * two) * pv + lengths[i] * 2.0 ** -148
                want, bar = want * g[i, h], bar * g[i, h] + 2.0 ** -148
                bar = bar + np.abs(want) * (2.0 ** -24 + 2.0 ** -21)
                fine = np.isfinite(want)
                assert (np.isnan(got[i, h]) == np.isnan(want)).all(), where
                inf = np.isinf(want)
                assert (got[i, h][inf] == want[inf]).all(), where
                off = np.abs(got[i, h] - want)[fine] / bar[fine]
                assert (off <= 1).all(), (*where, float(np.nanmax(off)))
        if kind == "key +inf":
            assert np.isnan(got[i, :hq // hk]).all()
        elif kind in ("key -inf", "plain", "columns", "small", "large"):
            if kind != "key -inf" or lengths[i] > 3:
                assert np.isfinite(got[i]).all() and (kind != "small" or (got[i] != 0).all())


@pytest.mark.parametrize("hq,hk", [(8, 8), (64, 8), (64, 4)])
def test_paged_attention_f32_queries_keep_their_bits(F, torch, hq, hk):
    """f32 queries over bf16 pages: bits of the queries and of the weights that only a
    third part of 8 holds.

    First two tokens whose scores 2^20 + 2^11 differ by 1 through elements 1 + 2^-9 +
    2^-20: f32 scores in powers of two are off by 2^-4 at most each, so the first
    token's weight 1 / (1 + e^-1) lies within [0.71, 0.75]; without that bit it is a half.
    Then weights p = e^-x of one element against 1, values 1 and -c with c the bf16 number
    nearest to p: (p - c) / (1 + p) is off by p (2^-23 of the power's argument, 2^-22 of the
    power) and 2^-22 of the sums, below 2^-20; two parts leave up to 2^-18 of p."""
    d, heads = 256, hq // hk
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    n = torch.full((1,), 2, dtype=torch.int32, device="cuda")
    cache = F.PagedCache.zeros(1, 16, hk, d)
    q = torch.full((1, hq, d), 1 + 2.0 ** -9, device="cuda")
    q[..., :d // 2] += 2.0 ** -20
    cache.k[0, 0, :, :d // 2], cache.k[0, 1, :, d // 2:] = 8192.0, 8192.0
    cache.v[0, 0] = 1.0
    out = F.paged_attention(q, cache, table, n, scale=1.0, out=torch.empty_like(q))
    assert 0.71 <= float(out.min()) and float(out.max()) <= 0.75
    rng = np.random.default_rng(hq + hk)
    x = np.float32(rng.uniform(0.01, 1.3, hq))
    q.zero_()
    q[0, :, 0] = -_dev(torch, x)
    cache.k.zero_()
    cache.k[0, 0, :, 0] = 1.0
    p = np.exp(-x.astype(np.float64))
    c = _host(_dev(torch, p.astype(np.float32)).bfloat16())
    cache.v.zero_()
    cache.v[0, 0, :, :heads] = 1.0
    cache.v[0, 1, :, :heads] = -_dev(torch, c.astype(np.float32)).bfloat16().view(hk, heads)
    out = _host(F.paged_attention(q, cache, table, n, scale=1.0, out=torch.empty_like(q)))[0]
    got = out[np.arange(hq), np.arange(hq) % heads]
    assert np.abs(got - (p - c) / (1 + p)).max() <= 2.0 ** -20


def test_paged_attention_outputs_beside_the_inputs(F, torch):
    """Next to the queries and the gate, and between their rows."""
    torch.manual_seed(7)
    rng = np.random.default_rng(7)
    q, gate, cache, table, n = _attention_case(F, torch, rng, [40, 70], 4, 2, 64, 16, "f32", "f32")
    want = F.paged_attention(q, cache, table, n, gate=gate)
    both = torch.zeros(4, 4, 64, device="cuda")
    both[:2] = q
    assert torch.equal(F.paged_attention(both[:2], cache, table, n, gate=gate, out=both[2:]), want)
    wide = torch.zeros(2, 4096, device="cuda")
    mine, g, out = wide[:, :256].unflatten(1, (4, 64)), wide[:, 256:512].unflatten(1, (4, 64)), wide[0, 512:1024].view(2, 4, 64)
    mine.copy_(q)
    g.copy_(gate)
    assert torch.equal(F.paged_attention(mine, cache, table, n, gate=g, out=out), want)
    for bad in (wide[0, 128:640], wide[0, 256:768], wide.view(-1)[3840:4352]):
        with pytest.raises(F.FpbError):
            F.paged_attention(mine, cache, table, n, gate=g, out=bad.view(2, 4, 64))
