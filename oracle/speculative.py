"""numpy restatement in 64 bits of speculative decoding over the 8-bit cache:
the checker of firepit_b200's append, attention and verification kernels.

TEST INFRASTRUCTURE ONLY: the product never imports it.
"""
from __future__ import annotations

import math

import numpy as np

# the 256 e4m3 values, from the format: sign, 4 exponent bits (bias 7), 3 mantissa bits, no infinities
E4M3 = np.array([math.nan if (c & 0x7f) == 0x7f else
                 (-1.0) ** (c >> 7) * (((c & 7) / 8 * 2.0 ** -6) if (c >> 3 & 15) == 0
                                       else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3 & 15) - 7)) for c in range(256)])
_POS = E4M3[:127]  # 0 .. 448, ascending


def values(codes, exps):
    """What codes [..., d] and exponent bytes [...] stand for."""
    return E4M3[codes] * 2.0 ** (exps.astype(np.int64) - 127)[..., None]


def exponent(amax):
    """Smallest e with amax <= 448 * 2^e, within [-100, 120]; -8 for zero."""
    out = np.full(np.shape(amax), -8, np.int64)
    for i in np.ndindex(*np.shape(amax)):
        a = float(amax[i])
        if a > 0:
            e = math.floor(math.log2(a)) - 12
            while e < 200 and a > 448.0 * 2.0 ** e:
                e += 1
            out[i] = min(120, max(-100, e))
    return out


def quantise(x):
    """(codes, exponent bytes) of head vectors x [..., d]: nearest e4m3 value,
    the even code among two as near."""
    x = np.asarray(x, np.float64)
    e = exponent(np.abs(x).max(-1))
    y = np.minimum(np.abs(x) / 2.0 ** e[..., None], 448.0)
    hi = np.clip(np.searchsorted(_POS, y), 1, 126)
    lo = hi - 1
    dl, dh = y - _POS[lo], _POS[hi] - y
    code = np.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, lo)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8), (e + 127).astype(np.uint8)


def ancestors(parents):
    """Each node's line from node 0 to itself, or None where it is not there."""
    line = []
    for i, p in enumerate(parents):
        if i == 0:
            line.append([0] if p == -1 else None)
        else:
            line.append(line[p] + [i] if 0 <= p < i and line[p] is not None else None)
    return line


def norm_rotate(x, gamma, eps, pos, rotary, theta):
    """RMSNorm (gamma None: none) and rotation of head vectors x [..., d] at one position."""
    x = np.asarray(x, np.float64)
    if gamma is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(gamma, np.float64)
    half = rotary // 2
    out = x.copy()
    if half:
        ang = pos * float(theta) ** (-np.arange(half) / half)
        c, s = np.cos(ang), np.sin(ang)
        out[..., :half] = x[..., :half] * c - x[..., half:rotary] * s
        out[..., half:rotary] = x[..., half:rotary] * c + x[..., :half] * s
    return out


def attend(q, k, v, scale):
    """One query q [d] over the visible rows k, v [t, d]: (output, sum of p
    |v|, largest sum of |q_i k_i| * scale), the latter two for error bounds."""
    s = (k @ q) * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ v, p @ np.abs(v), float((np.abs(k) @ np.abs(q)).max() * abs(scale))


def verify(logits, tokens, parents, temperature, accept=None, noise=None, draft=None):
    """(path, next) of one session's walk."""
    if parents[0] != -1:
        return [], -1
    n = len(tokens)
    vocab = logits.shape[-1]
    path, node = [0], 0
    while True:
        row = np.where(np.isfinite(logits[node]), logits[node].astype(np.float64), -np.inf)
        child = None
        if temperature == 0:
            best = int(np.argmax(row))
            for c in range(node + 1, n):
                if parents[c] == node and tokens[c] == best:
                    child = c
                    break
            if child is None:
                return path, best
        else:
            r = np.exp((row - row.max()) / np.float64(np.float32(temperature))) if np.isfinite(row.max()) else row * 0
            r = r / r.sum()
            for c in range(node + 1, n):
                x = tokens[c]
                if parents[c] != node or not 0 <= x < vocab:
                    continue
                qx = 1.0 if draft is None else float(draft[node, x])
                if float(accept[c]) * qx < r[x]:
                    child = c
                    break
                left = r.copy()
                if draft is None:
                    left[x] = 0.0
                else:
                    left = np.maximum(r - draft[node].astype(np.float64), 0.0)
                if left.sum() > 0:
                    r = left / left.sum()
            if child is None:
                return path, int(np.argmax(r / noise.astype(np.float64)))
        path.append(child)
        node = child
