"""The speculative-decoding operators over an 8-bit key/value cache: what is measured.

Four operators, each in its plain form (elementary torch operations in 32 bits) and through the framework's entry
points:

  append   head norms of q and k, rotation by position, and the new tokens' keys and values quantised into the cache;
           the rows just written are read back
  read     a range of the cache as the values that it stands for
  attend   attention of a tree of drafted tokens (one node: plain decoding) over the cache
  verify   the drafted tokens against the target's probabilities, from given random numbers

The cache holds e4m3 codes [batch, max_seq, kv_heads, head_dim] and one exponent byte for each head vector: a value is
code * 2^(byte - 127), and the exponent is the smallest one with amax <= 448 * 2^e (held within [-100, 120]; -8 for a
vector of zeros).  A tree is `parents` [batch, nodes]: -1 for node 0, an earlier node for the others, -2 for a node
that is not there.  Node i lies in cache row position + i and is rotated by position + depth(i); it sees the rows
before `position`, its ancestors and itself.
"""
import math

import torch

own = False

VOCAB = 151936  # the hybrid decoder's vocabulary


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    def append(name, **kw):
        return dict(dict(name=name, op="append", eps=1e-6), **kw)

    def attend(name, **kw):
        return dict(dict(name=name, op="attend"), **kw)

    def verify(name, **kw):
        return dict(dict(name=name, op="verify", vocab=VOCAB), **kw)

    return [
        # one decode step of eight sessions at the hybrid decoder's attention heads: latency alone
        append("append 8x1", batch=8, nodes=1, tree=False, q_heads=16, kv_heads=2, head_dim=256, rotary_dim=64,
               context=511, dtype="f32"),
        # a step that verifies 24 drafted tokens of 16 sessions
        append("append 16x24 tree", batch=16, nodes=24, tree=True, q_heads=16, kv_heads=2, head_dim=256,
               rotary_dim=64, context=2000, dtype="f32"),
        # two prompts written at once, bf16 projections, every dimension rotated
        append("append 2x4096 prompt", batch=2, nodes=4096, tree=False, q_heads=32, kv_heads=8, head_dim=128,
               rotary_dim=128, context=333, dtype="bf16"),
        # a short, odd range of one session in f32, as a check or a host copy reads it
        dict(name="read 1x1501", op="read", batch=1, rows=1501, kv_heads=3, head_dim=80, context=1700, dtype="f32"),
        # eight sessions' caches handed to a path that wants bf16
        dict(name="read 8x8192", op="read", batch=8, rows=8192, kv_heads=2, head_dim=256, context=8192, dtype="bf16"),
        # the smallest call: one session, one token, a context that ends inside a tile
        attend("attend 1x1 at 1000", batch=1, nodes=1, q_heads=8, kv_heads=2, head_dim=128, context=1000, dtype="f32"),
        # plain decoding of sixteen sessions over the 8-bit cache: bound by the cache's bytes
        attend("attend 16x1 at 8192", batch=16, nodes=1, q_heads=16, kv_heads=2, head_dim=256, context=8192,
               dtype="f32"),
        # sixteen drafted tokens of eight sessions: the group's eight heads make 128 rows a key/value head
        attend("attend 8x16 at 16384", batch=8, nodes=16, q_heads=16, kv_heads=2, head_dim=256, context=16384,
               dtype="f32"),
        # a large, odd tree over long odd contexts: bound by the products
        attend("attend 4x61 at 30011", batch=4, nodes=61, q_heads=32, kv_heads=4, head_dim=128, context=30011,
               dtype="bf16"),
        # greedy verification of a short chain of two sessions
        verify("verify 2x5 greedy", batch=2, nodes=5, tree=False, temperature=0.0, draft=False, dtype="f32"),
        # trees of drafts that are certain (look-up or top-k drafts), sampled target
        verify("verify 8x32 tree", batch=8, nodes=32, tree=True, temperature=0.8, draft=False, dtype="f32"),
        # trees of drafts drawn from a draft model's probabilities
        verify("verify 16x9 drawn", batch=16, nodes=9, tree=True, temperature=1.0, draft=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "verify"])
    dtype = rng.choice(["f32", "bf16"])
    head_dim = rng.choice([64, 80, 96, 128, 192, 256])
    kv_heads = rng.randint(1, 8)
    group = rng.choice([1, 2, 3, 4, 6, 8, 16])
    if op == "append":
        prompt = rng.random() < 0.4
        batch = _log(rng, 1, 4 if prompt else 32)
        nodes = _log(rng, 64, 2048) if prompt else _log(rng, 1, 64)
        return dict(op=op, eps=1e-6, batch=batch, nodes=nodes, tree=not prompt and rng.random() < 0.7,
                    q_heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                    rotary_dim=rng.choice([0, 32, 64, head_dim]), context=_log(rng, 1, 8192), dtype=dtype)
    if op == "read":
        rows = _log(rng, 1, 8192)
        return dict(op=op, batch=_log(rng, 1, 8), rows=rows, kv_heads=min(kv_heads, 2), head_dim=head_dim,
                    context=rows + rng.randint(0, 500), dtype=dtype)
    if op == "attend":
        while True:
            case = dict(op=op, batch=_log(rng, 1, 32), nodes=_log(rng, 1, 64), q_heads=kv_heads * group,
                        kv_heads=kv_heads, head_dim=head_dim, context=_log(rng, 1, 32768), dtype=dtype)
            w = work(case)
            if all(w[k] <= max(work(c)[k] for c in listed() if c["op"] == op) for k in w):
                return case
            kv_heads, group = rng.randint(1, 8), rng.choice([1, 2, 3, 4, 6, 8, 16])
    batch = _log(rng, 1, 16)
    return dict(op=op, batch=batch, nodes=_log(rng, 1, min(64, 256 // batch)), vocab=_log(rng, 1000, 160000),
                tree=rng.random() < 0.6, temperature=rng.choice([0.0, 0.6, 1.0]), draft=rng.random() < 0.5,
                dtype=dtype)


# ---- inputs --------------------------------------------------------------------------------------------------------
def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _positions(case):
    """Tokens of each session before node 0: sessions of different lengths, the first the longest."""
    c, b = case["context"], case["batch"]
    return [c - (i * c) // (4 * b) for i in range(b)]


def _present(case):
    """Nodes of each session's tree (the first session's is whole)."""
    n, b = case["nodes"], case["batch"]
    return [n - (i * n) // (3 * b) for i in range(b)]


def _parents(case, rnd):
    """Trees that mix long branches with forks; a session's missing nodes are -2."""
    rows = []
    for count in _present(case):
        draws = torch.rand(case["nodes"], 2, generator=rnd).tolist()
        row = [-1]
        for i in range(1, case["nodes"]):
            r, s = draws[i]
            row.append(-2 if i >= count else i - 1 if r < 0.5 else max(0, i - 1 - int(s * min(i, 8))))
        rows.append(row)
    return torch.tensor(rows, dtype=torch.int32)


def _pow2(e):
    """2^e for whole e within [-126, 127], from its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x):
    """e4m3 codes and exponent bytes of head vectors x [..., head_dim] in f32."""
    amax = x.abs().amax(-1)
    frac, n = torch.frexp(amax)
    e = (n - torch.where(frac <= 0.875, 9, 8)).clamp(-100, 120)
    e = torch.where(amax > 0, e, -8)
    codes = (x * _pow2(-e)[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8)


def _values(codes, exps):
    return codes.view(torch.float8_e4m3fn).float() * _pow2(exps.int() - 127)[..., None]


def prepare(case, seed):
    rnd = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=dev, device="cuda") * std

    st = dict(case=case)
    b = case["batch"]
    if case["op"] == "verify":
        return _prepare_verify(case, st, rnd, dev)
    hk, d = case["kv_heads"], case["head_dim"]
    n = case.get("nodes", 0)
    st["max_seq"] = s = case["context"] + n
    st["positions"] = torch.tensor(_positions(case), dtype=torch.int32).cuda()
    if case["op"] == "append":
        hq = case["q_heads"]
        # the projections' outputs: per query head its query, then its gate, as the decoder's w_qg gives them
        st["qg"] = normal(b, n, hq, 2 * d).to(_dtype(case))
        st["q"] = st["qg"][..., :d]
        st["k"] = normal(b, n, hk, d, std=2.0).to(_dtype(case))
        st["v"] = normal(b, n, hk, d, std=0.7).to(_dtype(case))
        st["q_gamma"] = 1.0 + normal(d, std=0.1)
        st["k_gamma"] = 1.0 + normal(d, std=0.1)
        st["parents"] = _parents(case, rnd).cuda() if case["tree"] else None
        for name in ("k_codes", "v_codes"):
            st[name] = torch.zeros(b, s, hk, d, dtype=torch.uint8, device="cuda")
        for name in ("k_exp", "v_exp"):
            st[name] = torch.full((b, s, hk), 119, dtype=torch.uint8, device="cuda")
        return st
    # normed and rotated keys have vectors of about sqrt(head_dim); values differ in size from token to token
    st["k_codes"], st["k_exp"] = _quantise(normal(b, s, hk, d, std=1.3))
    st["v_codes"], st["v_exp"] = _quantise(normal(b, s, hk, d) * torch.exp(normal(b, s, hk, 1, std=0.5)))
    if case["op"] == "read":
        st["begin"] = torch.tensor([p - p * case["rows"] // case["context"] for p in _positions(case)],
                                   dtype=torch.int32).cuda()
        return st
    hq = case["q_heads"]
    st["q"] = normal(b, n, hq, d, std=1.6).to(_dtype(case))
    st["gate"] = normal(b, n, hq, d)
    st["parents"] = _parents(case, rnd).cuda()
    return st


def _prepare_verify(case, st, rnd, dev):
    b, n, vocab, t = case["batch"], case["nodes"], case["vocab"], case["temperature"]
    logits = (torch.randn(b, n, vocab, generator=dev, device="cuda") * 2.5).to(_dtype(case))
    parents = _parents(case, rnd) if case["tree"] else torch.arange(-1, n - 1, dtype=torch.int32).repeat(b, 1)
    st["logits"], st["parents"] = logits, parents.cuda() if case["tree"] else None
    st["branch"] = max([row.count(p) for row in parents.tolist() for p in row if p >= 0], default=0)  # children, at most
    up = parents.clamp(min=0).long().cuda()
    rows = logits.float()
    of_parent = torch.gather(rows, 1, up[..., None].expand(b, n, vocab))  # the logits that each node is judged by
    if case["draft"]:
        # the draft model: the target's logits with an error, and its children drawn from it
        err = torch.randn(b, n, vocab, generator=dev, device="cuda")
        st["draft"] = torch.softmax((rows + 0.4 * err) / max(t, 0.5), -1)
        q = torch.gather(st["draft"], 1, up[..., None].expand(b, n, vocab))
    else:
        st["draft"] = None
        q = torch.softmax(of_parent / max(t, 0.5), -1)  # drafts that the target finds likely
    e = -torch.log(torch.rand(b, n, vocab, generator=dev, device="cuda").clamp_min(1e-30))
    drawn = torch.argmax(q / e, -1)
    likely = of_parent.argmax(-1)
    keep = torch.rand(b, n, generator=rnd).cuda() < (0.75 if t == 0.0 else 0.4)
    st["tokens"] = torch.where(keep & (not case["draft"]), likely, drawn).int()
    st["accept"] = torch.rand(b, n, generator=dev, device="cuda")
    st["noise"] = -torch.log(torch.rand(b, vocab, generator=dev, device="cuda").clamp(1e-30, 1 - 1e-7))
    return st


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _tree(parents, b, n):
    """(sees [b, n, n]: node i sees node j, present [b, n], depth [b, n]); parents None: a chain."""
    at = torch.arange(n, device="cuda")
    if parents is None:
        sees = (at[:, None] >= at[None, :]).expand(b, n, n)
    else:
        reach = (parents[..., None] == at).float() + torch.eye(n, device="cuda")
        for _ in range(max(1, (n - 1).bit_length())):  # paths of twice the length each time
            reach = (reach @ reach).clamp(max=1.0)
        sees = reach > 0
        present = sees[..., 0] & (parents[:, :1] == -1)  # the root is among its ancestors
        sees = sees & present[..., None]
    present = sees.diagonal(dim1=1, dim2=2)
    return sees, present, sees.sum(-1) - 1


def _rotate(x, pos, rotary):
    """Rotation of the first `rotary` dimensions, halves as pairs; the angles in 64 bits: 32 lose them at long
    positions."""
    if not rotary:
        return x
    half = rotary // 2
    freq = 1.0e7 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    ang = pos.double()[..., None, None] * freq
    c, s = ang.cos().float(), ang.sin().float()
    x0, x1 = x[..., :half], x[..., half:rotary]
    return torch.cat([x0 * c - x1 * s, x1 * c + x0 * s, x[..., rotary:]], -1)


def _plain_append(st):
    c = st["case"]
    b, n = c["batch"], c["nodes"]
    _, present, depth = _tree(st["parents"], b, n)
    pos = st["positions"][:, None] + depth

    def normed(x, gamma):
        x = x.float()
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + c["eps"]) * gamma

    q = _rotate(normed(st["q"], st["q_gamma"]), pos, c["rotary_dim"])
    k = _rotate(normed(st["k"], st["k_gamma"]), pos, c["rotary_dim"])
    q = torch.where(present[..., None, None], q, 0.0)
    rows = st["positions"].long()[:, None] + torch.arange(n, device="cuda")
    bi, ni = torch.nonzero(present, as_tuple=True)
    for codes, exps, x in ((st["k_codes"], st["k_exp"], k), (st["v_codes"], st["v_exp"], st["v"].float())):
        cx, ex = _quantise(x)
        codes[bi, rows[bi, ni]] = cx[bi, ni]
        exps[bi, rows[bi, ni]] = ex[bi, ni]
    return {"q": q.to(_dtype(c)), **_plain_read(st, st["positions"], n, torch.bfloat16)}


def _plain_read(st, begin, rows, dtype):
    at = begin.long()[:, None] + torch.arange(rows, device="cuda")
    bi = torch.arange(at.shape[0], device="cuda")[:, None]
    return {"k": _values(st["k_codes"][bi, at], st["k_exp"][bi, at]).to(dtype),
            "v": _values(st["v_codes"][bi, at], st["v_exp"][bi, at]).to(dtype)}


def _plain_attend(st):
    c = st["case"]
    b, n, hq, hk, d, s = c["batch"], c["nodes"], c["q_heads"], c["kv_heads"], c["head_dim"], st["max_seq"]
    sees, present, _ = _tree(st["parents"], b, n)
    pos = st["positions"].long()
    t = torch.arange(s, device="cuda")
    node = t[None, :] - pos[:, None]  # the tree node that a cache row holds, if any
    in_tree = (node >= 0) & (node < n)
    tree = torch.gather(sees, 2, node.clamp(0, n - 1)[:, None, :].expand(b, n, s))
    mask = (node < 0)[:, None, :] | (in_tree[:, None, :] & tree)  # [b, n, s]
    k = _values(st["k_codes"], st["k_exp"]).permute(0, 2, 3, 1)  # [b, hk, d, s]
    v = _values(st["v_codes"], st["v_exp"]).permute(0, 2, 1, 3)  # [b, hk, s, d]
    q = st["q"].float().view(b, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    x = (q @ k).view(b, hk, -1, n, s) * (1.0 / math.sqrt(d))
    x = torch.where(mask[:, None, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    o = (x.reshape(b, hk, -1, s) @ v).view(b, hk, hq // hk, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, hq, d)
    o = o / (1.0 + torch.exp(-st["gate"]))
    return torch.where(present[..., None, None], o, 0.0).to(torch.bfloat16)


def _plain_verify(st):
    c = st["case"]
    b, n, vocab, temp = c["batch"], c["nodes"], c["vocab"], c["temperature"]
    sees, present, depth = _tree(st["parents"], b, n)
    at = torch.arange(n, device="cuda")
    parents = (at - 1).expand(b, n) if st["parents"] is None else st["parents"]
    up = parents.clamp(min=0).long()
    child = present & (parents >= 0)
    logits = st["logits"].float()
    logits = torch.where(logits.isfinite(), logits, -math.inf)
    token = st["tokens"].long()
    sibling = (parents[:, :, None] == parents[:, None, :]) & (at[:, None] > at[None, :])  # j an earlier one of i's
    sibling = sibling & child[:, :, None] & child[:, None, :]
    rank = sibling.sum(-1)
    if temp == 0.0:
        best = logits.argmax(-1)
        ok = token == torch.gather(best, 1, up)
    else:
        p = torch.exp(logits / temp - (logits / temp).amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)  # [b, n, vocab]
        flat = up * vocab + token

        def judged(x):  # x[parent of i, token of i]
            return torch.gather(x.view(b, -1), 1, flat)

        if st["draft"] is None:
            px = judged(p)
            same = token[:, :, None] == token[:, None, :]
            px = torch.where((sibling & same).any(-1), 0.0, px)  # a token that was refused already
            ok = st["accept"] * (1.0 - (sibling * px[:, None, :]).sum(-1)) < px
        else:
            # r: what is left of p after the children so far of each node were refused
            r, ok, rounds = p, torch.zeros_like(child), [p]
            for k in range(st["branch"]):
                ok = ok | ((rank == k) & (st["accept"] * judged(st["draft"]) < judged(r)))
                left = (r - st["draft"]).clamp(min=0.0)
                z = left.sum(-1, keepdim=True)
                r = torch.where(z > 0, left / z, r)
                rounds.append(r)
    ok = ok & child
    first = ok & ~(sibling & ok[:, None, :]).any(-1)
    first[:, 0] = present[:, 0]
    on = present & ~(sees & ~first[:, None, :]).any(-1)  # every ancestor, and the node itself, was taken
    count = on.sum(-1)
    last = torch.where(on, depth, -1).argmax(-1)
    order = torch.where(on, at, n).sort(-1).values
    path = torch.where(order < n, order, -1)
    bi = torch.arange(b, device="cuda")
    if temp == 0.0:
        nxt = best[bi, last]
    else:
        mine = child & (parents == last[:, None])  # the refused children of the last node
        if st["draft"] is None:
            left = p[bi, last].scatter_reduce(1, token, torch.where(mine, 0.0, 2.0), "amin")
        else:
            refused = mine.sum(-1)
            left = torch.stack(rounds, 0)[refused, bi, last]
        nxt = (left / st["noise"]).argmax(-1)
    live = present[:, 0]
    return {"path": path.int(), "count": count.int(), "next": torch.where(live, nxt, -1).int()}


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(st):
    c = st["case"]
    op = c["op"]
    if own:
        import firepit_b200 as F
        if op == "verify":
            path, count, nxt = F.tree_verify(st["logits"], st["tokens"], st["parents"], temperature=c["temperature"],
                                             accept=st["accept"], noise=st["noise"], draft=st["draft"])
            return {"path": path, "count": count, "next": nxt}
        cache = F.Kv8Cache(st["k_codes"], st["v_codes"], st["k_exp"], st["v_exp"])
        if op == "append":
            q = F.kv8_append(cache, st["positions"], st["k"], st["v"], q=st["q"], parents=st["parents"],
                             q_gamma=st["q_gamma"], k_gamma=st["k_gamma"], eps=c["eps"],
                             rotary_dim=c["rotary_dim"], theta=1.0e7)
            k, v = F.kv8_read(cache, st["positions"], c["nodes"], torch.bfloat16)
            return {"q": q, "k": k, "v": v}
        if op == "read":
            k, v = F.kv8_read(cache, st["begin"], c["rows"], _dtype(c))
            return {"k": k, "v": v}
        return F.tree_attention(st["q"], cache, st["positions"], st["parents"], gate=st["gate"])
    if op == "append":
        return _plain_append(st)
    if op == "read":
        return _plain_read(st, st["begin"], c["rows"], _dtype(c))
    return _plain_attend(st) if op == "attend" else _plain_verify(st)


def work(case):
    """Bytes: inputs once, outputs once.  Products: two operations each.  verify: the rows that a walk down the tree
    visits, taken as half of the tree's longest branch or of eight nodes, whichever is less, and the last one's noise."""
    b = case["batch"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "verify":
        rows = 1 + min(case["nodes"] - 1, 8) / 2
        each = size + (4 if case["draft"] and case["temperature"] else 0)
        last = 4 if case["temperature"] else 0
        return {"bytes": b * case["vocab"] * (rows * each + last), "flops": b * case["vocab"] * rows * 4}
    hk, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        rows = b * case["nodes"]
        # q and q's copy, k and v, the codes written, read once and returned as bf16
        return {"bytes": rows * d * (2 * case["q_heads"] * size + 2 * hk * (size + 1 + 1 + 2)),
                "flops": rows * d * (case["q_heads"] + hk) * 10}
    if case["op"] == "read":
        n = 2 * b * case["rows"] * hk * d
        return {"bytes": n * (1 + size) + n / d, "flops": n}
    seen = sum(_positions(case)) + sum(_present(case))
    pairs = sum(p * c for p, c in zip(_positions(case), _present(case)))
    rows = b * case["nodes"] * case["q_heads"] * d
    return {"bytes": seen * hk * 2 * (d + 1) + rows * (size + 4 + 2), "flops": 4.0 * pairs * case["q_heads"] * d}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    """Session by session and head by head, from the inputs' values in 64 bits.  append: the keys and values before
    they are rounded to the cache's codes, so the error said is the codes' own.  verify: whole numbers only."""
    if case["op"] == "verify":
        return None
    st = prepare(case, seed)
    b, hk, d = case["batch"], case["kv_heads"], case["head_dim"]
    if case["op"] == "read":
        begin = st["begin"].tolist()
        out = {}
        for name in ("k", "v"):
            part = []
            for i in range(b):
                sl = slice(begin[i], begin[i] + case["rows"])
                code = st[name + "_codes"][i, sl].view(torch.float8_e4m3fn).double()
                part.append(code * torch.pow(2.0, st[name + "_exp"][i, sl].double() - 127.0)[..., None])
            out[name] = torch.stack(part)
        return out
    n, hq = case["nodes"], case["q_heads"]
    pos = st["positions"].tolist()
    parents = [list(range(-1, n - 1))] * b if st["parents"] is None else st["parents"].tolist()
    chain = st["parents"] is None
    lines = []  # for each session and node: its ancestors and itself, or None
    for row in parents if not chain else []:
        line = []
        for i, p in enumerate(row):
            line.append([0] if i == 0 and p == -1 else line[p] + [i] if 0 <= p < i and line[p] is not None else None)
        lines.append(line)
    if case["op"] == "append":
        half = case["rotary_dim"] // 2
        out = {"q": torch.zeros(b, n, hq, d, dtype=torch.float64, device="cuda")}
        for name in ("k", "v"):
            out[name] = torch.zeros(b, n, hk, d, dtype=torch.float64, device="cuda")
        for i in range(b):
            depth = torch.arange(n, device="cuda") if chain else torch.tensor(
                [-1 if x is None else len(x) - 1 for x in lines[i]], device="cuda")
            there = (depth >= 0)[:, None, None]
            z = torch.zeros(n, 1, max(half, 1), dtype=torch.complex128, device="cuda")
            if half:
                w = torch.exp(-math.log(1.0e7) * torch.arange(half, dtype=torch.float64, device="cuda") / half)
                z = torch.exp(1j * (pos[i] + depth).double()[:, None, None] * w)
            for name, gamma in (("q", st["q_gamma"]), ("k", st["k_gamma"])):
                x = st[name][i].double()
                x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + case["eps"]) * gamma.double()
                if half:
                    y = torch.complex(x[..., :half], x[..., half:2 * half]) * z
                    x = torch.cat([y.real, y.imag, x[..., 2 * half:]], -1)
                out[name][i] = torch.where(there, x, 0.0)
            out["v"][i] = torch.where(there, st["v"][i].double(), 0.0)
        return out
    out = torch.zeros(b, n, hq, d, dtype=torch.float64, device="cuda")
    group = hq // hk
    for i in range(b):
        t = pos[i] + n
        bias = torch.zeros(n, t, dtype=torch.float64, device="cuda")
        bias[:, pos[i]:] = -math.inf
        for j, line in enumerate(lines[i]):
            if line is not None:
                bias[j, [pos[i] + a for a in line]] = 0.0
        alive = [j for j, line in enumerate(lines[i]) if line is not None]
        for h in range(hk):
            kk = st["k_codes"][i, :t, h].view(torch.float8_e4m3fn).double()
            kk = kk * torch.pow(2.0, st["k_exp"][i, :t, h].double() - 127.0)[:, None]
            vv = st["v_codes"][i, :t, h].view(torch.float8_e4m3fn).double()
            vv = vv * torch.pow(2.0, st["v_exp"][i, :t, h].double() - 127.0)[:, None]
            for g in range(group):
                qq = st["q"][i, alive, h * group + g].double()
                w = torch.softmax(qq @ kk.T / math.sqrt(d) + bias[alive], -1)
                out[i, alive, h * group + g] = (w @ vv) * torch.sigmoid(st["gate"][i, alive, h * group + g].double())
    return out
