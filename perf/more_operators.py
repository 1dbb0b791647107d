"""The operators of serving over a paged key/value cache: what is measured.

Four operators, each in its plain form (elementary torch operations) and through the framework's entry points:

  pages    the requests of a step take pages from the pool for their new tokens (block tables, slot and position of each
           token), and give them back
  append   head norms of q and k, rotation by position, and the new tokens' keys and values written at their slots
  attend   attention of one new token a session over its pages, times the sigmoid of a gate
  sample   the next tokens from the logits: temperature, top-k, top-p and min-p of each session, from given exponential
           variates

The cache holds keys and values [pages, page_size, kv_heads, head_dim]; token t of session b lies in row t % page_size
of page table[b, t // page_size], and a slot is page * page_size + row.  The free pages are a stack: the i-th page that
a step takes (requests in order, their pages in order) is free[free_count - 1 - i], and pages given back go where they
came from.

Sampling orders a row's tokens by weight, falling, ties by index.  top-k keeps the first k; top-p the shortest prefix of
those whose weights reach p of their sum; min-p those whose weight is at least min_p of the largest.  Of what is kept
the token with the largest weight / noise is taken, which draws from it.  Temperature 0 takes the first token.
"""
import math

import torch

own = False

VOCAB = 151936  # the hybrid decoder's vocabulary
THETA = 1.0e7


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    def attend(name, **kw):
        return dict(dict(name=name, op="attend"), **kw)

    return [
        # a decode step's bookkeeping: 64 sessions of up to 9000 tokens, one new token each; latency alone
        dict(name="pages 64x1", op="pages", batch=64, tokens=1, context=9000, page_size=16),
        # 96 ragged prompts admitted at once
        dict(name="pages 96 prompts", op="pages", batch=96, tokens=2000, context=0, page_size=32),
        # one decode step of eight sessions at the hybrid decoder's attention heads, f32 pages as its caches are
        dict(name="append 8x1", op="append", batch=8, tokens=1, q_heads=16, kv_heads=2, head_dim=256, rotary_dim=64,
             context=511, page_size=16, dtype="f32", cache="f32", eps=1e-6),
        # ragged prompts written together, bf16 projections, every dimension rotated
        dict(name="append 11 prompts", op="append", batch=11, tokens=1501, q_heads=32, kv_heads=8, head_dim=128,
             rotary_dim=128, context=333, page_size=64, dtype="bf16", cache="bf16", eps=1e-6),
        # the smallest call: one session with a short context that ends inside a page
        attend("attend 1 at 777", batch=1, q_heads=16, kv_heads=2, head_dim=256, context=777, page_size=16, dtype="f32",
               cache="bf16"),
        # the hybrid decoder's eight sessions at the end of its workload, f32 pages
        attend("attend 8 at 2304, f32", batch=8, q_heads=16, kv_heads=2, head_dim=256, context=2304, page_size=16,
               dtype="f32", cache="f32"),
        # sixteen sessions of long contexts at the hybrid decoder's heads
        attend("attend 16 at 8192", batch=16, q_heads=16, kv_heads=2, head_dim=256, context=8192, page_size=64,
               dtype="f32", cache="bf16"),
        # a full server: many sessions of very different lengths, more blocks of work than the GPU holds at once
        attend("attend 200 ragged", batch=200, q_heads=32, kv_heads=8, head_dim=128, context=4001, page_size=32,
               dtype="bf16", cache="bf16"),
        # three documents read to the end: the splits of few sessions fill the GPU; 16 query heads share a key head
        attend("attend 3 at 100003", batch=3, q_heads=64, kv_heads=4, head_dim=128, context=100003, page_size=128,
               dtype="bf16", cache="bf16"),
        # one session's token
        dict(name="sample 1", op="sample", batch=1, vocab=VOCAB, dtype="f32", kinds="topp"),
        # the decoder's eight sessions, each with its own choice of filters
        dict(name="sample 8 mixed", op="sample", batch=8, vocab=VOCAB, dtype="f32", kinds="mixed"),
        # a full server's step, bf16 logits (equal ones are common)
        dict(name="sample 250 mixed", op="sample", batch=250, vocab=VOCAB, dtype="bf16", kinds="mixed"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["pages", "append", "attend", "attend", "sample"])
    page_size = rng.choice([8, 16, 16, 24, 32, 64, 128])
    dtype, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
    if op == "pages":
        batch = _log(rng, 1, 512)
        tokens = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, 190000 // batch))
        return dict(op=op, batch=batch, tokens=tokens, context=rng.choice([0, _log(rng, 1, 20000)]), page_size=page_size)
    if op == "sample":
        return dict(op=op, batch=_log(rng, 1, 128), vocab=_log(rng, 1000, 160000), dtype=dtype,
                    kinds=rng.choice(["greedy", "topk", "topp", "minp", "all", "plain", "mixed"]))
    while True:
        kv_heads, group = rng.randint(1, 8), rng.choice([1, 2, 3, 4, 6, 8, 16])
        case = dict(op=op, batch=_log(rng, 1, 32 if op == "append" else 256), q_heads=kv_heads * group,
                    kv_heads=kv_heads, head_dim=rng.choice([64, 80, 96, 128, 192, 256]), page_size=page_size,
                    dtype=dtype, cache=cache)
        if op == "append":
            case.update(tokens=1 if rng.random() < 0.5 else _log(rng, 1, 1500), context=_log(rng, 1, 8192), eps=1e-6)
            case["rotary_dim"] = rng.choice([0, 32, 64, case["head_dim"]])
        else:
            case["context"] = _log(rng, 1, 60000)
        w = work(case)
        if all(w[k] <= max(work(c)[k] for c in listed() if c["op"] == op) for k in w):
            return case


# ---- inputs --------------------------------------------------------------------------------------------------------
def _dtype(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _contexts(case):
    """Tokens that each session holds: the first the most; the last of many next to none."""
    c, b = case["context"], case["batch"]
    spread = 4 if b < 64 else 0
    return [c - (i * c) // (spread * b if spread else b) for i in range(b)]


def _counts(case):
    """New tokens of each session."""
    n, b = case["tokens"], case["batch"]
    return [n - (i * n) // (2 * b) for i in range(b)]


def prepare(case, seed):
    rnd = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=dev, device="cuda") * std).to(dtype)

    st = dict(case=case)
    b = case["batch"]
    if case["op"] == "sample":
        return _prepare_sample(case, st, rnd, dev)
    p = case["page_size"]
    held = _contexts(case)
    counts = [0] * b if case["op"] == "attend" else _counts(case)
    new = [h + n for h, n in zip(held, counts)]
    # each session's pages, in no order, and the pool that they are taken from
    pages = [-(-n // p) for n in (held if case["op"] == "pages" else new)]
    total = sum(pages)
    if case["op"] == "pages":
        total = sum(-(-n // p) for n in new) + 40
    order = torch.randperm(total, generator=rnd).int()
    width = max(-(-n // p) for n in new) + 3
    table = torch.full((b, width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    st["table"] = table.cuda()
    if case["op"] == "pages":
        free = torch.full((total,), -1, dtype=torch.int32)
        free[:total - at] = order[at:]
        st["free"], st["free_count"] = free.cuda(), torch.tensor([total - at], dtype=torch.int32).cuda()
        st["lengths"] = torch.tensor(held, dtype=torch.int32).cuda()
        st["before"] = st["lengths"].clone()
        st["counts"] = torch.tensor(counts, dtype=torch.int32).cuda()
        st["rows"] = sum(counts) if case["tokens"] == 1 else sum(counts) + 77  # a few rows to spare
        if own:
            import firepit_b200 as F
            st["tables"] = F.PageTables(st["table"], st["lengths"], st["free"], st["free_count"], p)
        return st
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    dt, ct = _dtype(case["dtype"]), _dtype(case["cache"])
    # normed and rotated keys have vectors of about sqrt(head_dim)
    st["k_pages"] = normal(total, p, hk, d, std=1.3, dtype=ct)
    st["v_pages"] = normal(total, p, hk, d, dtype=ct)
    if own:
        import firepit_b200 as F
        st["cache"] = F.PagedCache(st["k_pages"], st["v_pages"])
    if case["op"] == "attend":
        st["lengths"] = torch.tensor(held, dtype=torch.int32).cuda()
        # the projections' outputs: per query head its query, then its gate, as the decoder's w_qg gives them
        st["q"] = normal(b, hq, d, std=1.6, dtype=dt)
        st["gate"] = normal(b, hq, 2 * d)[..., d:]
        return st
    slots, positions = [], []
    for i in range(b):
        t = torch.arange(held[i], new[i])
        positions.append(t)
        slots.append(table[i, t // p].long() * p + t % p)
    pad = 5 if case["tokens"] > 1 else 0  # rows that hold no token
    none = torch.full((pad,), -1)
    st["slots"] = torch.cat(slots + [none]).int().cuda()
    st["positions"] = torch.cat(positions + [none]).int().cuda()
    n = st["slots"].numel()
    st["q"] = normal(n, hq, 2 * d, dtype=dt)[..., :d]
    st["k"] = normal(n, hk, d, std=2.0, dtype=dt)
    st["v"] = normal(n, hk, d, std=0.7, dtype=dt)
    st["q_gamma"] = 1.0 + normal(d, std=0.1)
    st["k_gamma"] = 1.0 + normal(d, std=0.1)
    return st


def _prepare_sample(case, st, rnd, dev):
    b, vocab = case["batch"], case["vocab"]
    # weights that fall with a power of the rank, from steep (a few likely tokens) to flat, in no order, with an error
    steep = torch.rand(b, 1, generator=dev, device="cuda") * 1.7 + 0.5
    base = -torch.log(1.0 + torch.arange(vocab, device="cuda", dtype=torch.float32))
    logits = torch.empty(b, vocab, device="cuda")
    for i in range(b):
        logits[i] = base[torch.randperm(vocab, generator=dev, device="cuda")]
    logits = logits * steep + 0.5 * torch.randn(b, vocab, generator=dev, device="cuda") + 12.0
    st["logits"] = logits.to(_dtype(case["dtype"]))
    kinds = ["topk", "topp", "all", "minp", "plain", "greedy"]
    st["kinds"] = [case["kinds"] if case["kinds"] != "mixed" else kinds[i % 6] for i in range(b)]
    u = torch.rand(b, 4, generator=rnd).tolist()
    temp, top_k, top_p, min_p = [], [], [], []
    for kind, r in zip(st["kinds"], u):
        temp.append(0.0 if kind == "greedy" else 0.6 + 0.6 * r[0])
        top_k.append(1 + int(99 * r[1]) if kind in ("topk", "all") else 0)
        top_p.append(0.8 + 0.19 * r[2] if kind in ("topp", "all") else 1.0)
        min_p.append(0.01 + 0.1 * r[3] if kind in ("minp", "all") else 0.0)
    st["temperature"], st["top_p"], st["min_p"] = (torch.tensor(x, dtype=torch.float32).cuda()
                                                   for x in (temp, top_p, min_p))
    st["top_k"] = torch.tensor(top_k, dtype=torch.int32).cuda()
    st["noise"] = -torch.log(torch.rand(b, vocab, generator=dev, device="cuda").clamp(1e-30, 1 - 1e-7))
    return st


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _plain_pages(st):
    p, rows = st["case"]["page_size"], st["rows"]
    lengths, counts, table, free, free_count = (st[k] for k in ("lengths", "counts", "table", "free", "free_count"))
    b, width = table.shape
    # (every request is served here: the pool and the tables hold what the step asks for)
    new = lengths + counts
    held, want = (lengths + p - 1) // p, (new + p - 1) // p
    take = want - held
    off = take.cumsum(0) - take
    col = torch.arange(width, device="cuda")
    fresh = (col >= held[:, None]) & (col < want[:, None])
    at = free_count - 1 - (off[:, None] + col - held[:, None])
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1).long()], table))
    free_count.sub_(take.sum())
    ends = counts.cumsum(0)
    starts = torch.cat([ends.new_zeros(1), ends]).int()
    r = torch.arange(rows, device="cuda")
    req = torch.searchsorted(ends, r, right=True)
    there = req < b
    req = req.clamp(max=b - 1)
    pos = lengths[req] + r - (ends - counts)[req]
    slot = table[req, torch.where(there, pos // p, 0).long()] * p + pos % p
    slots, positions, requests = (torch.where(there, x, -1).int() for x in (slot, pos, req))
    lengths.add_(counts)
    out = {"slots": slots, "positions": positions, "requests": requests, "starts": starts, "taken": table.clone()}
    # and back
    free_count.add_(take.sum())
    free.scatter_(0, torch.where(fresh, at, free.numel() - 1).long().view(-1),
                  torch.where(fresh, table, free[-1]).view(-1))
    table.masked_fill_(fresh, -1)
    lengths.copy_(st["before"])
    return {**out, "table": table, "lengths": lengths, "free": free, "free_count": free_count}


def _rotate(x, pos, rotary):
    """Rotation of the first `rotary` dimensions, halves as pairs; the angles in 64 bits: 32 lose them at long
    positions."""
    if not rotary:
        return x
    half = rotary // 2
    freq = THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    ang = pos.double()[:, None, None] * freq
    c, s = ang.cos().float(), ang.sin().float()
    x0, x1 = x[..., :half], x[..., half:rotary]
    return torch.cat([x0 * c - x1 * s, x1 * c + x0 * s, x[..., rotary:]], -1)


def _plain_append(st):
    c = st["case"]
    there = st["slots"] >= 0

    def normed(x, gamma):
        x = x.float()
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + c["eps"]) * gamma

    q = _rotate(normed(st["q"], st["q_gamma"]), st["positions"], c["rotary_dim"])
    k = _rotate(normed(st["k"], st["k_gamma"]), st["positions"], c["rotary_dim"])
    at = st["slots"][there].long()
    for pages, x in ((st["k_pages"], k), (st["v_pages"], st["v"])):
        pages.view(-1, *pages.shape[2:])[at] = x[there].to(pages.dtype)
    return {"q": torch.where(there[:, None, None], q, 0.0).to(_dtype(c["dtype"])), "k": st["k_pages"],
            "v": st["v_pages"]}


def _plain_attend(st):
    c = st["case"]
    b, hq, hk, d, p = c["batch"], c["q_heads"], c["kv_heads"], c["head_dim"], c["page_size"]
    s = max(1, c["context"])
    t = torch.arange(s, device="cuda")
    out = torch.empty(b, hq, d, dtype=torch.float32 if c["cache"] == "f32" else torch.bfloat16, device="cuda")
    step = max(1, 2 ** 28 // (s * hk * d))  # sessions at once
    for i in range(0, b, step):
        lengths, table = st["lengths"][i:i + step], st["table"][i:i + step]
        n = lengths.numel()
        seen = t < lengths[:, None]  # [n, s]
        slot = torch.where(seen, table[:, t // p].long() * p + t % p, 0)
        k = st["k_pages"].view(-1, hk, d)[slot].float().permute(0, 2, 3, 1)  # [n, hk, d, s]
        q = st["q"][i:i + step].float().view(n, hk, hq // hk, d)
        x = (q @ k) * (1.0 / math.sqrt(d))
        x = torch.where(seen[:, None, None], x, -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
        x = x / x.sum(-1, keepdim=True).clamp(min=1e-30)
        v = st["v_pages"].view(-1, hk, d)[slot].float().permute(0, 2, 1, 3)  # [n, hk, s, d]
        o = (x @ v).view(n, hq, d)
        out[i:i + step] = o / (1.0 + torch.exp(-st["gate"][i:i + step]))
    return out


def _plain_sample(st):
    # (64 bits: the sums of long rows decide which token is the last that top-p keeps)
    logits = st["logits"].double()
    logits = torch.where(logits.isfinite(), logits, -math.inf)
    greedy = st["temperature"] <= 0
    temp = torch.where(greedy, 1.0, st["temperature"]).double()[:, None]
    x = logits / temp
    w = torch.exp(x - x.amax(-1, keepdim=True))
    s, order = torch.sort(w, dim=-1, descending=True, stable=True)
    at = torch.arange(w.shape[1], device="cuda")
    k = torch.where(st["top_k"] > 0, st["top_k"], w.shape[1])[:, None]
    s = torch.where(at < k, s, 0.0)
    total = s.sum(-1, keepdim=True)
    p = st["top_p"].double()[:, None]
    keep = (at < k) & ((p >= 1) | (s.cumsum(-1) - s < p * total) | (at == 0)) & (s >= st["min_p"].double()[:, None])
    keep = torch.zeros_like(keep).scatter(1, order, keep)
    w = torch.where(keep, w, 0.0)
    token = torch.where(greedy, logits.argmax(-1), (w / st["noise"].double()).argmax(-1))
    logprob = torch.log(torch.gather(w, 1, token[:, None])[:, 0] / w.sum(-1))
    return {"tokens": token.int(), "logprobs": torch.where(greedy, 0.0, logprob).float()}


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(st):
    c = st["case"]
    op = c["op"]
    if own:
        import firepit_b200 as F
        if op == "pages":
            m = F.page_extend(st["tables"], st["counts"], st["rows"])
            out = {"slots": m.slots, "positions": m.positions, "requests": m.requests, "starts": m.starts,
                   "taken": st["table"].clone()}
            F.page_truncate(st["tables"], st["before"])
            return {**out, **{k: st[k] for k in ("table", "lengths", "free", "free_count")}}
        if op == "append":
            q = F.paged_append(st["cache"], st["slots"], st["positions"], st["k"], st["v"], q=st["q"],
                               q_gamma=st["q_gamma"], k_gamma=st["k_gamma"], eps=c["eps"],
                               rotary_dim=c["rotary_dim"], theta=THETA)
            return {"q": q, "k": st["k_pages"], "v": st["v_pages"]}
        if op == "attend":
            return F.paged_attention(st["q"], st["cache"], st["table"], st["lengths"], gate=st["gate"])
        tokens, logprobs = F.sample(st["logits"], st["temperature"], st["noise"], top_k=st["top_k"],
                                    top_p=st["top_p"], min_p=st["min_p"], logprobs=True)
        return {"tokens": tokens, "logprobs": logprobs}
    return {"pages": _plain_pages, "append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[op](st)


def work(case):
    """Bytes: inputs once, outputs once.  Products: two operations each."""
    b = case["batch"]
    size = 4 if case.get("dtype") == "f32" else 2
    if case["op"] == "sample":
        # the logits once; the noise of a row where nothing is filtered out
        whole = {"plain": b, "mixed": b // 6}.get(case["kinds"], 0)
        return {"bytes": case["vocab"] * (b * size + whole * 4) + b * 24, "flops": b * case["vocab"] * 4}
    p = case["page_size"]
    held = _contexts(case)
    if case["op"] == "pages":
        counts = _counts(case)
        fresh = sum(-(-(h + n) // p) - -(-h // p) for h, n in zip(held, counts))
        # slot, position and request of each row; each page taken from the stack, entered, returned and cleared; lengths
        # and counts read, starts written, lengths written twice; the copy of the table that the pass returns
        width = -(-(case["context"] + case["tokens"]) // p) + 3
        return {"bytes": 12 * sum(counts) + 16 * fresh + 20 * b + 8 * b * width, "flops": 4 * sum(counts)}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    cache = 4 if case["cache"] == "f32" else 2
    if case["op"] == "append":
        rows = sum(_counts(case))
        return {"bytes": rows * d * (2 * hq * size + 2 * hk * (size + cache)), "flops": rows * d * (hq + hk) * 10}
    seen = sum(held)
    return {"bytes": seen * hk * 2 * d * cache + b * hq * d * (size + 4 + cache), "flops": 4.0 * seen * hq * d}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    """Session by session, from the inputs' values in 64 bits.  append: the keys and values before they are rounded to
    the pages' type.  pages: whole numbers only."""
    if case["op"] == "pages":
        return None
    st = prepare(case, seed)
    b = case["batch"]
    if case["op"] == "sample":
        out = torch.zeros(b, dtype=torch.float64, device="cuda")
        vocab = case["vocab"]
        for i in range(b):
            t, k, p, m = (float(st[n][i]) for n in ("temperature", "top_k", "top_p", "min_p"))
            if t <= 0:
                continue
            row = st["logits"][i].double() / t
            best, where = torch.sort(row, descending=True, stable=True)
            n = vocab if k <= 0 else min(vocab, int(k))
            best, where = best[:n], where[:n]
            prob = torch.softmax(best, 0)
            if p < 1:
                before = torch.cat([prob.new_zeros(1), torch.cumsum(prob, 0)[:-1]])
                n = max(1, int((before < p).sum()))
            if m > 0:
                n = min(n, int((best >= best[0] + math.log(m)).sum()))
            left = best[:n]
            race = left - torch.log(st["noise"][i][where[:n]].double())
            out[i] = left[race.argmax()] - torch.logsumexp(left, 0)
        return {"tokens": None, "logprobs": out}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        half = case["rotary_dim"] // 2
        live = st["slots"] >= 0
        z = torch.zeros(live.numel(), 1, max(half, 1), dtype=torch.complex128, device="cuda")
        if half:
            w = torch.exp(-math.log(THETA) * torch.arange(half, dtype=torch.float64, device="cuda") / half)
            z = torch.exp(1j * st["positions"].double()[:, None, None] * w)
        out = {}
        for name, gamma in (("q", st["q_gamma"]), ("k", st["k_gamma"])):
            x = st[name].double()
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + case["eps"]) * gamma.double()
            if half:
                y = torch.complex(x[..., :half], x[..., half:2 * half]) * z
                x = torch.cat([y.real, y.imag, x[..., 2 * half:]], -1)
            out[name] = x
        out["q"][~live] = 0.0
        out["v"] = st["v"].double()
        for name in ("k", "v"):
            pages = st[name + "_pages"].double()
            pages.view(-1, hk, d).index_copy_(0, st["slots"][live].long(), out[name][live])
            out[name] = pages
        return out
    p = case["page_size"]
    out = torch.zeros(b, hq, d, dtype=torch.float64, device="cuda")
    group = hq // hk
    for i, n in enumerate(_contexts(case)):
        if n == 0:
            continue
        pages = st["table"][i, :-(-n // p)].long()
        kk = st["k_pages"][pages].reshape(-1, hk, d)[:n].double()
        vv = st["v_pages"][pages].reshape(-1, hk, d)[:n].double()
        for h in range(hk):
            sl = slice(h * group, (h + 1) * group)
            w = torch.softmax(st["q"][i, sl].double() @ kk[:, h].T / math.sqrt(d), -1)
            out[i, sl] = (w @ vv[:, h]) * torch.sigmoid(st["gate"][i, sl].double())
    return out
