"""The paged cache in the decoder: requests of different lengths that come and
go, each with its own sampling.

Bars: two ways to the same logits differ by bf16 roundings of the attention
outputs and GEMV inputs (2^-9 each, and the rows that they move) through the
layers: relative Frobenius 1e-2, as for the 8-bit cache's decoder; bf16 pages
round keys and values once more (2^-9): 2e-2.
"""
import numpy as np
import pytest

from oracle import oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


@pytest.fixture(scope="module")
def model(torch):
    """Recurrent and attention layers."""
    from firepit_b200.model import HybridConfig, HybridModel
    cfg = HybridConfig(layers=4, hidden=256, vocab=512, full_attention_interval=2, q_heads=4, kv_heads=2, head_dim=64,
                       rotary_dim=16, key_heads=2, value_heads=4, key_head_dim=32, value_head_dim=32, experts=8,
                       top_k=2, moe_inter=256)
    return HybridModel(cfg, seed=3)


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    import firepit_b200 as F
    assert F.device_error(reset=True) == 0


def _alone(torch, model, tokens, max_seq=64):
    """Logits after each token of a chain, on the contiguous f32 cache."""
    from firepit_b200.model import Decoder
    dec, out = Decoder(model, 1, max_seq), []
    for t in tokens:
        dec.tokens.fill_(int(t))
        dec.step(torch.cuda.current_stream().cuda_stream)
        out.append(dec.logits[0].clone())
    return torch.stack(out).cpu().numpy()


@pytest.mark.parametrize("pages,bar", [("f32", 1e-2), ("bf16", 2e-2)])
def test_paged_decoder_matches_the_contiguous_cache(torch, model, pages, bar):
    """Prompts of different lengths, one after another on the same row and beside
    one another: the logits of every token are those that its session alone gets."""
    from firepit_b200.model import PagedDecoder, Request
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, 512, n).tolist() for n in (9, 21, 1, 13, 30, 5)]
    dtype = torch.float32 if pages == "f32" else torch.bfloat16
    dec = PagedDecoder(model, 3, 32, 20, 4, dtype)
    sh = torch.cuda.current_stream().cuda_stream
    want = [_alone(torch, model, p) for p in prompts]
    live, at, seen = {}, 0, [0] * len(prompts)
    while live or at < len(prompts):
        for s in range(3):
            if s not in live and at < len(prompts) and dec.admit(s, Request(prompts[at], 1)):
                live[s] = at
                at += 1
        dec.step(sh)
        logits = dec.logits.cpu().numpy()
        done = []
        for s, r in live.items():
            assert O.rel_frobenius(logits[s], want[r][seen[r]]) <= bar, (r, seen[r])
            seen[r] += 1
            if seen[r] == len(prompts[r]):
                assert int(dec.emitted[s]) == int(logits[s].argmax())
                done.append(s)
            else:
                assert int(dec.emitted[s]) == -1
        if done:
            dec.release(*done)
            for s in done:
                del live[s]
    assert seen == [len(p) for p in prompts]
    assert int(dec.tables.free_count) == 20 and not dec.tables.lengths.any() and sum(dec.reserved) == 0
    assert sorted(dec.tables.free.tolist()) == list(range(20))


def test_serve_greedy_tokens_are_the_largest_logits(torch, model):
    """More requests than rows, more than the pool holds at once.  Every token is the
    largest of its step's logits, and those are the ones that its session alone gets
    on the contiguous cache, where the routers chose the same experts (a choice
    between two that lie as near as the bar may fall either way; nineteen of twenty
    tokens agree, and what follows one that does not has seen other keys)."""
    from types import SimpleNamespace

    from firepit_b200.model import Decoder, PagedDecoder, Request
    rng = np.random.default_rng(2)
    requests = [Request(rng.integers(0, 512, int(rng.integers(1, 20))).tolist(), int(rng.integers(1, 25)))
                for _ in range(11)]
    sh = torch.cuda.current_stream().cuda_stream
    c = model.cfg
    rows: list[dict] = [{} for _ in requests]

    class Logged(PagedDecoder):
        def admit(self, session, request):
            ok = super().admit(session, request)
            if ok:
                who[session] = next(i for i, r in enumerate(requests) if r is request)
            return ok

        def replay(self):
            self.step(sh)
            pos, logits, routes = self.map.positions.tolist(), self.logits.cpu().numpy(), self.route_log.cpu().numpy()
            for s, r in who.items():
                if pos[s] >= 0:
                    rows[r][pos[s]] = logits[s].copy(), np.sort(routes[:, s], -1)

    who: dict = {}
    dec = Logged(model, 4, 48, 13, 8)
    dec.route_log = torch.zeros(c.layers, 4, c.slots, dtype=torch.int32, device="cuda")
    dec.graph = SimpleNamespace(replay=dec.replay)
    out = dec.serve(requests)
    assert [len(o) for o in out] == [r.new_tokens for r in requests]
    assert int(dec.tables.free_count) == 13
    tokens = flips = 0
    for r, o, row in zip(requests, out, rows):
        alone = Decoder(model, 1, 64)
        alone.route_log = torch.zeros(c.layers, 1, c.slots, dtype=torch.int32, device="cuda")
        chain = r.prompt + o[:-1]
        assert sorted(row) == list(range(len(chain)))
        agreed = True
        for t, token in enumerate(chain):
            alone.tokens.fill_(int(token))
            alone.step(sh)
            agrees = (np.sort(alone.route_log[:, 0].cpu().numpy(), -1) == row[t][1]).all()
            tokens += 1
            flips += not agrees
            agreed &= agrees
            if agreed:
                assert O.rel_frobenius(row[t][0], alone.logits[0].cpu().numpy()) <= 2e-2, t
            if t >= len(r.prompt) - 1:
                assert o[t - len(r.prompt) + 1] == int(row[t][0].argmax())
    assert flips * 20 <= tokens
    graph = PagedDecoder(model, 4, 48, 13, 8)
    assert graph.serve(requests) == out  # replayed, with the same shares: the same bits
    assert graph.serve(requests) == out


def test_serve_draws_from_given_numbers(torch, model):
    """Requests with filters of their own: the same generator gives the same tokens,
    top_k 1 is greedy whatever the temperature, and eos ends a request."""
    from firepit_b200.model import PagedDecoder, Request
    prompt = [3, 1, 4, 1, 5]
    requests = [Request(prompt, 12), Request(prompt, 12, temperature=5.0, top_k=1),
                Request(prompt, 12, temperature=1.5, top_p=0.9), Request(prompt, 12, temperature=1.5, top_p=0.9),
                Request(prompt, 12, temperature=3.0, min_p=0.01), Request(prompt, 12, temperature=2.0, top_k=7, top_p=0.8)]
    dec = PagedDecoder(model, 3, 32, 12, 4)
    g = torch.Generator(device="cuda")
    first = dec.serve(requests, generator=g.manual_seed(7))
    assert first == dec.serve(requests, generator=g.manual_seed(7))
    assert first != dec.serve(requests, generator=g.manual_seed(8))
    assert first[0] == first[1] and first[2] != first[3]
    assert all(0 <= t < 512 for o in first for t in o)
    eos = first[0][4]
    short = dec.serve(requests[:1], eos=eos)[0]
    assert short == first[0][:first[0].index(eos) + 1]


def test_paged_decoder_on_a_side_stream_equals_the_graph(torch, model):
    """Eager steps on another stream and replayed ones: the same tokens, bit for bit."""
    from firepit_b200.model import PagedDecoder, Request
    requests = [Request([5, 77, 301], 9, temperature=1.0, top_p=0.95), Request([8], 6), Request([2, 2], 8, temperature=0.7)]
    side = torch.cuda.Stream()
    runs = []
    for graph in (False, True):
        dec = PagedDecoder(model, 3, 16, 9, 4)
        dec.step(torch.cuda.current_stream().cuda_stream)
        if graph:
            dec.capture()
        dec.reset()
        g = torch.Generator(device="cuda").manual_seed(3)
        for s, r in enumerate(requests):
            assert dec.admit(s, r)
        got = []
        for _ in range(8):
            dec.draw(g)
            torch.cuda.synchronize()
            if graph:
                dec.graph.replay()
            else:
                dec.step(side.cuda_stream)
            torch.cuda.synchronize()
            got.append(dec.emitted.tolist() + dec.tokens.tolist())
        runs.append(got)
    assert runs[0] == runs[1]


def test_paged_decoder_refuses_what_does_not_fit(torch, model):
    import firepit_b200 as F
    from firepit_b200.model import PagedDecoder, Request
    dec = PagedDecoder(model, 2, 16, 5, 4)
    for r in (Request([], 3), Request([1], 0), Request([1] * 10, 8), Request([512], 2), Request([-1], 2)):
        with pytest.raises(F.ShapeError):
            dec.admit(0, r)
    assert dec.admit(0, Request([1] * 10, 6))  # 15 tokens run: four pages
    assert not dec.admit(1, Request([1] * 3, 3))  # two more
    assert dec.admit(1, Request([1] * 3, 2))  # one more
    with pytest.raises(F.ShapeError):
        dec.admit(1, Request([1], 1))
    with pytest.raises(F.ShapeError):
        PagedDecoder(model, 2, 100, 5, 4).serve([Request([1] * 18, 4)])
    for bad in ((0, 16, 5, 4), (2, 0, 5, 4), (2, 16, 0, 4), (2, 16, 5, 0)):
        with pytest.raises(F.ShapeError):
            PagedDecoder(model, *bad)


def test_paged_decoder_takes_no_batch(torch, model):
    """The other decoders' prefill and generate would run steps beside the requests:
    they say what to call instead, and leave the sessions as they were."""
    from firepit_b200.model import PagedDecoder, Request
    dec = PagedDecoder(model, 2, 16, 8, 4)
    dec.step(torch.cuda.current_stream().cuda_stream)
    dec.capture()
    dec.reset()
    assert dec.admit(0, Request([3, 1, 4], 4))
    before = [t.clone() for t in (dec.tokens, dec.tables.lengths, dec.active, dec.prompt)]
    for call in (lambda: dec.prefill(torch.ones(2, 3, dtype=torch.int32, device="cuda")), lambda: dec.generate(3)):
        with pytest.raises(NotImplementedError, match="serve"):
            call()
    for t, w in zip((dec.tokens, dec.tables.lengths, dec.active, dec.prompt), before):
        assert torch.equal(t, w)


def test_paged_decoder_sessions_end_by_themselves(torch, model):
    """A session that has its tokens takes no further page, released or not: what was
    counted for the others stays theirs."""
    from firepit_b200.model import PagedDecoder, Request
    a, b = Request([1, 2, 3], 2), Request([9, 8, 7, 6, 5], 16)  # four tokens run, and twenty: one page and five
    runs = []
    for late in (False, True):
        dec = PagedDecoder(model, 2, 32, 6, 4, torch.float32)
        assert dec.admit(0, a) and dec.admit(1, b)
        out = [[], []]
        for step in range(22):
            dec.step(torch.cuda.current_stream().cuda_stream)
            for o, t in zip(out, dec.emitted.tolist()):
                o.append(t)
            assert dec.tables.lengths.tolist()[0] <= 4 and dec.tables.lengths.tolist()[1] == min(step + 1, 20)
            if step == 3 and not late:
                dec.release(0)
        runs.append(out)
        assert [t >= 0 for t in out[0]] == [2 <= step < 4 for step in range(22)]
        assert [t >= 0 for t in out[1]] == [4 <= step < 20 for step in range(22)]
        dec.release(0, 1)
        assert int(dec.tables.free_count) == 6 and dec.admit(0, b) and dec.reserved == [5, 0]
    assert runs[0] == runs[1]


def test_paged_decoder_a_refused_request_leaves_the_row_free(torch, model):
    import firepit_b200 as F
    from firepit_b200.model import PagedDecoder, Request
    dec = PagedDecoder(model, 2, 16, 8, 4)
    for bad in (dict(temperature=None), dict(top_k=2 ** 40), dict(top_k=0.5), dict(top_p="x"), dict(min_p=float("nan")),
                dict(temperature=float("nan"))):
        with pytest.raises(F.ShapeError):
            dec.admit(0, Request([1, 2], 3, **bad))
        with pytest.raises(F.ShapeError):
            dec.serve([Request([1, 2], 3), Request([1, 2], 3, **bad)])
        assert dec.reserved == [0, 0] and not dec.active.any()
    assert dec.admit(0, Request([1, 2], 3, temperature=1, top_k=2 ** 31 - 1, top_p=0, min_p=2))
    assert dec.admit(1, Request([1, 2], 3, temperature=1e300, top_p=-1e300, min_p=float("inf")))  # (no f32 numbers)
