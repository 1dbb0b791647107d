"""The 8-bit cache and speculative decoding in the decoder.

Bars: two ways to the same logits over the same 8-bit cache differ by bf16
roundings of the attention outputs and GEMV inputs (2^-9 each, and the few
codes that they flip) through the layers: relative Frobenius 1e-2.
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
    from firepit_b200.model import HybridConfig, HybridModel
    cfg = HybridConfig(layers=3, hidden=256, vocab=512, full_attention_interval=1, q_heads=4, kv_heads=2, head_dim=64,
                       rotary_dim=16, experts=8, top_k=2, moe_inter=256)
    return HybridModel(cfg, seed=3)


def _no_error():
    import firepit_b200 as F
    assert F.device_error(reset=True) == 0


def _chain_logits(torch, model, tokens, kv8):
    """Logits after each token of a chain, one decode step a token."""
    from firepit_b200.model import Decoder
    dec = Decoder(model, 1, 64, kv8=kv8)
    out = []
    for t in tokens:
        dec.tokens.fill_(int(t))
        dec.step(torch.cuda.current_stream().cuda_stream)
        out.append(dec.logits[0].clone())
    return torch.stack(out).cpu().numpy()


def test_decoder_on_the_8_bit_cache(torch, model):
    """Against the f32-cache decoder whose rows are rounded to the 8-bit
    cache's values as they are written.  One layer: its keys and values come
    from the tokens alone, so both sides round the same numbers (further down a
    difference of 2^-9 between two inputs flips codes, and those are 2^-4
    apart)."""
    from dataclasses import replace

    from firepit_b200 import _native as N
    from firepit_b200.model import Decoder, HybridModel
    model = HybridModel(replace(model.cfg, layers=1), seed=4)
    from oracle import speculative as R

    class Rounded(Decoder):
        def _attend(self, i, L, sh):
            call = N.call
            pos = self.positions.tolist()

            def between(name, *args):  # between the append and the attention
                if name == "fpb_attn_decode":
                    for t in self.kv[i]:
                        for b, p in enumerate(pos):
                            t[b, p] = torch.from_numpy(R.values(*R.quantise(t[b, p].cpu().numpy()))).to(t)
                call(name, *args)

            N.call = between
            try:
                super()._attend(i, L, sh)
            finally:
                N.call = call

    toks = [5, 77, 301, 8, 8, 19, 400, 2]
    got = _chain_logits(torch, model, toks, True)
    dec, want = Rounded(model, 1, 64), []
    for t in toks:
        dec.tokens.fill_(t)
        dec.step(torch.cuda.current_stream().cuda_stream)
        want.append(dec.logits[0].clone())
    want = torch.stack(want).cpu().numpy()
    for t in range(len(toks)):
        assert O.rel_frobenius(got[t], want[t]) <= 1e-2, t
    _no_error()


def test_hybrid_decoder_on_the_8_bit_cache_replays(torch):
    """Recurrent and attention layers together, eager and as a graph."""
    from firepit_b200.model import Decoder, HybridConfig, HybridModel
    cfg = HybridConfig(layers=4, hidden=256, vocab=512, full_attention_interval=2, q_heads=4, kv_heads=2, head_dim=64,
                       rotary_dim=16, key_heads=2, value_heads=4, key_head_dim=32, value_head_dim=32, experts=8,
                       top_k=2, moe_inter=128)
    m = HybridModel(cfg, seed=3)
    prompt = torch.tensor([[1, 2, 3, 4, 5], [9, 8, 7, 6, 5]], dtype=torch.int32, device="cuda")
    dec = Decoder(m, 2, 24, history_len=6, kv8=True)
    s = torch.cuda.current_stream().cuda_stream
    for t in range(prompt.shape[1]):
        dec.tokens.copy_(prompt[:, t])
        dec.step(s)
    dec.step_ctr.zero_()
    for _ in range(6):
        dec.step(s)
    torch.cuda.synchronize()
    eager = dec.history.clone()
    dec.reset()
    dec.capture()
    dec.reset()
    dec.prefill(prompt)
    dec.generate(6)
    torch.cuda.synchronize()
    assert torch.equal(dec.history, eager)
    _no_error()


def test_tree_logits_are_each_branch_s_own(torch, model):
    """Every node of a tree gets the logits that its line alone gets, token by
    token; the rows of the context were fed as a chain."""
    from firepit_b200.model import SpeculativeDecoder
    dec = SpeculativeDecoder(model, 2, 8, 64)
    context = [[3, 14, 15, 92, 65, 35, 89, 79, 32, 38, 46], [26, 43, 38, 32, 79, 50, 28, 84, 19, 71, 69]]
    dec.feed(torch.tensor(context, dtype=torch.int32, device="cuda"))
    assert dec.positions.tolist() == [11, 11]
    tree = np.array([[100, 7, 8, 9, 10, 11, 12, 13], [200, 1, 2, 3, 4, 5, 0, 0]], np.int32)
    par = np.array([[-1, 0, 0, 1, 1, 2, 5, 3], [-1, 0, 1, 2, 0, 4, -2, -2]], np.int32)
    dec.tree.copy_(torch.from_numpy(tree))
    dec.parents.copy_(torch.from_numpy(par))
    dec.step(torch.cuda.current_stream().cuda_stream)
    got = dec.logits.view(2, 8, -1).cpu().numpy()
    from oracle import speculative as R
    for s in range(2):
        for node, line in enumerate(R.ancestors(par[s])):
            if line is not None:
                want = _chain_logits(torch, model, context[s] + [int(tree[s, j]) for j in line], True)[-1]
                assert O.rel_frobenius(got[s, node], want) <= 1e-2, (s, node)
    _no_error()


def test_a_step_emits_what_it_accepts_and_leaves_the_cache_in_order(torch, model):
    """Drafts that hold the model's own continuation on a later branch: the step
    emits it whole, and the next step goes on from a cache in order."""
    from firepit_b200.model import Decoder, SpeculativeDecoder
    prompt = torch.tensor([[7, 1, 9, 30, 2]], dtype=torch.int32, device="cuda")
    plain = Decoder(model, 1, 64, history_len=12, kv8=True)
    plain.capture()
    plain.reset()
    plain.prefill(prompt)
    first = int(plain.tokens[0])
    plain.generate(11)
    greedy = [first] + plain.history[0, :11].tolist()
    dec = SpeculativeDecoder(model, 1, 8, 64)
    dec.feed(prompt[:, :-1])
    dec.tree.copy_(torch.tensor([[2, 500, 501, greedy[0], 502, greedy[1], greedy[2], 503]], dtype=torch.int32))
    dec.parents.copy_(torch.tensor([[-1, 0, 0, 0, 3, 3, 5, 5]], dtype=torch.int32))
    sh = torch.cuda.current_stream().cuda_stream
    dec.step(sh)
    assert dec.path[0].tolist() == [0, 3, 5, 6, -1, -1, -1, -1] and dec.count.item() == 4
    assert dec.emitted[0].tolist() == greedy[:4] + [-1] * 4 and dec.positions.item() == 8
    assert dec.tree[0, 0].item() == greedy[3]
    dec.parents.fill_(-2)
    dec.parents[:, 0] = -1
    dec.step(sh)
    assert dec.emitted[0, :2].tolist() == [greedy[4], -1] and dec.positions.item() == 9
    _no_error()


def test_generation_with_drafts_equals_greedy_decoding(torch, model):
    """Look-up drafts, drafts that are right by half and no drafts: the same
    tokens, in fewer steps where drafts are right."""
    from firepit_b200.model import SpeculativeDecoder, lookup_drafts
    prompt = torch.tensor([[4, 8, 15, 16, 23, 42, 4, 8], [1, 2, 3, 1, 2, 3, 1, 2]], dtype=torch.int32, device="cuda")
    dec = SpeculativeDecoder(model, 2, 6, 96)
    steps = [0]
    inner = dec.step
    dec.step = lambda sh: (steps.__setitem__(0, steps[0] + 1), inner(sh))[1]
    want = dec.generate(prompt, 24, lambda h, n: ([], []))
    slow, steps[0] = steps[0], 0
    got = dec.generate(prompt, 24, lookup_drafts)
    assert [g[:24] for g in got] == [w[:24] for w in want]
    full = {tuple(p): p + w for p, w in zip(prompt.tolist(), want)}

    def half_right(history, nodes):  # the true continuation as a chain, with its third token wrong every other time
        line = next(f for p, f in full.items() if tuple(history[:8]) == p)
        drafts = line[len(history):len(history) + nodes - 1]
        if len(history) % 2 and len(drafts) > 2:
            drafts = drafts[:2] + [(drafts[2] + 1) % 512] + drafts[3:]
        return drafts, list(range(len(drafts)))

    steps[0] = 0
    got = dec.generate(prompt, 20, half_right)
    assert [g[:20] for g in got] == [w[:20] for w in want]
    assert steps[0] < slow - 8
    _no_error()


def test_sampled_generation_is_a_graph_too(torch, model):
    """Above temperature 0 with given random numbers: eager and replayed steps
    emit the same tokens."""
    from firepit_b200.model import SpeculativeDecoder
    outs = []
    for graph in (False, True):
        dec = SpeculativeDecoder(model, 2, 4, 64, temperature=0.9)
        gen = torch.Generator(device="cuda").manual_seed(5)
        sh = torch.cuda.current_stream().cuda_stream
        if graph:
            dec.step(sh)
            dec.reset()
            dec.capture()
            dec.reset()
        dec.feed(torch.tensor([[1, 2, 3], [4, 5, 6]], dtype=torch.int32, device="cuda"))
        dec.tree[:, 0] = 7
        got = []
        for k in range(5):
            dec.draw(gen)
            dec.parents.copy_(torch.tensor([[-1, 0, 0, 1]] * 2, dtype=torch.int32))
            dec.tree[:, 1:] = torch.tensor([[11 + k, 12, 13], [14, 15 + k, 16]], dtype=torch.int32, device="cuda")
            dec.graph.replay() if graph else dec.step(sh)
            got.append(dec.emitted.tolist())
        outs.append(got)
    assert outs[0] == outs[1]
    _no_error()


def test_a_session_without_a_tree_keeps_its_place(torch, model):
    """A session whose node 0 is absent for a step: no token, no row, no error,
    and it goes on after it as if the step had not been."""
    from firepit_b200.model import SpeculativeDecoder
    sh = torch.cuda.current_stream().cuda_stream
    runs = []
    for parked in (False, True):
        dec = SpeculativeDecoder(model, 2, 4, 64)
        dec.feed(torch.tensor([[3, 14, 15], [92, 65, 35]], dtype=torch.int32, device="cuda"))
        dec.tree[:, 0] = torch.tensor([7, 8], dtype=torch.int32)
        dec.parents.copy_(torch.tensor([[-1, -2, -2, -2]] * 2, dtype=torch.int32))
        if parked:
            dec.parents[1, 0] = -2
            dec.step(sh)
            assert dec.count.tolist() == [1, 0] and dec.positions.tolist() == [4, 3]
            assert dec.emitted[1].tolist() == [-1] * 4 and dec.tree[1, 0].item() == 8
            dec.parents[1, 0], dec.parents[0, 0] = -1, -2
        else:
            dec.parents[0, 0] = -2
        got = []
        for _ in range(4):
            dec.step(sh)
            got.append(dec.emitted[1, 0].item())
        runs.append((got, dec.positions[1].item()))
    assert runs[0] == runs[1] and min(runs[0][0]) >= 0
    _no_error()


@pytest.mark.parametrize("fast", [0, 1])
def test_generation_of_sessions_that_advance_unevenly(torch, model, fast):
    """One session's drafts are all taken and the other's none, in the smallest
    cache that is accepted: every returned token is greedy decoding's."""
    from firepit_b200.model import SpeculativeDecoder
    new, nodes = 40, 8
    prompt = torch.tensor([[4, 8, 15, 16, 23, 42, 4, 8], [1, 2, 3, 1, 2, 3, 1, 2]], dtype=torch.int32, device="cuda")
    want = SpeculativeDecoder(model, 2, nodes, 128).generate(prompt, new + nodes, lambda h, n: ([], []))
    dec = SpeculativeDecoder(model, 2, nodes, prompt.shape[1] + new + 2 * nodes)
    start, line = prompt[fast].tolist(), prompt[fast].tolist() + want[fast]
    asked = [0, 0]

    def drafter(history, n):
        mine = history[:len(start)] == start
        asked[0 if mine else 1] += 1
        drafts = line[len(history):len(history) + n - 1] if mine else [(history[-1] + 1) % 512] * (n - 1)
        return drafts, list(range(len(drafts)))

    got = dec.generate(prompt, new, drafter)
    assert len(got[fast]) >= new and len(got[1 - fast]) >= new
    for g, w in zip(got, want):
        assert len(g) <= len(w) and g == w[:len(g)]
    assert asked[0] <= new // nodes + 2 and asked[1] > new // 2  # a session that has its tokens is not drafted for
    assert max(dec.positions.tolist()) <= prompt.shape[1] + new + nodes
    _no_error()


def test_generation_reports_a_device_error(torch, model):
    """What a kernel records while tokens are made is raised, not left behind."""
    import firepit_b200 as F
    from firepit_b200.model import SpeculativeDecoder
    prompt = torch.tensor([[1, 2, 3]], dtype=torch.int32, device="cuda")
    dec = SpeculativeDecoder(model, 1, 4, 64)
    with pytest.raises(RuntimeError, match="50[145]"):
        dec.generate(prompt, 4, lambda h, n: ([5], [3]))  # node 1's parent is a later node
    assert F.device_error(reset=True) == 504
    assert len(dec.generate(prompt, 4, lambda h, n: ([], []))[0]) >= 4
    _no_error()


def test_a_step_keeps_to_its_stream(torch, model):
    """Steps on a side stream that still has work ahead of them, issued while
    torch's current stream is another: the results are those of the current
    stream's, once the side stream alone is done."""
    from firepit_b200.model import SpeculativeDecoder
    tree = torch.tensor([[7, 8, 9, 10], [11, 12, 13, 14]], dtype=torch.int32, device="cuda")
    par = torch.tensor([[-1, 0, 0, 1]] * 2, dtype=torch.int32, device="cuda")
    runs = []
    for side in (None, torch.cuda.Stream()):
        dec = SpeculativeDecoder(model, 2, 4, 64)
        dec.feed(torch.tensor([[3, 14, 15], [92, 65, 35]], dtype=torch.int32, device="cuda"))
        got, stream = [], side or torch.cuda.current_stream()
        for _ in range(3):
            dec.tree[:, 1:].copy_(tree[:, 1:])
            dec.parents.copy_(par)
            torch.cuda.synchronize()
            if side:
                with torch.cuda.stream(side):  # some milliseconds of work ahead of the step
                    big = torch.zeros(1 << 28, device="cuda")
                    for _ in range(20):
                        big.add_(1.0)
            dec.step(stream.cuda_stream)
            stream.synchronize()
            got.append((dec.emitted.tolist(), dec.positions.tolist(), dec.tree[:, 0].tolist()))
        runs.append(got)
    assert runs[0] == runs[1]
    _no_error()


def test_a_step_with_drawn_drafts(torch, model):
    """``draft`` through the decoder: the walk is the definition's on the step's own
    logits, eager and captured; what does not fit is refused, and a step captured
    with other probabilities is dropped."""
    import firepit_b200 as F
    from firepit_b200.model import SpeculativeDecoder
    from oracle import speculative as R
    vocab, par = model.cfg.vocab, [[-1, 0, 0, 1], [-1, 0, 1, 1]]
    dec = SpeculativeDecoder(model, 2, 4, 64, temperature=0.9)
    gen = torch.Generator(device="cuda").manual_seed(6)
    sh, draft = torch.cuda.current_stream().cuda_stream, torch.empty(2, 4, vocab, device="cuda")
    for bad in (draft[:, :3], draft[..., 1:], draft.double(), draft.cpu(), draft[:1]):
        with pytest.raises(F.ShapeError):
            dec.draft = bad
    assert dec.draft is None
    dec.step(sh)
    dec.capture()
    dec.draft = draft
    assert not hasattr(dec, "graph")
    dec.step(sh)
    dec.capture()
    dec.draft = draft  # the same: the captured step stays
    dec.reset()
    dec.feed(torch.tensor([[1, 2, 3], [4, 5, 6]], dtype=torch.int32, device="cuda"))
    lengths = set()
    for k in range(8):
        dec.draw(gen)
        # flat and peaked drafts by turns; the children drawn from their parents' rows
        draft.copy_(torch.softmax(torch.randn(2, 4, vocab, generator=gen, device="cuda") * (k % 4), -1))
        dec.parents.copy_(torch.tensor(par, dtype=torch.int32))
        up = dec.parents.clamp(min=0).long()
        drawn = torch.multinomial(draft.view(8, vocab), 4, True, generator=gen).view(2, 4, 4)
        dec.tree[:, 1:] = torch.gather(drawn.permute(0, 2, 1), 2, up[..., None]).squeeze(2)[:, 1:].int()
        tokens = dec.tree.cpu().numpy().copy()
        dec.graph.replay() if k % 2 else dec.step(sh)
        logits, q = dec.logits.view(2, 4, vocab).cpu().numpy(), draft.cpu().numpy()
        for s in range(2):
            path, token = R.verify(logits[s], tokens[s], par[s], dec.temperature, dec.accept[s].cpu().numpy(),
                                   dec.noise[s].cpu().numpy(), q[s])
            assert dec.path[s].tolist() == path + [-1] * (4 - len(path)) and dec.next[s].item() == token
            assert dec.tree[s, 0].item() == token
            lengths.add(len(path))
    assert len(lengths) > 1
    _no_error()


@pytest.mark.parametrize("length", [1, 4, 5, 9])
def test_prefill_leads_to_the_first_token(torch, model, length):
    """The decoder's prefill on the speculative one: chunks of four rows, whole or
    not, and a prompt of one token; the steps after it emit greedy decoding's
    tokens, with what an earlier step left in the tree."""
    from firepit_b200.model import Decoder, SpeculativeDecoder
    prompt = torch.tensor([[7, 1, 9, 30, 2, 8, 8, 1, 3], [4, 8, 15, 16, 23, 42, 4, 8, 5]], dtype=torch.int32,
                          device="cuda")[:, :length].contiguous()
    plain = Decoder(model, 2, 64, history_len=8, kv8=True)
    plain.capture()
    plain.reset()
    plain.prefill(prompt)
    first = plain.tokens.tolist()
    plain.generate(3)
    want = [[f] + h[:3] for f, h in zip(first, plain.history.tolist())]
    dec = SpeculativeDecoder(model, 2, 4, 64)
    sh = torch.cuda.current_stream().cuda_stream
    dec.tree.fill_(77)
    dec.parents.copy_(torch.tensor([[-1, 0, 0, 0]] * 2, dtype=torch.int32))
    dec.step(sh)
    dec.positions.zero_()
    dec.prefill(prompt)
    assert dec.positions.tolist() == [length - 1] * 2
    got = []
    for _ in range(4):
        dec.step(sh)
        assert dec.count.tolist() == [1, 1]
        got.append(dec.emitted[:, 0].tolist())
    assert [list(g) for g in zip(*got)] == want
    _no_error()
