"""Host-side checks of speculative decoding over the 8-bit cache: refusals of
the entry points and of their Python wrappers, the oracle's formats."""
import numpy as np
import pytest

import firepit_b200 as F
from firepit_b200 import _native as N


def test_speculative_entry_points_check_arguments_first():
    """The 8-bit cache, tree attention and verification reject bad pointers,
    shapes and workspaces on the host, before any CUDA call."""
    f = 1 << 20  # a 16-byte-aligned address that is never dereferenced
    lib, bad, shape = N.lib, N.FPB_ERR_INVALID_ARGUMENT, N.FPB_ERR_SHAPE

    def append(**kw):
        a = dict(q=f, q_pitch=512, q_head=64, k=f, k_pitch=128, v=f, v_pitch=128, dtype=N.FPB_F32, qg=f, kg=f, pos=f,
                 par=f, batch=2, nodes=4, hq=4, hk=2, d=64, rot=64, theta=1e4, eps=1e-6, max_seq=128, out=f,
                 out_dtype=N.FPB_F32, kc=f, vc=f, ke=f, ve=f, stream=None)
        assert set(kw) <= set(a)
        return lib.fpb_kv8_append(*dict(a, **kw).values())

    for kw in (dict(k=None), dict(q=None), dict(hq=0), dict(out=None), dict(pos=None), dict(kc=None), dict(kc=f + 8),
               dict(ve=None), dict(dtype=2), dict(out_dtype=7), dict(q=f + 2), dict(out=f + 4), dict(kg=f + 4)):
        assert append(**kw) == bad, kw
    for kw in (dict(d=72), dict(d=272), dict(d=0), dict(batch=0), dict(batch=65536), dict(nodes=0), dict(nodes=65),
               dict(nodes=129, par=None), dict(rot=63), dict(rot=66), dict(theta=0.5), dict(theta=float("nan")),
               dict(k_pitch=127), dict(v_pitch=64), dict(q_head=32), dict(max_seq=0), dict(hk=0)):
        assert append(**kw) == shape, kw
    read = [f, f, f, f, 2, 128, 2, 64, None, 0, 16, f, f, N.FPB_F32, None]
    for i, val, want in ((0, None, bad), (11, None, bad), (12, f + 8, bad), (13, 5, bad), (9, 113, shape),
                         (10, 0, shape), (10, 129, shape), (7, 60, shape)):
        assert lib.fpb_kv8_read(*[val if j == i else x for j, x in enumerate(read)]) == want, (i, val)
    keep = [f, f, f, f, 2, 128, 2, 64, f, f, 4, None]
    for i, val, want in ((8, None, bad), (9, None, bad), (10, 0, shape), (10, 129, shape), (1, f + 1, bad)):
        assert lib.fpb_kv8_keep(*[val if j == i else x for j, x in enumerate(keep)]) == want, (i, val)
    need = lib.fpb_tree_attn_workspace_bytes(2, 4, 4, 2, 64, 128)

    def attn(**kw):
        a = dict(q=f, dtype=N.FPB_F32, q_pitch=256, q_head=64, kc=f, vc=f, ke=f, ve=f, pos=f, par=f, gate=None,
                 gate_pitch=0, gate_head=0, batch=2, nodes=4, hq=4, hk=2, d=64, max_seq=128, scale=0.1, ws=f,
                 ws_bytes=need, out=f, stream=None)
        assert set(kw) <= set(a)
        return lib.fpb_tree_attn(*dict(a, **kw).values())

    for kw in (dict(q=None), dict(kc=None), dict(ke=None), dict(pos=None), dict(ws=None), dict(out=None), dict(dtype=3),
               dict(vc=f + 8), dict(out=f + 8), dict(ws=f + 4), dict(q=f + 1), dict(gate=f + 2, gate_head=64)):
        assert attn(**kw) == bad, kw
    for kw in (dict(hq=3), dict(hq=0), dict(d=40), dict(d=320), dict(nodes=0), dict(nodes=65), dict(batch=0),
               dict(nodes=129, par=None), dict(q_head=32), dict(gate=f, gate_head=32), dict(scale=float("inf")),
               dict(scale=float("nan")), dict(max_seq=0)):
        assert attn(**kw) == shape, kw
    assert need >= 16 and attn(ws_bytes=need - 1) == N.FPB_ERR_WORKSPACE

    def verify(**kw):
        a = dict(logits=f, dtype=N.FPB_F32, pitch=100, draft=None, draft_pitch=0, tokens=f, par=f, accept=f, noise=f,
                 noise_pitch=100, batch=2, nodes=4, vocab=100, temperature=1.0, path=f, count=f, next=f, stream=None)
        assert set(kw) <= set(a)
        return lib.fpb_tree_verify(*dict(a, **kw).values())

    for kw in (dict(logits=None), dict(tokens=None), dict(path=None), dict(count=None), dict(next=None), dict(dtype=4),
               dict(accept=None), dict(noise=None), dict(temperature=-1.0), dict(temperature=float("nan")),
               dict(temperature=float("inf")), dict(temperature=1e-30)):
        assert verify(**kw) == bad, kw
    for kw in (dict(batch=0), dict(batch=65536), dict(nodes=0), dict(nodes=65), dict(vocab=0), dict(pitch=99),
               dict(noise_pitch=99), dict(draft=f, draft_pitch=99)):
        assert verify(**kw) == shape, kw
    assert verify(vocab=442369, pitch=442369, noise_pitch=442369) == N.FPB_ERR_UNSUPPORTED


def test_speculative_wrappers_check_tensors():
    torch = pytest.importorskip("torch")
    cache = F.Kv8Cache.zeros(2, 32, 2, 64, device="cpu")
    assert cache.nbytes() == 2 * (2 * 32 * 2 * 65)
    pos = torch.zeros(2, dtype=torch.int32)
    kv = torch.zeros(2, 4, 2, 64)
    q = torch.zeros(2, 4, 6, 64)
    par = torch.zeros(2, 4, dtype=torch.int32)
    calls = [
        lambda: F.Kv8Cache(cache.k[..., :40], cache.v, cache.k_exp, cache.v_exp),
        lambda: F.Kv8Cache(cache.k, cache.v[:, :, :1], cache.k_exp, cache.v_exp),
        lambda: F.Kv8Cache(cache.k, cache.v, cache.k_exp.float(), cache.v_exp),
        lambda: F.kv8_append(cache, pos, kv[:1], kv[:1]),
        lambda: F.kv8_append(cache, pos, kv, kv.bfloat16()),
        lambda: F.kv8_append(cache, pos.long(), kv, kv),
        lambda: F.kv8_append(cache, pos, kv.half(), kv.half()),
        lambda: F.kv8_append(cache, pos, kv, kv, parents=par[:, :3]),
        lambda: F.kv8_append(cache, pos, kv, kv, q=q.bfloat16()),
        lambda: F.kv8_append(cache, pos, kv, kv, q_out=q),
        lambda: F.kv8_append(cache, pos, kv, kv, q=q, q_gamma=torch.zeros(32)),
        lambda: F.kv8_append(cache, pos, kv.transpose(0, 1).contiguous().transpose(0, 1), kv),
        lambda: F.kv8_read(cache, 0, 0),
        lambda: F.kv8_read(cache, pos[:1], 4),
        lambda: F.kv8_keep(cache, pos, par.long()),
        lambda: F.tree_attention(q[:, :, :5], cache, pos, par),
        lambda: F.tree_attention(q, cache, pos, par, gate=q.bfloat16()),
        lambda: F.tree_attention(q, cache, pos, par, out=q),
        lambda: F.tree_verify(torch.zeros(2, 4, 10), par.long()),
        lambda: F.tree_verify(torch.zeros(2, 65, 10), torch.zeros(2, 65, dtype=torch.int32)),
        lambda: F.tree_verify(torch.zeros(2, 4, 10), par, par, 1.0),
        lambda: F.tree_verify(torch.zeros(2, 4, 10), par, par, 1.0, torch.zeros(2, 4), torch.zeros(2, 9)),
        lambda: F.tree_verify(torch.zeros(4, 2, 10).transpose(0, 1), par),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(F.ShapeError):
            call()
            pytest.fail(f"call {i} was taken")


def test_speculative_oracle_agrees_with_the_formats():
    """The oracle's e4m3 table and rounding against the library's host codec."""
    from oracle import speculative as R
    for c in range(256):
        if c & 0x7f != 0x7f:  # the NaN code, which the host codec reads as 480
            assert N.lib.fpb_e4m3_to_f32(c) == R.E4M3[c]
    assert np.isnan(R.E4M3[[0x7f, 0xff]]).all()
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(500) * 30, [448.0, 17.0, 19.0, 0.0, -1.0625]])
    codes, exps = R.quantise(x[None])
    assert exps[0] == 127
    assert [int(c) for c in codes[0]] == [N.lib.fpb_f32_to_e4m3(float(v)) for v in x]


def test_speculative_decoder_refuses_what_it_cannot_run():
    torch = pytest.importorskip("torch")
    from types import SimpleNamespace

    from firepit_b200.model import HybridConfig, SpeculativeDecoder, lookup_drafts
    full = SimpleNamespace(cfg=HybridConfig(layers=2, full_attention_interval=1), device=torch.device("cpu"))
    hybrid = SimpleNamespace(cfg=HybridConfig(layers=4), device=torch.device("cpu"))
    for model, sessions, nodes, max_seq in ((hybrid, 1, 4, 64), (full, 0, 4, 64), (full, 1, 0, 64), (full, 2, 9, 64),
                                            (full, 1, 8, 7)):
        with pytest.raises(F.ShapeError):
            SpeculativeDecoder(model, sessions, nodes, max_seq)
    assert lookup_drafts([1, 2, 3, 4, 1, 2], 3) == ([3, 4], [0, 1])
    assert lookup_drafts([1, 2, 3], 3) == ([], [])
    assert lookup_drafts([5], 3) == ([], [])


def test_speculative_wrappers_check_devices():
    """Tensors that are right in every other way, but not on a CUDA device: no
    address of theirs reaches a kernel."""
    torch = pytest.importorskip("torch")
    cache = F.Kv8Cache.zeros(2, 32, 2, 64, device="cpu")
    pos = torch.zeros(2, dtype=torch.int32)
    par = torch.zeros(2, 4, dtype=torch.int32)
    q, kv, gamma = torch.zeros(2, 4, 6, 64), torch.zeros(2, 4, 2, 64), torch.ones(64)
    logits, unit = torch.zeros(2, 4, 10), torch.ones(2, 10)
    ws = torch.zeros(F.tree_attention_workspace_bytes(cache, 4, 6), dtype=torch.uint8)
    for call in (lambda: F.kv8_append(cache, pos, kv, kv, q=q, parents=par, q_gamma=gamma, k_gamma=gamma),
                 lambda: F.kv8_append(cache, pos, kv, kv),
                 lambda: F.kv8_read(cache, pos, 4), lambda: F.kv8_read(cache, 0, 4),
                 lambda: F.kv8_keep(cache, pos, par),
                 lambda: F.tree_attention(q, cache, pos, par, gate=q), lambda: F.tree_attention(q, cache, pos),
                 lambda: F.tree_attention(q, cache, pos, par, out=q.bfloat16(), workspace=ws),
                 lambda: F.tree_verify(logits, par, par),
                 lambda: F.tree_verify(logits, par, par, 1.0, torch.zeros(2, 4), unit, draft=logits)):
        with pytest.raises(F.ShapeError, match="device"):
            call()
    with pytest.raises(F.ShapeError, match="workspace"):
        F.tree_attention(q, cache, pos, par, workspace=ws.float())
