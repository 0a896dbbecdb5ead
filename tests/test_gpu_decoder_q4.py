"""The decoder with what it holds in 4 bits: linears stored as q4_k blocks, the paged 4-bit KV cache; and scoring. Against a
plain 64-bit decoder over the same weights, which keeps keys and values as the cache holds them."""
import numpy as np
import pytest
import torch

import cortexsdr_b200 as cs
from tests import operator_refs as ref
from tests.test_gpu_decoder import LOGIT_TOL, _build_model, make_decoder, oracle_forward

pytestmark = pytest.mark.gpu

CFG = dict(n_layers=2, hidden=256, q_heads=4, kv_heads=2, head_dim=64, inter=512, vocab=300)
EPS, THETA = 1e-6, 1e6
RAW = {"token_embd.weight": "q4_k", "output.weight": "q4_k", "blk.0.ffn_down.weight": "q4_k", "blk.0.attn_k.weight": "q4_k",
       "blk.1.attn_q.weight": "q4_k", "blk.1.ffn_up.weight": "q4_k", "blk.1.attn_output.weight": "q4_k"}


@pytest.fixture(scope="module")
def model_packed(tmp_path_factory, oracle):
    return _build_model(tmp_path_factory, oracle, "packed", CFG=CFG, raw_formats=RAW, n_atoms=32, kv_atoms=16)


@pytest.fixture(scope="module")
def model_tc(tmp_path_factory, oracle):
    """Steps of eight tokens or more hand activations on as bf16 planes."""
    return _build_model(tmp_path_factory, oracle, "tcq4", CFG=CFG, n_atoms=128, kv_atoms=128)


def plain(weights, tokens, held):
    """Final logits of every position, (T, vocab)."""
    f = lambda a: np.asarray(a, np.float64)
    norm = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * f(w)
    t, hd = len(tokens), CFG["head_dim"]
    x, pos = f(weights["tok"])[np.asarray(tokens)], np.arange(t)
    for b in weights["blocks"]:
        h = norm(x, b["attn_norm"])
        q, k, v = ((h @ f(b[n]).T).reshape(t, -1, hd) for n in ("wq", "wk", "wv"))
        q, k = ref.rotate(q, pos, THETA), ref.rotate(k, pos, THETA)
        if held:
            k, v = ref.held(k), ref.held(v)
        x = x + ref.attention(q, k, v, pos, hd ** -0.5).reshape(t, -1) @ f(b["wo"]).T
        h = norm(x, b["ffn_norm"])
        g = h @ f(b["w_gate"]).T
        x = x + (g / (1 + np.exp(-g)) * (h @ f(b["w_up"]).T)) @ f(b["w_down"]).T
    return norm(x, weights["out_norm"]) @ f(weights["head"]).T


def test_the_plain_decoder_is_the_oracles(oracle, model_tc):
    tokens = np.random.default_rng(0).integers(0, CFG["vocab"], 9)
    _, logits = oracle_forward(oracle, model_tc[1], tokens, eps=EPS, theta=THETA, CFG=CFG)
    assert np.abs(plain(model_tc[1], tokens, False)[-1] - logits).max() < 1e-3


def test_packed_linears(ctx, oracle, model_packed):
    path, weights = model_packed
    tokens = np.random.default_rng(1).integers(0, CFG["vocab"], 40)
    want = plain(weights, tokens, False)
    dec = make_decoder(path, ctx, CFG=CFG)
    got, _ = dec.forward(tokens[:36])
    assert np.abs(got - want[35]).max() < LOGIT_TOL
    for t in range(36, 40):
        _, lg = dec.step([tokens[t]], want_logits=True)
        assert np.abs(lg[0] - want[t]).max() < LOGIT_TOL
    dec.close()


@pytest.mark.parametrize("which", ["packed", "planes"])
def test_cache_in_four_bits(ctx, model_packed, model_tc, which):
    path, weights = model_packed if which == "packed" else model_tc
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, CFG["vocab"], n) for n in (70, 1, 13, 5, 8, 9, 2, 30, 11)]
    dec = make_decoder(path, ctx, CFG=CFG, max_seq=96, max_batch=9, kv_dtype="q4")
    exact = make_decoder(path, ctx, CFG=CFG, max_seq=96)
    for s, p in enumerate(prompts):
        want = plain(weights, p, True)[-1]
        got, _ = dec.forward(p, seq=s)
        assert np.abs(got - want).max() < LOGIT_TOL, s
    assert np.abs(plain(weights, prompts[0], True)[-1] - exact.forward(prompts[0])[0]).max() > 1e-4      # it is another cache
    # a prompt in two pieces, and steps of all sequences
    more = [rng.integers(0, CFG["vocab"], 3) for _ in prompts]
    got, _ = dec.forward(more[0], seq=0)
    assert np.abs(got - plain(weights, np.r_[prompts[0], more[0]], True)[-1]).max() < LOGIT_TOL
    full = [np.r_[prompts[0], more[0]]] + [np.array(p) for p in prompts[1:]]
    for _ in range(2):
        new = rng.integers(0, CFG["vocab"], len(full))
        _, lg = dec.step(new, want_logits=True)
        full = [np.append(p, n) for p, n in zip(full, new)]
        for s, p in enumerate(full):
            assert np.abs(lg[s] - plain(weights, p, True)[-1]).max() < LOGIT_TOL, s
    dec.reset()
    got, _ = dec.forward(prompts[2], seq=4)
    assert np.abs(got - plain(weights, prompts[2], True)[-1]).max() < LOGIT_TOL
    dec.close()
    exact.close()


def test_captured_steps_over_the_four_bit_cache(model_packed):
    path, _ = model_packed
    side = torch.cuda.Stream()
    own = cs.Context(0, side.cuda_stream)
    prompt = np.random.default_rng(3).integers(0, CFG["vocab"], 20)
    a, b = (make_decoder(path, own, CFG=CFG, max_seq=64, kv_dtype="q4") for _ in range(2))
    first = int(a.forward(prompt)[0].argmax())
    b.forward(prompt)
    want, nxt = [], first
    for _ in range(6):
        nxt = int(a.step([nxt])[0][0])
        want.append(nxt)
    tok = torch.tensor([first], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        b.step_device(tok.data_ptr(), 1, tok.data_ptr())
        side.synchronize()
        got = [int(tok[0])]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            b.step_device(tok.data_ptr(), 1, tok.data_ptr())
        for _ in range(5):
            g.replay()
            side.synchronize()
            got.append(int(tok[0]))
    assert got == want
    del g
    a.close()
    b.close()
    own.close()


@pytest.mark.parametrize("which,kv", [("packed", "f32"), ("planes", "f32"), ("planes", "q4")])
def test_scores(ctx, model_packed, model_tc, which, kv):
    path, weights = model_packed if which == "packed" else model_tc
    tokens = np.random.default_rng(4).integers(0, CFG["vocab"], 100)
    dec = make_decoder(path, ctx, CFG=CFG, max_seq=128, kv_dtype=kv)
    lp, ent, ids, alt = dec.score(tokens[:90], top=5)
    logits = plain(weights, tokens, kv == "q4")
    want = ref.logprobs(logits, np.append(tokens[1:], 0), 5)
    assert np.isnan(lp[89])
    assert np.abs(lp[:89] - want[0][:89]).max() < LOGIT_TOL and np.abs(ent - want[1][:90]).max() < LOGIT_TOL
    assert np.abs(alt - want[3][:90]).max() < LOGIT_TOL
    # an alternative is the token that the plain decoder has there, or one as likely
    assert np.abs(np.take_along_axis(logits - np.log(np.exp(logits).sum(1, keepdims=True)), np.r_[ids, ids[:10]].astype(np.int64), 1)[:90]
                  - want[3][:90]).max() < 2 * LOGIT_TOL
    # the sequence went on; targets of one's own; steps find their logits as before
    lp, ent, ids, alt = dec.score(tokens[90:99], targets=np.full(9, 7))
    want = ref.logprobs(logits[90:99], np.full(9, 7), 0)
    assert np.abs(lp - want[0]).max() < LOGIT_TOL and ids.shape == (9, 0)
    _, lg = dec.step([tokens[99]], want_logits=True)
    assert np.abs(lg[0] - logits[99]).max() < LOGIT_TOL
    with pytest.raises(ValueError, match="at most 32"):
        dec.score(tokens[:2], top=33)
    with pytest.raises(ValueError, match="max_seq"):
        dec.score(tokens[:90])
    with pytest.raises(ValueError, match="one target"):
        dec.score(tokens[:3], targets=[1])
    dec.close()


def test_refuses_heads_the_cache_does_not_take(ctx, tmp_path_factory, oracle):
    cfg = dict(CFG, head_dim=32)
    path, _ = _build_model(tmp_path_factory, oracle, "hd32", CFG=cfg, n_atoms=32, kv_atoms=16)
    with pytest.raises(cs.CompressionError, match="head_dim"):
        make_decoder(path, ctx, CFG=cfg, kv_dtype="q4")


@pytest.mark.parametrize("theta", [0.0, -1.0, 0.5, float("nan"), float("inf")])
def test_refuses_rotations_that_the_cache_does_not_have(ctx, model_packed, theta):
    """When it is made, not at its first step."""
    loader = cs.SDRModelLoader(model_packed[0], ctx)
    with pytest.raises(ValueError, match="rope_theta"):
        cs.Decoder(loader, **CFG, max_seq=64, rms_eps=EPS, rope_theta=theta, kv_dtype="q4")
    dec = cs.Decoder(loader, **CFG, max_seq=64, rms_eps=EPS, rope_theta=1.0, kv_dtype="q4")
    assert np.isfinite(dec.forward([1, 2, 3])[0]).all()
    dec.close()
