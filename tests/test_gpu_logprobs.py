"""Log probabilities of given tokens, entropy and top alternatives against 64-bit restatements."""
import numpy as np
import pytest
import torch

import cortexsdr_b200 as cs
from tests import operator_refs as ref

pytestmark = pytest.mark.gpu
DTYPES = {"f32": (torch.float32, 0), "bf16": (torch.bfloat16, 1), "f16": (torch.float16, 2)}


def run(x, targets, top, ctx, stride=None):
    rows, vocab = x.shape
    xd = x.cuda() if x.device.type == "cpu" else x
    t = torch.tensor(np.asarray(targets), dtype=torch.int32, device="cuda")
    lp, ent = (torch.full((rows + 1,), 7.0, device="cuda") for _ in range(2))
    ids = torch.full((rows + 1, max(top, 1)), 77, dtype=torch.int32, device="cuda")
    alt = torch.full((rows + 1, max(top, 1)), 7.0, device="cuda")
    torch.cuda.synchronize()
    dtype = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[x.dtype]
    cs.token_logprobs_device(xd.data_ptr(), dtype, rows, vocab, t.data_ptr(), lp.data_ptr(), ent.data_ptr(), top, ids.data_ptr(),
                             alt.data_ptr(), stride=xd.stride(0) if rows > 1 else 0, ctx=ctx)
    ctx.synchronize()
    assert lp[-1] == 7 and ent[-1] == 7 and (ids[-1] == 77).all() and (alt[-1] == 7).all()
    return [a[:-1].cpu().numpy() for a in (lp, ent, ids, alt)]


def check(got, x, targets, top):
    """S carries at most a few 2^-22 (exponentials 2^-22 each, sums of at most 300 terms a thread then a tree), its
    logarithm and the two differences 2^-24 of |x - M| each: 1e-5 + 2^-22 |value| covers both; the entropy is two
    numbers of that size."""
    lp, ent, ids, alt = got
    want = ref.logprobs(x.to(torch.float64).cpu().numpy(), targets, top)
    tol = lambda w: 1e-5 + 2.0 ** -22 * np.abs(w)
    assert (np.abs(lp - want[0]) <= tol(want[0])).all()
    assert (np.abs(ent - want[1]) <= 2 * tol(want[1])).all()
    if top:
        np.testing.assert_array_equal(ids[:, :top], want[2])
        assert (np.abs(alt[:, :top] - want[3]) <= tol(want[3])).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 7, 7), (1, 32, 32), (2, 33, 5), (5, 1000, 20), (1, 151936, 5), (17, 32000, 20),
                                            (2, 100003, 32), (200, 4099, 3), (64, 32768, 0), (300, 50257, 10)])
def test_matches_the_definition(ctx, rows, vocab, top, dtype):
    rng = np.random.default_rng(vocab)
    x = torch.tensor(rng.normal(0, 3, (rows, vocab)), dtype=torch.float32)
    x[:, vocab // 2] += 9
    x = x.to(DTYPES[dtype][0])
    targets = rng.integers(0, vocab, rows)
    check(run(x, targets, top, ctx), x, targets, top)


@pytest.mark.parametrize("order", ["rising", "falling", "equal", "two", "blocks"])
def test_orders_that_are_not_random(ctx, order):
    v = 20000
    row = {"rising": np.arange(v) / 1000.0, "falling": -np.arange(v) / 1000.0, "equal": np.full(v, 0.5), "two": np.arange(v) % 2 * 1.0,
           "blocks": (np.arange(v) // 512 % 7) * 1.5}[order]
    x = torch.tensor(np.stack([row, row[::-1].copy()]), dtype=torch.float32)
    check(run(x, [0, v - 1], 32, ctx), x, [0, v - 1], 32)


def test_unaligned_rows_and_strides(ctx):
    rng = np.random.default_rng(3)
    for dtype in (torch.float32, torch.bfloat16):
        for vocab, stride, off in ((1003, 1003, 1), (999, 1100, 3), (8, 9, 1), (5, 5, 2)):
            room = torch.full((6 * stride + 8,), 50.0, dtype=dtype, device="cuda")     # what lies between is louder
            x = room[off:off + 6 * stride].view(6, stride)[:, :vocab]
            x.copy_(torch.tensor(rng.normal(0, 2, (6, vocab))).to(dtype))
            t = rng.integers(0, vocab, 6)
            check(run(x, t, 5, ctx), x, t, 5)


def test_masked_tokens_and_rows_without_a_softmax(ctx):
    rng = np.random.default_rng(4)
    v, inf = 5000, float("inf")
    x = torch.tensor(rng.normal(0, 2, (9, v)), dtype=torch.float32)
    x[0, 10:] = -inf                                   # ten tokens left, twelve asked for
    x[1, 1:] = torch.finfo(torch.float32).min          # masked by the lowest value
    x[2] = -inf
    x[3, 77] = float("nan")
    x[4, 78] = inf
    x[5] = torch.finfo(torch.float32).min
    x[6] = -0.0
    x[6, 100] = 0.0                                    # equal to its neighbours
    x[7, :] = -inf
    x[7, v - 1] = 3.0
    lp, ent, ids, alt = run(x, [3, 0, 1, 2, 3, 4, 5, v - 1, -1], 12, ctx)
    for r in (2, 3, 4):
        assert np.isnan(lp[r]) and np.isnan(ent[r]) and (ids[r] == -1).all() and np.isnan(alt[r]).all()
    for r in (0, 1, 5, 6, 7):
        with np.errstate(invalid="ignore"):
            want = ref.logprobs(np.maximum(x[r:r + 1].numpy().astype(np.float64), -1e300), [[3, 0, 0, 0, 0, 4, 5, v - 1][r]], 12)
        assert abs(lp[r] - want[0][0]) < 1e-5 and abs(ent[r] - want[1][0]) < 2e-5
        np.testing.assert_array_equal(ids[r], want[2][0])
        seen = np.isfinite(x[r].numpy()[want[2][0]])
        np.testing.assert_allclose(alt[r][seen], want[3][0][seen], rtol=2.0 ** -22, atol=1e-5)
        assert (alt[r][~seen] == -inf).all()
    assert np.isnan(lp[8]) and np.isfinite(ent[8]) and ids[8, 0] == int(x[8].argmax())


def test_targets_outside_answer_nan_and_parts_can_be_left_out(ctx):
    x = torch.randn(3, 700, device="cuda")
    t = torch.tensor([700, -100, 5], dtype=torch.int32, device="cuda")
    lp, ent = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    torch.cuda.synchronize()
    cs.token_logprobs_device(x.data_ptr(), 0, 3, 700, t.data_ptr(), lp.data_ptr(), ctx=ctx)
    cs.token_logprobs_device(x.data_ptr(), 0, 3, 700, 0, 0, ent.data_ptr(), ctx=ctx)
    ctx.synchronize()
    want = torch.log_softmax(x.double(), -1)
    assert torch.isnan(lp[:2]).all() and abs(float(lp[2] - want[2, 5])) < 1e-5
    assert torch.allclose(ent.double(), -(want.exp() * want).sum(-1), atol=2e-5)


def test_refusals(ctx):
    x = torch.zeros(2, 10, device="cuda")
    p = x.data_ptr()
    for args, kw, what in [((p, 0, 2, 10, 0, p), {}, "null"), ((0, 0, 2, 10, p, p), {}, "null"), ((p, 9, 2, 10, p, p), {}, "dtype"),
                           ((p, 0, 2, 10, p, p, 0, 11, p, p), {}, "more alternatives"), ((p, 0, 2, 100, p, p, 0, 33, p, p), {}, "at most"),
                           ((p, 0, 2, 10, p, p, 0, 3, p, 0), {}, "null"), ((p, 0, 2, 0, p, p), {}, "range"),
                           ((p, 0, 2, 10, p, p), {"stride": 9}, "stride")]:
        with pytest.raises(ValueError, match=what):
            cs.token_logprobs_device(*args, ctx=ctx, **kw)
    before = ctx.launch_count
    cs.token_logprobs_device(p, 0, 0, 10, 0, 0, ctx=ctx)
    assert ctx.launch_count == before


def test_refuses_pointers_inside_an_element(ctx):
    p = torch.zeros(2, 10, device="cuda").data_ptr()
    for args in [(p + 2, 0, 2, 8, p, p), (p + 1, 1, 2, 8, p, p), (p, 0, 2, 8, p + 2, p), (p, 0, 2, 8, p, p + 1), (p, 0, 2, 8, p, p, p + 3),
                 (p, 0, 2, 8, p, p, 0, 2, p + 2, p), (p, 0, 2, 8, p, p, 0, 2, p, p + 2)]:
        with pytest.raises(ValueError, match="whole element"):
            cs.token_logprobs_device(*args, ctx=ctx)


@pytest.mark.parametrize("rows,vocab", [(2, 50000), (700, 1000)])
def test_on_a_stream_of_its_own_captured_and_replayed(rows, vocab):
    side = torch.cuda.Stream()
    own = cs.Context(0, side.cuda_stream)
    x = torch.zeros(rows, vocab, device="cuda", dtype=torch.bfloat16)
    t = torch.randint(0, vocab, (rows,), dtype=torch.int32, device="cuda")
    lp, ids, alt = torch.zeros(rows, device="cuda"), torch.zeros(rows, 4, dtype=torch.int32, device="cuda"), torch.zeros(rows, 4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            cs.token_logprobs_device(x.data_ptr(), 1, rows, vocab, t.data_ptr(), lp.data_ptr(), 0, 4, ids.data_ptr(), alt.data_ptr(), ctx=own)
        for seed in range(2):
            torch.manual_seed(seed)
            x.copy_(torch.randn(rows, vocab, device="cuda") * 3)
            g.replay()
            side.synchronize()
            want = torch.log_softmax(x.double(), -1)
            # 2e-5: an fp32 sum of `vocab` terms and the logarithm's own rounding, next to values of about 10
            assert (lp.double() - want.gather(1, t.long()[:, None])[:, 0]).abs().max() < 2e-5
            order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :4]
            assert torch.equal(ids.long(), order)
    del g
    own.close()


@pytest.mark.parametrize("dtype,vocab", [("f32", 33000), ("bf16", 70001)])
@pytest.mark.parametrize("top", [0, 7])
def test_rows_around_a_row_an_sm(ctx, dtype, vocab, top):
    """From rows cut in four parts over rows cut in two to rows that are not cut: each row's answer is the same."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    rng = np.random.default_rng(vocab)
    x = torch.tensor(rng.normal(0, 3, (sms + 1, vocab)), dtype=torch.float32).to(DTYPES[dtype][0])
    targets = rng.integers(0, vocab, sms + 1)
    every = run(x, targets, top, ctx)
    check(every, x, targets, top)
    for rows in (sms, sms // 2 + 1, sms // 2, sms // 4 + 1, sms // 4):
        got = run(x[:rows], targets[:rows], top, ctx)
        check(got, x[:rows], targets[:rows], top)
        for a, b in zip(got, every):
            np.testing.assert_allclose(a, b[:rows], rtol=2.0 ** -20, atol=2e-5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_past_32_bits(ctx, dtype):
    rows, vocab, stride = 3, 50001, (1 << 31) + 8
    rng = np.random.default_rng(7)
    x = torch.tensor(rng.normal(0, 3, (rows, vocab)), dtype=torch.float32).to(DTYPES[dtype][0])
    room = torch.empty((rows - 1) * stride + vocab, dtype=x.dtype, device="cuda")
    wide = torch.as_strided(room, (rows, vocab), (stride, 1))
    wide.copy_(x.cuda())
    targets = rng.integers(0, vocab, rows)
    check(run(wide, targets, 20, ctx), x, targets, 20)
