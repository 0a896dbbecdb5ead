"""Paged 4-bit key/value cache: what is stored, and attention over it, against 64-bit restatements."""
import numpy as np
import pytest
import torch

import cortexsdr_b200 as cs
from cortexsdr_b200 import _lib
from tests import operator_refs as ref

pytestmark = pytest.mark.gpu
THETA = 1e6
DTYPES = {"f32": (torch.float32, 0), "bf16": (torch.bfloat16, 1), "f16": (torch.float16, 2)}


class Case:
    """A ragged batch over a paged cache, with what each sequence holds."""

    def __init__(self, ctx, lengths, fresh, kvh, hd, page, seed=0, dtype="f32", spare=0, tail=0, layers=1, ptr_pages=None):
        self.rng = np.random.default_rng(seed)
        self.ctx, self.lengths, self.fresh, self.kvh, self.hd, self.page, self.tail = ctx, lengths, fresh, kvh, hd, page, tail
        self.tdtype, self.dtype = DTYPES[dtype]
        n = len(lengths)
        counts = [-(-max(a, 0) // page) for a in lengths]
        self.per = max(1, max(counts)) + spare
        self.n_pages = max(1, sum(counts))
        order = self.rng.permutation(self.n_pages)
        self.pages = np.full((n, self.per), -1, np.int32)
        at = 0
        for s, c in enumerate(counts):
            self.pages[s, :c] = order[at:at + c]
            at += c
        self.cache = cs.KVCache(self.n_pages, page, kvh, hd, layers=layers, rope_theta=THETA, ctx=ctx)
        self.k = [self.values((max(a, 0), kvh, hd)) for a in lengths]
        self.v = [self.values((max(a, 0), kvh, hd)) for a in lengths]

    def values(self, shape):
        x = self.rng.normal(0, 1, shape) * (1 + 3 * (self.rng.random(shape[-2:]) < 0.05))
        return torch.tensor(x, dtype=torch.float32).to(self.tdtype)

    def batch(self, lengths, fresh, tail=0):
        first = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
        dev = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in (first, lengths, self.pages)]
        b = cs.KVBatch(len(lengths), int(first[-1]) + tail, *[t.data_ptr() for t in dev], self.per)
        b.keep = dev
        return b

    def rows(self, parts, tail=0, fill=0.0):
        x = torch.cat([p for p in parts if p.shape[0]] + [torch.full((tail, *parts[0].shape[1:]), fill, dtype=parts[0].dtype)])
        return x.cuda().contiguous()

    def store(self, rotate=False, layer=0):
        """Everything into the cache, each sequence's tokens in two calls."""
        for lo, hi in ((0, 2), (2, 3)):
            a = [n * lo // 3 for n in self.lengths]
            e = [n * hi // 3 for n in self.lengths]
            b = self.batch(e, [y - x for x, y in zip(a, e)])
            k, v = (self.rows([t[x:y] for t, x, y in zip(src, a, e)]) for src in (self.k, self.v))
            torch.cuda.synchronize()
            self.cache.append(b, k.data_ptr(), v.data_ptr(), self.dtype, rotate=rotate, layer=layer)
            self.ctx.synchronize()

    def held(self, rotated=False):
        def f(t, turn):
            x = t.to(torch.float64).numpy()
            return ref.held(ref.rotate(x, np.arange(len(x)), THETA) if turn else x) if len(x) else x
        return [f(t, rotated) for t in self.k], [f(t, False) for t in self.v]

    def attend(self, q, qh, layer=0, **kw):
        out = torch.full_like(q, 7.0)
        torch.cuda.synchronize()
        self.cache.attention(self.batch(self.lengths, self.fresh, self.tail), q.data_ptr(), self.dtype, qh, out.data_ptr(), layer=layer, **kw)
        self.ctx.synchronize()
        return out


def close(out, want, tdtype, largest, widened=None):
    """fp32 arithmetic: a score's error is at most sum |q k| scale 2^-21 (two 11-bit halves of q, fp32 sums), here
    under 64 * 16 * 2^-21 / 8 < 1e-4 of a weight for the loudest rows, an output that times the largest value; and
    half a step of the output's type. `widened` (bf16 prompts, whose keys, values and weights are operands in fp16): what their
    roundings come to, operator_refs.widened_bound; on the whole such an output is bf16's: its roundings are spread over
    half a step, 2^-8 / sqrt(3) of the value at most, and a quarter of that again."""
    half = 2.0 ** -24 if tdtype == torch.float32 else torch.finfo(tdtype).eps / 2
    bound = half * np.abs(want) + 1e-4 * largest
    if widened is not None:
        bound = bound + (1 + half) * widened
    err = np.abs(out.to(torch.float64).cpu().numpy() - want)
    assert (err <= bound).all(), f"off by up to {np.nanmax(err - bound)} past the bound"
    if tdtype == torch.float32:
        # the errors of many terms do not all point one way: over all rows, fp32's own
        assert np.linalg.norm(err) <= 4e-6 * np.linalg.norm(want) + 1e-30
    if widened is not None:
        # (fp16: the roundings of weights times steps come to about as much as the output's)
        assert np.linalg.norm(err) <= (1.25 if tdtype == torch.bfloat16 else 4) * half / 3 ** 0.5 * np.linalg.norm(want)


def bound_of(c, fresh, qh, hd, q, k, v, pos, scale):
    """widened_bound where the call's operands are widened: bf16, heads of at most 128, 96 query rows of a kv head a
    sequence; steps_bound where fp16 rows go by sixteen."""
    rows = sum(fresh) * (qh // c.kvh) // len(fresh)
    if c.tdtype == torch.float16 and hd <= 128 and rows >= 192:
        return ref.steps_bound(q.to(torch.float64).numpy(), k, v, pos, scale)
    if c.tdtype != torch.bfloat16 or hd > 128 or rows < 96:
        return None
    return ref.widened_bound(q.to(torch.float64).numpy(), k, v, pos, scale)


SHAPES = [
    # lengths, new tokens, kv heads, query heads, head_dim, page
    ([1], [1], 1, 1, 64, 16),
    ([17], [1], 2, 14, 64, 16),
    ([512], [1], 2, 14, 64, 64),
    ([5, 64, 65, 1, 200], [1, 1, 1, 1, 1], 4, 4, 128, 64),
    ([1024, 3, 700], [1, 1, 1], 8, 32, 128, 64),
    ([130, 33], [1, 1], 2, 32, 256, 32),
    ([5000], [1], 1, 8, 128, 128),
    ([9, 100, 40], [9, 0, 40], 2, 6, 128, 16),
    ([300, 77], [100, 77], 2, 8, 64, 32),
    ([1000], [333], 1, 16, 128, 64),
    ([70, 129], [70, 65], 3, 15, 256, 16),
    ([2048, 513], [3, 17], 2, 8, 128, 256),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,kvh,page", [(64, 3, 16), (128, 2, 64), (256, 1, 32)])
def test_append_holds_what_the_definition_says(ctx, hd, kvh, page, dtype):
    c = Case(ctx, [7, 0, 90, 33], [7, 0, 90, 33], kvh, hd, page, seed=hd, dtype=dtype)
    qh = 5
    q = [c.values((n, qh, hd)) for n in c.lengths]
    b = c.batch(c.lengths, c.fresh)
    dq, dk, dv = c.rows(q), c.rows(c.k), c.rows(c.v)
    q_out = torch.empty_like(dq)
    k_out, v_out = (torch.empty(dk.shape, dtype=torch.float32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    c.cache.append(b, dk.data_ptr(), dv.data_ptr(), c.dtype, q_ptr=dq.data_ptr(), q_heads=qh, q_out_ptr=q_out.data_ptr())
    c.cache.read(b, k_out.data_ptr(), v_out.data_ptr())
    ctx.synchronize()
    k, v = c.held(rotated=True)
    np.testing.assert_array_equal(k_out.cpu().numpy(), np.concatenate(k).astype(np.float32))
    np.testing.assert_array_equal(v_out.cpu().numpy(), np.concatenate(v).astype(np.float32))
    want = np.concatenate([ref.rotate(t.to(torch.float64).numpy(), np.arange(len(t)), THETA) for t in q])
    half = torch.finfo(c.tdtype).eps / 2
    assert (np.abs(q_out.to(torch.float64).cpu().numpy() - want) <= 1.01 * half * np.abs(want) + 1e-6).all()


def test_append_at_far_positions(ctx):
    n, far = 5, 100_000
    c = Case(ctx, [far + n], [n], 1, 128, 64, seed=3)
    k, v = c.values((n, 1, 128)).cuda(), c.values((n, 1, 128)).cuda()
    b = c.batch([far + n], [n])
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    torch.cuda.synchronize()
    c.cache.append(b, k.data_ptr(), v.data_ptr(), 0)
    c.cache.read(b, ko.data_ptr(), vo.data_ptr())
    ctx.synchronize()
    want = ref.held(ref.rotate(k.cpu().numpy(), far + np.arange(n), THETA))
    np.testing.assert_array_equal(ko.cpu().numpy(), want.astype(np.float32))


def test_append_takes_strided_rows_and_queries_in_place(ctx):
    c = Case(ctx, [40, 21], [40, 21], 2, 128, 16, seed=4, dtype="bf16")
    qh, t = 4, 61
    rows = c.values((t, qh + 4 + 3, 128)).cuda()       # q | k | v | padding
    keep = rows.clone()
    b = c.batch(c.lengths, c.fresh)
    ko, vo = (torch.empty(t, 2, 128, device="cuda") for _ in range(2))
    stride, es = rows.stride(0), 2
    torch.cuda.synchronize()
    c.cache.append(b, rows.data_ptr() + qh * 128 * es, rows.data_ptr() + (qh + 2) * 128 * es, 1, kv_stride=stride, q_ptr=rows.data_ptr(),
                   q_stride=stride, q_heads=qh, q_out_ptr=rows.data_ptr(), q_out_stride=stride)
    c.cache.read(b, ko.data_ptr(), vo.data_ptr())
    ctx.synchronize()
    pos = np.concatenate([np.arange(40), np.arange(21)])
    x = keep.to(torch.float64).cpu().numpy()
    np.testing.assert_array_equal(ko.cpu().numpy(), ref.held(ref.rotate(x[:, qh:qh + 2], pos, THETA)).astype(np.float32))
    np.testing.assert_array_equal(vo.cpu().numpy(), ref.held(x[:, qh + 2:qh + 4]).astype(np.float32))
    want = ref.rotate(x[:, :qh], pos, THETA)
    assert (np.abs(rows[:, :qh].to(torch.float64).cpu().numpy() - want) <= 2.0 ** -8 * 1.01 * np.abs(want) + 1e-6).all()
    assert torch.equal(rows[:, qh:], keep[:, qh:])


def test_append_odd_element_offsets(ctx):
    # operands that start between 16-byte boundaries, rows of an odd number of elements
    for dtype in ("f32", "f16"):
        c = Case(ctx, [19], [19], 1, 64, 16, seed=5, dtype=dtype)
        room = torch.zeros(19 * 201 + 1, dtype=c.tdtype, device="cuda")
        rows = room[1:].view(19, 201)
        rows[:, :128] = c.values((19, 2, 64)).view(19, 128).cuda()
        b = c.batch(c.lengths, c.fresh)
        ko, vo = (torch.empty(19, 1, 64, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        es = room.element_size()
        c.cache.append(b, rows.data_ptr(), rows.data_ptr() + 64 * es, c.dtype, kv_stride=201, rotate=False)
        c.cache.read(b, ko.data_ptr(), vo.data_ptr())
        ctx.synchronize()
        x = rows.to(torch.float64).cpu().numpy()
        np.testing.assert_array_equal(ko.cpu().numpy()[:, 0], ref.held(x[:, :64]).astype(np.float32))
        np.testing.assert_array_equal(vo.cpu().numpy()[:, 0], ref.held(x[:, 64:128]).astype(np.float32))


def test_append_borders(ctx):
    # constant groups, ties between codes, saturation, and values that are not finite
    c = Case(ctx, [6], [6], 1, 64, 16)
    k = np.zeros((6, 1, 64), np.float32)
    k[0] = 1.25
    k[1, 0] = np.arange(64) % 31 / 2.0                    # step 1: halves are ties
    k[2, 0, 3] = 1e6
    k[3, 0, 5] = np.nan
    k[4, 0, 7] = -np.inf
    k[5, 0] = np.linspace(-3e-7, 3e-7, 64)                # the step is a subnormal fp16 or nothing
    dk = torch.tensor(k).cuda()
    ko, vo = torch.empty_like(dk), torch.empty_like(dk)
    b = c.batch([6], [6])
    torch.cuda.synchronize()
    c.cache.append(b, dk.data_ptr(), dk.data_ptr(), 0, rotate=False)
    c.cache.read(b, ko.data_ptr(), vo.data_ptr())
    ctx.synchronize()
    np.testing.assert_array_equal(vo.cpu().numpy(), ref.held(k).astype(np.float32))
    np.testing.assert_array_equal(ko.cpu().numpy(), vo.cpu().numpy())


def test_append_touches_its_slots_only(ctx):
    # idle sequences, rows behind the last, tokens without a place: nothing else changes
    c = Case(ctx, [20, 33, 16], [20, 33, 16], 2, 64, 16, seed=6)
    c.store()
    whole = c.batch(c.lengths, c.lengths)
    before = [torch.empty(sum(c.lengths), 2, 64, device="cuda") for _ in range(2)]
    c.cache.read(whole, *[t.data_ptr() for t in before])
    ctx.synchronize()
    good = c.pages.copy()
    c.pages[1, 2] = -1                       # sequence 1: position 32 has no place
    c.pages[2, 0] = c.n_pages                # sequence 2: no such page
    b = c.batch([20, 33, 16], [0, 2, 3], tail=4)
    k, v = c.values((9, 2, 64)).cuda(), c.values((9, 2, 64)).cuda()
    ko, vo = torch.full_like(k, 5.0), torch.full_like(v, 5.0)
    torch.cuda.synchronize()
    c.cache.append(b, k.data_ptr(), v.data_ptr(), 0, rotate=False)
    c.cache.read(b, ko.data_ptr(), vo.data_ptr())
    c.pages = good
    after = [torch.empty_like(t) for t in before]
    c.cache.read(whole, *[t.data_ptr() for t in after])
    ctx.synchronize()
    for old, new, src in zip(before, after, (k, v)):
        want = old.cpu().numpy()
        want[20 + 31] = ref.held(src[:1].cpu().numpy())[0]       # position 31 of sequence 1
        np.testing.assert_array_equal(new.cpu().numpy(), want)
    assert (ko[5:] == 5).all() and (vo[5:] == 5).all()           # rows of no sequence
    assert (ko[1:5] == 0).all()                                  # rows without a place


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_matches_the_definition(ctx, shape, dtype):
    lengths, fresh, kvh, qh, hd, page = shape
    c = Case(ctx, lengths, fresh, kvh, hd, page, seed=len(lengths) + qh, dtype=dtype, spare=2, tail=3)
    c.store()
    q = [c.values((n, qh, hd)) * 0.7 for n in fresh]
    out = c.attend(c.rows(q, c.tail), qh)
    k, v = c.held()
    at = 0
    for s, n in enumerate(fresh):
        if n:
            pos = lengths[s] - n + np.arange(n)
            want = ref.attention(q[s].to(torch.float64).numpy(), k[s], v[s], pos, hd ** -0.5)
            close(out[at:at + n], want, c.tdtype, np.abs(v[s]).max(), bound_of(c, fresh, qh, hd, q[s], k[s], v[s], pos, hd ** -0.5))
        at += n
    assert (out[at:] == 7).all()             # rows behind the last sequence


@pytest.mark.parametrize("n,most_new,dtype", [(33, 1, "f32"), (150, 1, "bf16"), (300, 1, "f32"), (40, 9, "f16"), (140, 30, "bf16")])
def test_attention_of_many_sequences(ctx, n, most_new, dtype):
    rng = np.random.default_rng(n)
    fresh = [0 if i % 9 == 4 else int(rng.integers(1, most_new + 1)) for i in range(n)]
    lengths = [f + int(rng.integers(0, 200)) for f in fresh]
    c = Case(ctx, lengths, fresh, 2, 64, 16, seed=n, dtype=dtype)
    c.store()
    qh = 6
    q = [c.values((f, qh, 64)) for f in fresh]
    out = c.attend(c.rows(q), qh)
    k, v = c.held()
    at = 0
    for s, f in enumerate(fresh):
        if f:
            pos = lengths[s] - f + np.arange(f)
            want = ref.attention(q[s].to(torch.float64).numpy(), k[s], v[s], pos, 0.125)
            close(out[at:at + f], want, c.tdtype, max(1.0, np.abs(v[s]).max()), bound_of(c, fresh, qh, 64, q[s], k[s], v[s], pos, 0.125))
        at += f


def test_attention_sees_what_has_a_place(ctx):
    # a page that is not there inside a sequence, a length past the table, a length that is less than the new rows
    c = Case(ctx, [100, 64, 2, 0], [1, 1, 5, 3], 2, 64, 16, seed=8)
    c.store()
    k, v = c.held()
    qh = 6
    q = [c.values((n, qh, 64)) for n in c.fresh]
    c.pages[0, 2], c.pages[0, 4] = -1, c.n_pages + 5
    c.lengths = [100, 64 + 3 * 16 * c.per, 2, 0]
    out = c.attend(c.rows(q), qh).cpu().numpy()
    keep = np.r_[0:32, 48:64, 80:100]
    np.testing.assert_allclose(out[:1], ref.attention(q[0].numpy(), k[0][keep], v[0][keep], [len(keep) - 1], 0.125), rtol=0, atol=2e-5)
    np.testing.assert_allclose(out[1:2], ref.attention(q[1].numpy(), k[1], v[1], [63], 0.125), rtol=0, atol=2e-5)
    want = ref.attention(q[2].numpy(), k[2], v[2], [-3, -2, -1, 0, 1], 0.125)
    np.testing.assert_allclose(out[2:7], want, rtol=0, atol=2e-5)
    assert (out[2:5] == 0).all() and (out[7:] == 0).all()


def test_attention_does_not_see_later_tokens(ctx):
    # NaN and loud values behind a sequence's end, in the same pages
    c = Case(ctx, [64], [64], 1, 128, 64, seed=9)
    c.k[0][37:] = float("nan")
    c.v[0][37:] = float("nan")
    c.k[0][37, 0, :64] = 6e4
    c.store()
    k, v = c.held()
    for n, length in ((1, 37), (5, 37), (37, 37)):
        c.lengths, c.fresh = [length], [n]
        q = [c.values((n, 8, 128))]
        out = c.attend(c.rows(q), 8)
        close(out, ref.attention(q[0].numpy(), k[0], v[0], length - n + np.arange(n), 128 ** -0.5), torch.float32, np.abs(v[0][:37]).max())
    c.lengths, c.fresh = [40], [4]
    out = c.attend(c.rows([c.values((4, 8, 128))]), 8)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1:]).all()


@pytest.mark.parametrize("vscale,qscale", [(1e-6, 1.0), (1e-3, 30.0), (2000.0, 1e-4), (1.0, 0.0)])
def test_attention_keeps_its_precision_at_any_magnitude(ctx, vscale, qscale):
    c = Case(ctx, [700], [2], 2, 128, 64, seed=10)
    c.v[0] = c.v[0] * vscale
    c.v[0][300:320] = c.v[0][300:320] * 20          # steps grow on the way
    c.store()
    q = [c.values((2, 8, 128)) * qscale]
    out = c.attend(c.rows(q), 8).to(torch.float64).cpu().numpy()
    k, v = c.held()
    want = ref.attention(q[0].numpy(), k[0], v[0], [698, 699], 128 ** -0.5)
    # sharp rows (|q| 30): a score of ~500 carries 2^-21 of itself
    tol = 4e-6 if qscale < 10 else 1e-3
    assert np.linalg.norm(out - want) <= tol * np.linalg.norm(want)


def test_attention_strides_scale_and_layers(ctx):
    c = Case(ctx, [90, 20], [3, 1], 2, 64, 16, seed=11, layers=3)
    c.store(layer=2)
    qh = 4
    rows = c.values((4, qh + 2, 64)).cuda()
    out = torch.full((4, qh + 1, 64), 7.0, device="cuda")
    torch.cuda.synchronize()
    c.cache.attention(c.batch(c.lengths, c.fresh), rows.data_ptr(), 0, qh, out.data_ptr(), q_stride=(qh + 2) * 64, out_stride=(qh + 1) * 64,
                      scale=0.3, layer=2)
    ctx.synchronize()
    k, v = c.held()
    q = rows[:, :qh].cpu().numpy()
    want = np.concatenate([ref.attention(q[:3], k[0], v[0], [87, 88, 89], 0.3), ref.attention(q[3:], k[1], v[1], [19], 0.3)])
    close(out[:, :qh], want, torch.float32, 16.0)
    assert (out[:, qh:] == 7).all()
    zeros = c.attend(rows[:, :qh].contiguous(), qh, layer=0)       # nothing was stored there: zero keys and values
    assert (zeros == 0).all()


def test_attention_repeats_itself_and_follows_a_stream(ctx):
    lengths = [3000, 11, 700, 64] * 5
    c = Case(ctx, lengths, [1] * 20, 2, 128, 64, seed=12)
    c.store()
    q = c.rows([c.values((1, 16, 128)) for _ in lengths])
    a, b = c.attend(q, 16), c.attend(q, 16)
    assert torch.equal(a, b)
    side = torch.cuda.Stream()
    other = cs.Context(0, side.cuda_stream)
    d = Case(other, lengths, [1] * 20, 2, 128, 64, seed=12)
    d.store()
    batch, out = d.batch(lengths, [1] * 20), torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        x = torch.empty_like(q)
        x.copy_(q)                           # the operator's input is made on its stream
        d.cache.attention(batch, x.data_ptr(), 0, 16, out.data_ptr())
        y = out * 2
    side.synchronize()
    assert torch.equal(y, a * 2)
    d.cache.close()
    other.close()


def test_graph_replays_with_new_lengths(ctx):
    side = torch.cuda.Stream()
    own = cs.Context(0, side.cuda_stream)
    c = Case(own, [150, 90], [1, 1], 2, 128, 16, seed=13)
    qh = 8
    b = c.batch([1, 1], [1, 1])
    kv = [torch.empty(2, 2, 128, device="cuda") for _ in range(2)]
    q, qr, out = (torch.empty(2, qh, 128, device="cuda") for _ in range(3))
    torch.cuda.synchronize()

    def step():
        c.cache.append(b, kv[0].data_ptr(), kv[1].data_ptr(), 0, q_ptr=q.data_ptr(), q_heads=qh, q_out_ptr=qr.data_ptr())
        c.cache.attention(b, qr.data_ptr(), 0, qh, out.data_ptr())

    with torch.cuda.stream(side):
        step()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            step()
    queries = [c.values((150, qh, 128)), c.values((90, qh, 128))]
    got = []
    for i in range(150):
        at = [i, min(i, 89)]
        with torch.cuda.stream(side):
            b.keep[1].copy_(torch.tensor([a + 1 for a in at], dtype=torch.int32))
            for s in range(2):
                kv[0][s].copy_(c.k[s][at[s]])
                kv[1][s].copy_(c.v[s][at[s]])
                q[s].copy_(queries[s][at[s]])
            g.replay()
            got.append(out.cpu())
    k, v = c.held(rotated=True)
    for s, n in ((0, 150), (1, 90)):
        qq = ref.rotate(queries[s].numpy(), np.arange(n), THETA)
        want = ref.attention(qq, k[s], v[s], np.arange(n), 128 ** -0.5)
        close(torch.stack([got[i][s] for i in range(n)]), want, torch.float32, 16.0)
    del g
    c.cache.close()
    own.close()


def test_refusals(ctx, lib):
    with pytest.raises(ValueError, match="power of two"):
        cs.KVCache(4, 24, 1, 64, ctx=ctx)
    with pytest.raises(cs.CompressionError, match="head_dim"):
        cs.KVCache(4, 16, 1, 96, ctx=ctx)
    with pytest.raises(ValueError, match="zero"):
        cs.KVCache(0, 16, 1, 64, ctx=ctx)
    with pytest.raises(ValueError, match="finite"):
        cs.KVCache(4, 16, 1, 64, rope_theta=float("nan"), ctx=ctx)
    c = Case(ctx, [16], [16], 2, 64, 16)
    b = c.batch([16], [16])
    x = torch.zeros(16, 4, 64, device="cuda")
    p = x.data_ptr()
    plain = cs.KVCache(1, 16, 2, 64, rope_theta=0.0, ctx=ctx)
    with pytest.raises(ValueError, match="rotation"):
        plain.append(b, p, p, 0)
    for call, what in [
        (lambda: c.cache.append(b, p, p, 3), "dtype"),
        (lambda: c.cache.append(b, p, p, 0, layer=1), "layer"),
        (lambda: c.cache.append(b, 0, p, 0), "null"),
        (lambda: c.cache.append(b, p, p, 0, kv_stride=127), "stride"),
        (lambda: c.cache.append(b, p, p, 0, q_ptr=p, q_heads=4), "q_out"),
        (lambda: c.cache.append(b, p, p, 0, q_ptr=p, q_out_ptr=p), "head count"),
        (lambda: c.cache.attention(b, p, 0, 3, p), "multiple"),
        (lambda: c.cache.attention(b, p, 0, 0, p), "multiple"),
        (lambda: c.cache.attention(b, p, 0, 4, 0), "null"),
        (lambda: c.cache.attention(b, p, 0, 4, p, scale=float("inf")), "scale"),
        (lambda: c.cache.attention(b, p, 7, 4, p), "dtype"),
        (lambda: c.cache.read(b, p, 0), "null"),
        (lambda: c.cache.read(cs.KVBatch(1, 16, 0, 0, 0, 1), p, p), "null array"),
        (lambda: c.cache.read(cs.KVBatch(1, 16, p, p, p, 0), p, p), "range"),
    ]:
        with pytest.raises(ValueError, match=what):
            call()
    before = ctx.launch_count
    c.cache.append(cs.KVBatch(0, 0, 0, 0, 0, 1), 0, 0, 0)          # nothing to do
    c.cache.attention(cs.KVBatch(1, 0, 0, 0, 0, 1), 0, 0, 4, 0)
    assert ctx.launch_count == before
    assert lib.csdr_kv_cache_read_device_async(None, 0, b._ref, p, p) == _lib.ERR_INVALID_ARG


def test_refuses_pointers_inside_an_element_and_angles_without_a_bound(ctx):
    c = Case(ctx, [16], [16], 2, 64, 16)
    b = c.batch([16], [16])
    x = torch.zeros(16, 5, 64, device="cuda")
    p = x.data_ptr()
    off = cs.KVBatch(1, 16, p + 2, p, p, 1)
    for call in [
        lambda: c.cache.append(b, p + 2, p, 0), lambda: c.cache.append(b, p, p + 1, 1), lambda: c.cache.append(b, p, p + 1, 2),
        lambda: c.cache.append(b, p, p, 0, q_ptr=p + 2, q_heads=4, q_out_ptr=p),
        lambda: c.cache.append(b, p, p, 0, q_ptr=p, q_heads=4, q_out_ptr=p + 3),
        lambda: c.cache.append(off, p, p, 0), lambda: c.cache.read(off, p, p), lambda: c.cache.read(b, p + 2, p),
        lambda: c.cache.attention(b, p + 2, 0, 4, p), lambda: c.cache.attention(b, p, 1, 4, p + 1), lambda: c.cache.attention(off, p, 0, 4, p),
    ]:
        with pytest.raises(ValueError, match="whole element"):
            call()
    with pytest.raises(ValueError, match="stride is another"):
        c.cache.append(b, p, p, 0, q_ptr=p, q_stride=256, q_heads=4, q_out_ptr=p, q_out_stride=260)
    with pytest.raises(ValueError, match="at least 1"):
        cs.KVCache(4, 16, 1, 64, rope_theta=0.5, ctx=ctx)
    c.cache.close()


@pytest.mark.parametrize("fresh", [1, 40])
def test_negative_scale(ctx, fresh):
    c = Case(ctx, [150, 40], [fresh, fresh], 2, 128, 32, seed=5)
    c.store(rotate=False)
    qs = [c.values((fresh, 4, 128)) for _ in range(2)]
    got = c.attend(c.rows(qs), 4, scale=-0.05)
    hk, hv = c.held()
    want = np.concatenate([ref.attention(q.to(torch.float64).numpy(), k, v, np.arange(n - fresh, n), -0.05) for q, k, v, n in zip(qs, hk, hv, c.lengths)])
    close(got, want, torch.float32, 16.0)


@pytest.mark.parametrize("dtype,fresh", [("f32", 1), ("bf16", 200)])
def test_a_wait_that_runs_out_is_reported_and_leaves_the_cache_usable(dtype, fresh):
    """The shortest limit: whether it runs out or not, a later call with the usual one is right."""
    own = cs.Context(0)
    c = Case(own, [9000, 500, 2000], [fresh] * 3, 2, 128, 64, seed=6, dtype=dtype)
    c.store(rotate=False)
    q = c.rows([c.values((fresh, 8, 128)) for _ in range(3)])
    want = c.attend(q, 8)
    own.set_wait_limits(barrier_rounds=1)
    for _ in range(3):
        try:
            got = c.attend(q, 8)
        except cs.CudaError:
            continue
        assert torch.equal(got, want)
    own.set_wait_limits()
    assert torch.equal(c.attend(q, 8), want)
    c.cache.close()
    own.close()


def prompts(c, qh, scale=None, keep=None, **kw):
    """The call's rows against the definition; keep: positions of sequence 0 that have a page."""
    hd = c.hd
    scale = hd ** -0.5 if scale is None else scale
    qs = [c.values((f, qh, hd)) for f in c.fresh]
    out = c.attend(c.rows(qs, c.tail), qh, scale=scale, **kw)
    k, v = c.held()
    at = 0
    for s, (n, f) in enumerate(zip(c.lengths, c.fresh)):
        pos = n - f + np.arange(f)
        kk, vv = k[s], v[s]
        if s == 0 and keep is not None:
            kk, vv, pos = kk[keep], vv[keep], np.array([(keep <= t).sum() - 1 for t in pos])
        if f:
            want = ref.attention(qs[s].to(torch.float64).numpy(), kk, vv, pos, scale)
            close(out[at:at + f], want, c.tdtype, max(1.0, np.nanmax(np.abs(vv), initial=0)), bound_of(c, c.fresh, qh, hd, qs[s], kk, vv, pos, scale))
        at += f
    assert (out[at:] == 7).all()
    return out


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lengths,fresh,kvh,qh,page", [
    ([128], [128], 1, 1, 16),                      # a tile of rows, two blocks of keys
    ([129, 1, 0, 64], [129, 1, 0, 64], 2, 6, 32),  # whole prompts, an idle sequence
    ([70, 400, 65], [17, 130, 65], 1, 7, 64),      # rows that end inside a tile, keys inside a block
    ([3000], [24], 2, 8, 256),                     # few tiles, cut along the keys
    ([40] * 70, [3] * 70, 2, 16, 16),              # more sequences than a warp has lanes; few rows
    ([40] * 45, [13] * 45, 2, 16, 16),             # and many
])
def test_bf16_prompts(ctx, lengths, fresh, kvh, qh, page, hd):
    c = Case(ctx, lengths, fresh, kvh, hd, page, seed=len(lengths) + hd, dtype="bf16", spare=1, tail=5)
    c.store()
    prompts(c, qh)
    prompts(c, qh, scale=-0.03)


def test_bf16_prompts_see_what_has_a_place(ctx):
    c = Case(ctx, [300, 64], [100, 64], 2, 128, 16, seed=21, dtype="bf16", tail=2)
    c.store()
    c.pages[0, 2], c.pages[0, 7], c.pages[0, 13] = -1, c.n_pages + 5, -9
    keep = np.array([t for t in range(300) if t // 16 not in (2, 7, 13)])
    prompts(c, 8, keep=keep)
    # lengths that are less than the new rows: the first see nothing
    c.lengths, c.fresh = [20, 0], [50, 30]
    q = [c.values((f, 8, 128)) for f in c.fresh]
    out = c.attend(c.rows(q), 8)
    assert (out[:30] == 0).all() and (out[50:] == 0).all() and (out[30:50] != 0).any(-1).all()


def test_bf16_prompts_do_not_see_later_tokens(ctx):
    # NaN among values that some rows of a tile see and others do not, in one group of 64; then among keys
    c = Case(ctx, [150], [150], 1, 128, 64, seed=22, dtype="bf16")
    c.v[0][100, 0, 70] = float("nan")
    c.k[0][120, 0, 3] = float("inf")
    c.store()
    k, v = c.held()
    q = [c.values((150, 4, 128))]
    out = c.attend(c.rows(q), 4)
    want = ref.attention(q[0][:100].to(torch.float64).numpy(), k[0], v[0], np.arange(100), 128 ** -0.5)
    close(out[:100], want, torch.bfloat16, np.abs(v[0][:100]).max(), ref.widened_bound(q[0][:100].to(torch.float64).numpy(), k[0], v[0], np.arange(100), 128 ** -0.5))
    assert torch.isfinite(out[100:120, :, :64]).all() and torch.isnan(out[100:, :, 64:]).all() and torch.isnan(out[120:]).all()


@pytest.mark.parametrize("vscale", [1e-6, 3000.0, 65504.0])
def test_bf16_prompts_of_any_magnitude(ctx, vscale):
    c = Case(ctx, [200], [60], 2, 64, 32, seed=23, dtype="bf16")
    c.v[0] = (c.v[0] / c.v[0].abs().max() * vscale).to(torch.bfloat16)
    c.k[0] = c.k[0] / 1024
    c.store()
    q = [c.values((60, 8, 64)) * 1e20, c.values((60, 8, 64)) * 0]
    k, v = c.held()
    for x in q:
        out = c.attend(c.rows([x]), 8, scale=1e-18)
        pos = 140 + np.arange(60)
        want = ref.attention(x.to(torch.float64).numpy(), k[0], v[0], pos, 1e-18)
        bound = ref.widened_bound(x.to(torch.float64).numpy(), k[0], v[0], pos, 1e-18) + 2.0 ** -8 * np.abs(want) + 2.0 ** -24
        assert (np.abs(out.to(torch.float64).cpu().numpy() - want) <= bound).all()


def test_bf16_prompts_strides_layers_and_odd_offsets(ctx):
    c = Case(ctx, [90, 40], [70, 40], 2, 64, 16, seed=24, layers=2, dtype="bf16")
    c.store(layer=1)
    rows = torch.zeros(110 * 6 * 64 + 200, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(rows, 7.0)
    q = c.values((110, 4, 64)).cuda()
    k, v = c.held()
    for off, stride in ((0, 6 * 64), (1, 4 * 64 + 1)):
        rows[off:off + 110 * stride].view(110, stride)[:, :256] = q.view(110, 256)
        torch.cuda.synchronize()
        c.cache.attention(c.batch(c.lengths, c.fresh), rows.data_ptr() + 2 * off, 1, 4, out.data_ptr() + 2 * off, q_stride=stride, out_stride=stride, layer=1)
        ctx.synchronize()
        got = out[off:off + 110 * stride].view(110, stride)
        at = 0
        for s, f in enumerate(c.fresh):
            pos = c.lengths[s] - f + np.arange(f)
            x = q[at:at + f].cpu().to(torch.float64).numpy()
            close(got[at:at + f, :256].reshape(f, 4, 64), ref.attention(x, k[s], v[s], pos, 0.125), torch.bfloat16, 16.0, ref.widened_bound(x, k[s], v[s], pos, 0.125))
            at += f
        assert (got[:, 256:] == 7).all()
        out.fill_(7.0)


def test_captured_bf16_prompts_follow_new_lengths():
    """A graph of append and attention for pieces of prompts, replayed back to back as sequences grow; two caches' graphs in turn."""
    side = torch.cuda.Stream()
    own = cs.Context(0, side.cuda_stream)
    kvh, qh, hd, page, piece, n = 2, 8, 128, 64, 48, 3
    rng = np.random.default_rng(31)
    runs = []
    for _ in range(2):
        per = 4
        cache = cs.KVCache(n * per, page, kvh, hd, rope_theta=THETA, ctx=own)
        first = torch.tensor([0, piece, piece, 2 * piece], dtype=torch.int32, device="cuda")      # the second sequence idles
        length = torch.zeros(n, dtype=torch.int32, device="cuda")
        pages = torch.tensor(rng.permutation(n * per).reshape(n, per), dtype=torch.int32, device="cuda")
        b = cs.KVBatch(n, 2 * piece, first.data_ptr(), length.data_ptr(), pages.data_ptr(), per)
        k, v, q = (torch.zeros(2 * piece, h, hd, dtype=torch.bfloat16, device="cuda") for h in (kvh, kvh, qh))
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
            cache.append(b, k.data_ptr(), v.data_ptr(), 1, rotate=False)
            cache.attention(b, q.data_ptr(), 1, qh, out.data_ptr())
        runs.append((cache, b, first, length, pages, k, v, q, out, g, [], []))
    for step in range(4):
        for cache, b, first, length, pages, k, v, q, out, g, ks, vs in runs:
            with torch.cuda.stream(side):
                for t in (k, v, q):
                    t.copy_(torch.tensor(rng.normal(0, 1, t.shape), dtype=torch.bfloat16))
                length.copy_(torch.tensor([piece * (step + 1), 0, piece * (step + 1)], dtype=torch.int32))
                g.replay()
            ks.append(k.cpu())
            vs.append(v.cpu())
        own.synchronize()
        for cache, b, first, length, pages, k, v, q, out, g, ks, vs in runs:
            for i in range(2):
                rows = slice(i * piece, (i + 1) * piece)
                hk, hv = (ref.held(torch.cat([t[rows] for t in src]).to(torch.float64).numpy()) for src in (ks, vs))
                pos = piece * step + np.arange(piece)
                x = q[rows].cpu().to(torch.float64).numpy()
                close(out[rows], ref.attention(x, hk, hv, pos, hd ** -0.5), torch.bfloat16, 5.0, ref.widened_bound(x, hk, hv, pos, hd ** -0.5))
    for cache, *_, g, _, _ in runs:
        del g
        cache.close()
    runs.clear()
    own.close()


@pytest.mark.parametrize("hd,dtype", [(64, "f32"), (128, "f32"), (256, "f32"), (256, "bf16"), (256, "f16"), (64, "f16"), (128, "f16")])
def test_long_prompts(ctx, hd, dtype):
    """Rows enough for warps to have rows of their own."""
    c = Case(ctx, [280, 270], [265, 260], 1, hd, 32, seed=hd, dtype=dtype, tail=2)
    c.store()
    prompts(c, 4)


# the kernels whose warps share rows; have rows of their own, eight or sixteen; prompts on the tensor cores
@pytest.mark.parametrize("dtype,hd,fresh", [("f32", 64, 1), ("f32", 128, 1), ("bf16", 256, 1), ("f16", 128, 1), ("f32", 128, 300), ("f16", 64, 60),
                                            ("f16", 128, 60), ("bf16", 64, 60), ("bf16", 128, 60), ("bf16", 256, 300)])
def test_waits_that_are_given_up(dtype, hd, fresh):
    """Every wait is given up with copies on their way: the call says so, units that CTAs share are arrived at all the same, and
    the next call finds its counters and the shared memory as it needs them."""
    own = cs.Context(0)
    c = Case(own, [9000, 500, 2000], [fresh] * 3, 2, hd, 64, seed=6, dtype=dtype)
    c.store(rotate=False)
    q = c.rows([c.values((fresh, 8, hd)) for _ in range(3)])
    want = c.attend(q, 8)
    for _ in range(2):
        own.set_wait_limits(barrier_rounds=_lib.WAIT_GIVE_UP)
        for _ in range(2):
            with pytest.raises(cs.CudaError, match="wait ran out"):
                c.attend(q, 8)
        own.set_wait_limits()
        for _ in range(2):
            assert torch.equal(c.attend(q, 8), want)
    c.cache.close()
    own.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,kvh,page", [(64, 3, 16), (128, 2, 64), (256, 1, 32)])
def test_prompts_of_many_tokens_are_held_as_the_definition_says(ctx, hd, kvh, page, dtype):
    """Enough tokens for a CTA to take four of them: keys, values and queries, with rotation, value for value; a sequence that
    goes on far behind its start, an idle one, rows of no sequence; then the same without rotation, queries copied."""
    many = 16 * torch.cuda.get_device_properties(0).multi_processor_count
    qh, tail, far = 3, 3, 70_001
    fresh = [many - 700, 0, 650, 59]
    lengths = [many - 700, 7, far + 650, 59]
    assert sum(fresh) >= many and sum(fresh) % 4
    c = Case(ctx, lengths, fresh, kvh, hd, page, seed=hd, dtype=dtype)
    new = [slice(n - f, n) for n, f in zip(lengths, fresh)]
    q = [c.values((f, qh, hd)) for f in fresh]
    dq, dk, dv = c.rows(q, tail, 5.0), c.rows([t[n] for t, n in zip(c.k, new)], tail, 5.0), c.rows([t[n] for t, n in zip(c.v, new)], tail, 5.0)
    b = c.batch(lengths, fresh, tail)
    t = sum(fresh)
    pos = [np.arange(n.start, n.stop) for n in new]
    half = torch.finfo(c.tdtype).eps / 2
    for rotate in (True, False):
        q_out = torch.full_like(dq, 7.0)
        k_out, v_out = (torch.full(dk.shape, 7.0, dtype=torch.float32, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        c.cache.append(b, dk.data_ptr(), dv.data_ptr(), c.dtype, rotate=rotate, q_ptr=dq.data_ptr(), q_heads=qh, q_out_ptr=q_out.data_ptr())
        c.cache.read(b, k_out.data_ptr(), v_out.data_ptr())
        ctx.synchronize()
        turned = lambda x, p: ref.rotate(x.to(torch.float64).numpy(), p, THETA) if rotate else x.to(torch.float64).numpy()
        want_k = np.concatenate([ref.held(turned(x[n], p)) for x, n, p in zip(c.k, new, pos) if len(p)])
        want_v = np.concatenate([ref.held(x[n].to(torch.float64).numpy()) for x, n, p in zip(c.v, new, pos) if len(p)])
        np.testing.assert_array_equal(k_out[:t].cpu().numpy(), want_k.astype(np.float32))
        np.testing.assert_array_equal(v_out[:t].cpu().numpy(), want_v.astype(np.float32))
        want_q = np.concatenate([turned(x, p) for x, p in zip(q, pos) if len(p)])
        got_q = q_out[:t].to(torch.float64).cpu().numpy()
        if rotate:
            # cos and sin are off by 2^-24.9, two products and their sum round: 2.6 2^-24 (|x0| + |x1|); then half a step of the
            # type: 2^-11 of a fp16 value, and under 2^-14, where its steps are 2^-24 however small it is, 2^-25
            smallest = 2.0 ** -25 if c.tdtype == torch.float16 else 0.0
            x = np.abs(np.concatenate([a.to(torch.float64).numpy() for a in q if len(a)]))
            both = np.repeat(x[..., 0::2] + x[..., 1::2], 2, axis=-1)
            assert (np.abs(got_q - want_q) <= np.maximum(half * np.abs(want_q), smallest) + (1 + half) * 2.6 * 2.0 ** -24 * both).all()
        else:
            np.testing.assert_array_equal(got_q, want_q)
        for out in (q_out, k_out, v_out):
            assert (out[t:] == 7).all()


@pytest.mark.parametrize("dtype,prompt,singles", [("bf16", 300, 31), ("bf16", 1100, 31), ("f16", 300, 31), ("f16", 1000, 12), ("f32", 300, 31),
                                                  ("f32", 1100, 2)])
def test_a_prompt_among_single_tokens(ctx, dtype, prompt, singles):
    """One call for both, on either side of the mean of rows that chooses the kernel; an idle sequence counts among them."""
    rng = np.random.default_rng(prompt + singles)
    lengths = [prompt + 100] + [int(n) for n in rng.integers(1, 400, singles)] + [50]
    fresh = [prompt] + [1] * singles + [0]
    c = Case(ctx, lengths, fresh, 2, 128, 32, seed=prompt, dtype=dtype, spare=1, tail=3)
    c.store()
    prompts(c, 8)


def test_fp32_sums_do_not_drift(ctx):
    """Over 1024 keys of ordinary scores the outputs are no further off than those of fp32 products and sums, a quarter to spare
    (sums that are cut off instead of rounded were twice as far)."""
    torch.backends.cuda.matmul.allow_tf32 = False
    n, length, heads, hd = 16, 1024, 32, 128
    for seed in range(3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        loud = lambda: 1.0 + 3.0 * (torch.rand(heads, hd, generator=gen, device="cuda") < 0.05)
        k, v = (torch.randn(n * length, heads, hd, generator=gen, device="cuda") * loud() for _ in range(2))
        q = 1.5 * torch.randn(n, heads, hd, generator=gen, device="cuda")
        cache = cs.KVCache(n * length // 64, 64, heads, hd, rope_theta=0.0, ctx=ctx)
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        lens, pages = ints([length] * n), ints(rng_pages(seed, n, length // 64))
        whole, last = ints([length * i for i in range(n + 1)]), ints(list(range(n + 1)))
        batch = lambda f, t: cs.KVBatch(n, t, f.data_ptr(), lens.data_ptr(), pages.data_ptr(), length // 64)
        out, hk, hv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        torch.cuda.synchronize()
        cache.append(batch(whole, n * length), k.data_ptr(), v.data_ptr(), 0, rotate=False)
        cache.read(batch(whole, n * length), hk.data_ptr(), hv.data_ptr())
        cache.attention(batch(last, n), q.data_ptr(), 0, heads, out.data_ptr())
        ctx.synchronize()

        def attend(x):
            kk, vv = (a.to(x).view(n, length, heads, hd).transpose(1, 2) for a in (hk, hv))
            s = torch.matmul(kk, q.to(x)[..., None])[..., 0] / hd ** 0.5
            e = torch.exp(s - s.amax(-1, keepdim=True))
            return (torch.matmul(e[:, :, None], vv)[:, :, 0] / e.sum(-1, keepdim=True)).to(torch.float64)

        want = attend(torch.float64)
        own, plain = (float((a.to(torch.float64) - want).norm() / want.norm()) for a in (out, attend(torch.float32)))
        assert own <= 1.25 * plain, (own, plain)
        cache.close()


def rng_pages(seed, n, per):
    return np.random.default_rng(seed).permutation(n * per).reshape(n, per).tolist()


@pytest.mark.parametrize("dtype,hd,fresh", [("f32", 128, 1), ("f32", 64, 260), ("f16", 128, 60), ("bf16", 128, 60), ("bf16", 256, 3)])
def test_pages_and_layers_past_32_bits(ctx, dtype, hd, fresh):
    """Two layers of more than 4 GB each, pages at their ends."""
    kvh, page = 8, 256
    each = kvh * page // 16 * 18 * hd
    n_pages = (1 << 32) // each + 40
    c = Case(ctx, [700, 300], [fresh, min(fresh, 300)], kvh, hd, page, seed=9, dtype=dtype)
    c.cache.close()
    c.cache = cs.KVCache(n_pages, page, kvh, hd, layers=2, rope_theta=THETA, ctx=ctx)
    assert c.cache.nbytes > 2 << 32
    c.pages = np.where(c.pages >= 0, c.pages + n_pages - c.n_pages, -1).astype(np.int32)
    c.store(layer=1)
    qs = [c.values((f, 4 * kvh, hd)) for f in c.fresh]
    out = c.attend(c.rows(qs), 4 * kvh, layer=1)
    k, v = c.held()
    at = 0
    for s, (n, f) in enumerate(zip(c.lengths, c.fresh)):
        pos = n - f + np.arange(f)
        want = ref.attention(qs[s].to(torch.float64).numpy(), k[s], v[s], pos, hd ** -0.5)
        close(out[at:at + f], want, c.tdtype, np.abs(v[s]).max(), bound_of(c, c.fresh, 4 * kvh, hd, qs[s], k[s], v[s], pos, hd ** -0.5))
        at += f
    b = c.batch([700, 300], [700, 300])
    ko, vo = (torch.empty(1000, kvh, hd, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    c.cache.read(b, ko.data_ptr(), vo.data_ptr(), layer=1)
    ctx.synchronize()
    np.testing.assert_array_equal(ko.cpu().numpy(), np.concatenate(k).astype(np.float32))
    np.testing.assert_array_equal(vo.cpu().numpy(), np.concatenate(v).astype(np.float32))
    c.cache.read(b, ko.data_ptr(), vo.data_ptr(), layer=0)
    ctx.synchronize()
    assert (ko == 0).all() and (vo == 0).all()
    c.cache.close()


@pytest.mark.parametrize("dtype,group", [("f32", 2), ("bf16", 2), ("bf16", 64)])
def test_strides_past_32_bits(ctx, dtype, group):
    """Rows of q, k, v and the results 2^31 elements apart."""
    hd, rows, stride = 64, 3, (1 << 31) + 16
    c = Case(ctx, [40 + rows], [rows], 1, hd, 16, seed=10, dtype=dtype)
    wide = torch.empty((rows - 1) * stride + (2 * group + 4) * hd, dtype=c.tdtype, device="cuda")
    es = wide.element_size()
    part = lambda at, heads: torch.as_strided(wide, (rows, heads, hd), (stride, hd, 1), at * hd)
    b = c.batch([40], [40])
    old_k, old_v = (t[0][:40].cuda() for t in (c.k, c.v))
    new = [c.values((rows, h, hd)) for h in (group, 1, 1)]
    for at, t in zip((0, group, group + 1), new):
        part(at, t.shape[1]).copy_(t.cuda())
    part(group + 2, group).fill_(7.0)
    torch.cuda.synchronize()
    c.cache.append(b, old_k.data_ptr(), old_v.data_ptr(), c.dtype, rotate=False)
    b = c.batch([40 + rows], [rows])
    p = wide.data_ptr()
    c.cache.append(b, p + group * hd * es, p + (group + 1) * hd * es, c.dtype, kv_stride=stride, rotate=False, q_ptr=p, q_stride=stride,
                   q_heads=group, q_out_ptr=p, q_out_stride=stride)
    c.cache.attention(b, p, c.dtype, group, p + (group + 2) * hd * es, q_stride=stride, out_stride=stride)
    ctx.synchronize()
    k, v = (ref.held(torch.cat([t[0][:40], x]).to(torch.float64).numpy()) for t, x in ((c.k, new[1]), (c.v, new[2])))
    q = new[0].to(torch.float64).numpy()
    assert torch.equal(part(0, group).cpu(), new[0])
    pos = 40 + np.arange(rows)
    close(part(group + 2, group), ref.attention(q, k, v, pos, hd ** -0.5), c.tdtype, np.abs(v).max(),
          bound_of(c, [rows], group, hd, new[0], k, v, pos, hd ** -0.5))
    c.cache.close()


@pytest.mark.parametrize("dtype,fresh", [("f32", 1), ("f32", 260), ("bf16", 1), ("bf16", 60)])
def test_queries_of_the_greatest_magnitude(ctx, dtype, fresh):
    """Queries up to the type's largest number, with a scale that brings scores back to where they tell keys apart."""
    c = Case(ctx, [300], [fresh], 2, 128, 32, seed=11, dtype=dtype)
    c.store()
    k, v = c.held()
    pos = 300 - fresh + np.arange(fresh)
    for top in (2.0 ** 122, 2.0 ** 125, 3e38):
        q = c.values((fresh, 8, 128)).to(torch.float64)
        scale = float(np.float32(float(q.abs().max()) / top / 128 ** 0.5))
        q = (q * (top / q.abs().max())).to(c.tdtype)
        out = c.attend(c.rows([q]), 8, scale=scale)
        x = q.to(torch.float64).numpy()
        close(out, ref.attention(x, k[0], v[0], pos, scale), c.tdtype, np.abs(v[0]).max(), bound_of(c, [fresh], 8, 128, q, k[0], v[0], pos, scale))
    # scores past fp32: the greatest alone weighs
    q = torch.sign(c.values((fresh, 8, 128)).to(torch.float64)) * 3e38
    out = c.attend(c.rows([q.to(c.tdtype)]), 8)
    x = q.to(c.tdtype).to(torch.float64).numpy()
    if fresh == 1:
        close(out, ref.attention(x, k[0], v[0], pos, 128 ** -0.5), c.tdtype, np.abs(v[0]).max())
    assert torch.isfinite(out).all()
    c.cache.close()


@pytest.mark.parametrize("dtype,fresh", [("f32", 1), ("f32", 260), ("bf16", 1), ("bf16", 60)])
def test_queries_of_the_least_magnitude(ctx, dtype, fresh):
    """Queries down to numbers that are not normal, with a scale that brings scores up to where they tell keys apart."""
    c = Case(ctx, [300], [fresh], 2, 128, 32, seed=12, dtype=dtype)
    c.store()
    k, v = c.held()
    pos = 300 - fresh + np.arange(fresh)
    for top in (2.0 ** -80, 2.0 ** -100, 2.0 ** -115, 2.0 ** -123):
        q = c.values((fresh, 8, 128)).to(torch.float64)
        scale = float(np.float32(float(q.abs().max()) / top / 128 ** 0.5))
        q = (q * (top / q.abs().max())).to(c.tdtype)
        out = c.attend(c.rows([q]), 8, scale=scale)
        x = q.to(torch.float64).numpy()
        close(out, ref.attention(x, k[0], v[0], pos, scale), c.tdtype, np.abs(v[0]).max(), bound_of(c, [fresh], 8, 128, q, k[0], v[0], pos, scale))
    c.cache.close()


def test_refuses_more_heads_than_queries_can_have(ctx):
    """One page of the smallest: what would fit the device, but no call could attend over."""
    with pytest.raises(ValueError, match="out-of-range"):
        cs.KVCache(1, 16, 65536, 64, ctx=ctx)
    cs.KVCache(1, 16, 65535, 64, ctx=ctx).close()
