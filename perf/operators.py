"""Operators of a served decoder, as cases that can be timed and checked.

Four operators, each through the package's public entry points where `own` is true and in elementary
torch operations where it is not:

* ``append``  - new keys and values of a ragged batch into a paged cache held in 4 bits (groups of 64 along
  the head: fp16 minimum and step), keys and queries rotated on the way; what was written is read back as the
  values it stands for
* ``attend``  - causal grouped-query attention of the new tokens over that cache
* ``q4``      - products with weights stored in 4 bits (q4_0: 32 weights a scale; q4_k: 256 weights with
  6-bit scales and minima of 32)
* ``logprob`` - log probabilities of given tokens, entropy and the top alternatives of rows of logits
"""
import math

import numpy as np
import torch

own = False

GROUP, THETA = 64, 1e6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _append(name, seqs, context, new, q_heads, kv_heads, head_dim, dtype, ragged, packed, page):
    return dict(name=name, kind="append", seqs=seqs, context=context, new=new, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, dtype=dtype, ragged=ragged, packed=packed, page=page)


def _attend(name, seqs, context, new, q_heads, kv_heads, head_dim, dtype, ragged, page):
    return dict(name=name, kind="attend", seqs=seqs, context=context, new=new, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, dtype=dtype, ragged=ragged, page=page)


def _q4(name, rows, cols, batch, format, dtype, layout):
    return dict(name=name, kind="q4", rows=rows, cols=cols, batch=batch, format=format, dtype=dtype, layout=layout)


def _logprob(name, rows, vocab, top, dtype):
    return dict(name=name, kind="logprob", rows=rows, vocab=vocab, top=top, dtype=dtype)


def listed():
    return [
        # one layer of a decode step: sixteen sequences of a 7B-class decoder, a token each
        _append("append_16x1_32kv", 16, 1024, 1, 32, 32, 128, "f32", False, False, 64),
        # prompts of many users of a decoder with grouped heads, q|k|v rows as one projection leaves them
        _append("append_prompts_8kv_bf16", 13, 2011, 2011, 32, 8, 128, "bf16", True, True, 64),
        # the smallest attention of a step: one sequence of a 0.5B-class decoder
        _attend("attend_1x512_14q2kv", 1, 512, 1, 14, 2, 64, "f32", False, 64),
        # sixteen sequences of a 7B-class decoder at context 1024 (every query head has keys of its own)
        _attend("attend_16x1024_32q32kv", 16, 1024, 1, 32, 32, 128, "f32", False, 64),
        # long contexts of many users, grouped heads, lengths as they come
        _attend("attend_32x8k_32q8kv_bf16", 32, 8192, 1, 32, 8, 128, "bf16", True, 64),
        # pieces of prompts behind what is cached already
        _attend("attend_pieces_512of2k_bf16", 3, 2048, 512, 32, 8, 128, "bf16", True, 32),
        # a query projection of a 0.5B-class decoder for one token
        _q4("q4_0_896x896_m1", 896, 896, 1, "q4_0", "f32", "token"),
        # the MLP of a 7B-class decoder for one token
        _q4("q4_k_11008x4096_m1", 11008, 4096, 1, "q4_k", "f32", "token"),
        # and its way back for sixteen sequences
        _q4("q4_0_4096x11008_m16", 4096, 11008, 16, "q4_0", "bf16", "token"),
        # the alternatives of one sampled token
        _logprob("logprob_1x151936", 1, 151936, 5, "f32"),
        # a decode step of sixteen sequences
        _logprob("logprob_16x32000", 16, 32000, 20, "f32"),
        # a long text scored under the largest vocabulary
        _logprob("logprob_2048x151936_bf16", 2048, 151936, 20, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "q4", "q4", "logprob"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind in ("append", "attend"):
        kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
        q_heads = kv_heads * rng.choice([g for g in (1, 2, 4, 7, 8, 16) if kv_heads * g <= 64])
        head_dim, page, ragged = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128]), rng.random() < 0.7
        if kind == "append":
            seqs = _log(rng, 1, 64)
            new = _log(rng, 1, max(1, min(4096, (1 << 25) // (seqs * (q_heads + 2 * kv_heads) * head_dim))))
            context = new + _log(rng, 1, max(1, min(65536, (1 << 28) // (seqs * kv_heads * head_dim)))) - 1
            return {k: v for k, v in _append("", seqs, context, new, q_heads, kv_heads, head_dim, dtype, ragged,
                                             rng.random() < 0.5, page).items() if k != "name"}
        seqs = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.6 else _log(rng, 2, 512)
        context = max(new, _log(rng, 1, max(1, min(32768, (1 << 28) // (seqs * kv_heads * head_dim)))))
        while seqs * new * context * q_heads * head_dim > 1 << 33 and new > 1:
            new = (new + 1) // 2
        return {k: v for k, v in _attend("", seqs, context, new, q_heads, kv_heads, head_dim, dtype, ragged, page).items()
                if k != "name"}
    if kind == "q4":
        fmt = rng.choice(["q4_0", "q4_k"])
        unit = 32 if fmt == "q4_0" else 256
        cols = unit * max(1, _log(rng, 256, 14336) // unit)
        return {k: v for k, v in _q4("", _log(rng, 64, 32000), cols, _log(rng, 1, 64), fmt, dtype,
                                     rng.choice(["token", "feature"])).items() if k != "name"}
    vocab = _log(rng, 1000, 200000)
    return {k: v for k, v in _logprob("", _log(rng, 1, max(1, min(4096, (1 << 27) // vocab))), vocab, rng.choice([0, 1, 5, 20, 32]),
                                      dtype).items() if k != "name"}


# ---- a ragged batch over a paged cache ----

def _lengths(case):
    """(tokens in the cache with the new ones, new tokens) of every sequence."""
    s, context, new = case["seqs"], case["context"], case["new"]
    if not case["ragged"]:
        return [context] * s, [new] * s
    fresh = [0 if i % 7 == 5 else 1 + (new - 1) * (997 * (i + 1) % 1000) // 1000 for i in range(s)]
    fresh[0] = new
    return [max(n, context - (context // 2) * (613 * i % 1000) // 1000) for i, n in enumerate(fresh)], fresh


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _batch(case, gen):
    """The batch as tensors: first row and length of every sequence, its pages in shuffled order."""
    lengths, fresh = _lengths(case)
    page = case["page"]
    per = max(1, -(-max(lengths) // page))
    counts = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(counts), generator=gen, device="cuda").to(torch.int32)
    used = torch.tensor([[i < n for i in range(per)] for n in counts]).cuda()
    pages = torch.full((case["seqs"], per), -1, dtype=torch.int32, device="cuda")
    pages[used] = order
    first = torch.tensor([0] + list(np.cumsum(fresh)), dtype=torch.int32, device="cuda")
    rows_seq = torch.tensor([s for s, n in enumerate(fresh) for _ in range(n)], dtype=torch.int64, device="cuda")
    rows_new = torch.tensor([j for n in fresh for j in range(n)], dtype=torch.int64, device="cuda")
    rows_pos = torch.tensor([lengths[s] - n + j for s, n in enumerate(fresh) for j in range(n)], dtype=torch.int64, device="cuda")
    return dict(first=first, length=torch.tensor(lengths, dtype=torch.int32, device="cuda"), pages=pages, n_pages=sum(counts),
                tokens=sum(fresh), rows_seq=rows_seq, rows_new=rows_new, rows_pos=rows_pos, most_new=max(fresh), most=max(lengths))


def _context():
    import cortexsdr_b200 as cs
    return cs.default_context()


def _own_batch(b, seqs):
    import cortexsdr_b200 as cs
    return cs.KVBatch(seqs, b["tokens"], b["first"].data_ptr(), b["length"].data_ptr(), b["pages"].data_ptr(), b["pages"].shape[1])


def _own_dtype(case):
    from cortexsdr_b200 import _lib
    return {"f32": _lib.DTYPE_F32, "bf16": _lib.DTYPE_BF16, "f16": _lib.DTYPE_F16}[case["dtype"]]


def _keys(gen, shape, dtype):
    """Keys and values as projections give them: normal, a few channels of every head larger."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    loud = 1.0 + 3.0 * (torch.rand(shape[-2:], generator=gen, device="cuda") < 0.05)
    return (x * loud).to(dtype)


# ---- plain forms ----

def _angles(pos, head_dim):
    i = torch.arange(0, head_dim, 2, dtype=torch.float64, device=pos.device)
    a = pos.to(torch.float64)[:, None] * THETA ** (-i / head_dim)
    return torch.cos(a)[:, None, :], torch.sin(a)[:, None, :]


def _rotated(x, pos):
    """(T, heads, head_dim) with adjacent pairs rotated, in 64 bits."""
    c, s = _angles(pos, x.shape[-1])
    a, b = x[..., 0::2].to(torch.float64), x[..., 1::2].to(torch.float64)
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _quantised(x):
    """Codes, step and minimum of groups of 64 (64-bit input): step and minimum in fp16, codes against both as rounded."""
    g = x.unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1), g.amax(-1)
    minimum = low.to(torch.float32).to(torch.float16)
    step = ((high - low) / 15.0).to(torch.float32).to(torch.float16)
    m, s = minimum.to(torch.float64)[..., None], step.to(torch.float64)[..., None]
    codes = torch.where(s > 0, torch.clamp(torch.round((g - m) / torch.where(s > 0, s, 1.0)), 0, 15), 0.0)
    return codes.to(torch.uint8), step, minimum


def _values(codes, step, minimum):
    v = codes.to(torch.float64) * step.to(torch.float64)[..., None] + minimum.to(torch.float64)[..., None]
    return v.flatten(-2).to(torch.float32)


def _plain_append(st):
    b, x = st["batch"], st["dtype"]
    kv = [_values(*_quantised(t)) for t in (_rotated(st["k"], b["rows_pos"]), st["v"].to(torch.float64))]
    return {"q": _rotated(st["q"], b["rows_pos"]).to(x), "k": kv[0], "v": kv[1]}


def _unpacked(st, which):
    """(sequences, positions, kv heads, head_dim) in 32 bits, gathered through the page table."""
    b = st["batch"]
    pages = b["pages"].clamp(min=0).to(torch.int64)
    codes, step, minimum = (st[which + n][pages].flatten(1, 2)[:, :b["most"]] for n in ("_codes", "_step", "_min"))
    low, high = codes & 15, codes >> 4
    c = torch.stack((low, high), -1).flatten(-2).to(torch.float32).unflatten(-1, (-1, GROUP))
    return (c * step.to(torch.float32)[..., None] + minimum.to(torch.float32)[..., None]).flatten(-2)


def _plain_attend(st):
    b, case = st["batch"], st["case"]
    s, kvh, d, group = case["seqs"], case["kv_heads"], case["head_dim"], case["q_heads"] // case["kv_heads"]
    q = torch.zeros(s, b["most_new"], kvh, group, d, device="cuda")
    q[b["rows_seq"], b["rows_new"]] = st["q"].to(torch.float32).view(-1, kvh, group, d)
    pos = torch.full((s, b["most_new"]), -1, dtype=torch.int64, device="cuda")
    pos[b["rows_seq"], b["rows_new"]] = b["rows_pos"]
    k, v = _unpacked(st, "k"), _unpacked(st, "v")
    score = torch.matmul(q.permute(0, 2, 3, 1, 4).flatten(2, 3), k.permute(0, 2, 3, 1)) / math.sqrt(d)
    score = score.view(s, kvh, group, b["most_new"], -1)
    seen = torch.arange(b["most"], device="cuda")[None, None, :] <= pos[:, :, None]
    score = torch.where(seen[:, None, None], score, float("-inf"))
    high = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isinf(high), 0.0, high))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p.flatten(2, 3), v.permute(0, 2, 1, 3)).view(s, kvh, group, b["most_new"], d)
    return o.permute(0, 3, 1, 2, 4)[b["rows_seq"], b["rows_new"]].flatten(1, 2).to(st["dtype"])


def _weights(payload, rows, cols, fmt, dtype):
    """The matrix that the stored blocks stand for."""
    if fmt == "q4_0":    # fp16 scale, then 32 codes, two a byte, the first in the low half
        p = payload.view(rows, cols // 32, 18)
        d = p[..., :2].contiguous().view(torch.float16).to(dtype)
        c = torch.stack((p[..., 2:] & 15, p[..., 2:] >> 4), -1).flatten(-2)
        return ((c.to(dtype) - 8.0) * d).view(rows, cols)
    # q4_k: fp16 scale of the steps and of the minima, eight 6-bit steps and minima, then runs of 64 codes:
    # 32 low halves, 32 high halves
    p = payload.view(rows, cols // 256, 144)
    d = p[..., :4].contiguous().view(torch.float16).to(dtype)
    a, b, c = p[..., 4:8], p[..., 8:12], p[..., 12:16]
    step = torch.cat((a & 63, (c & 15) | (a >> 6 << 4)), -1).to(dtype) * d[..., :1]
    low = torch.cat((b & 63, (c >> 4) | (b >> 6 << 4)), -1).to(dtype) * d[..., 1:]
    n = p[..., 16:].unflatten(-1, (4, 32))
    code = torch.stack((n & 15, n >> 4), -2).flatten(-3, -2).to(dtype)
    return (code * step[..., None] - low[..., None]).reshape(rows, cols)


def _plain_q4(st):
    case = st["case"]
    w = _weights(st["payload"], case["rows"], case["cols"], case["format"], torch.float32)
    x = st["x"].to(torch.float32)
    return torch.matmul(x, w.t()) if case["layout"] == "token" else torch.matmul(w, x)


def _plain_logprob(st):
    x = st["logits"].to(torch.float32)
    high = x.amax(-1, keepdim=True)
    e = torch.exp(x - high)
    total = e.sum(-1, keepdim=True)
    norm = high + torch.log(total)
    out = {"logprob": (torch.gather(x, 1, st["targets"].to(torch.int64)[:, None]) - norm)[:, 0],
           "entropy": (torch.log(total) - (e * (x - high)).sum(-1, keepdim=True) / total)[:, 0]}
    if st["case"]["top"]:
        order = torch.sort(x, dim=-1, descending=True, stable=True)
        out["ids"] = order.indices[:, :st["case"]["top"]].to(torch.int32)
        out["top"] = order.values[:, :st["case"]["top"]] - norm
    return out


# ---- inputs ----

def _inputs(case, seed):
    """What a case's operator is given; `exact` starts from the same."""
    gen = _generator(seed)
    st = dict(case=case, dtype=DTYPES[case["dtype"]])
    if case["kind"] == "append":
        b = st["batch"] = _batch(case, gen)
        qh, kvh, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        row = _keys(gen, (b["tokens"], qh + 2 * kvh, d), st["dtype"])
        parts = row[:, :qh], row[:, qh:qh + kvh], row[:, qh + kvh:]
        st["q"], st["k"], st["v"] = parts if case["packed"] else [t.contiguous() for t in parts]
    elif case["kind"] == "attend":
        b = st["batch"] = _batch(case, gen)
        st["q"] = (1.5 * torch.randn(b["tokens"], case["q_heads"], case["head_dim"], generator=gen, device="cuda")).to(st["dtype"])
        # the cached rows, all sequences one behind the other
        st["total"] = sum(_lengths(case)[0])
        shape = (st["total"], case["kv_heads"], case["head_dim"])
        st["k"], st["v"] = _keys(gen, shape, torch.bfloat16), _keys(gen, shape, torch.bfloat16)
    elif case["kind"] == "q4":
        rows, cols = case["rows"], case["cols"]
        unit, block = (32, 18) if case["format"] == "q4_0" else (256, 144)
        n = rows * (cols // unit)
        payload = torch.empty(n, block, dtype=torch.uint8, device="cuda")
        scale = 0.006 * torch.exp(0.3 * torch.randn(n, 1, generator=gen, device="cuda"))
        code = (torch.randn(n, unit // 2, 2, generator=gen, device="cuda") * 2.6 + 8).round().clamp(0, 15).to(torch.uint8)
        payload[:, -(unit // 2):] = code[..., 0] | (code[..., 1] << 4)
        if case["format"] == "q4_0":
            payload[:, :2] = scale.to(torch.float16).view(torch.uint8)
        else:
            payload[:, :4] = torch.cat((scale / 40, scale / 5), 1).to(torch.float16).view(torch.uint8)
            payload[:, 4:16] = torch.randint(0, 256, (n, 12), generator=gen, device="cuda", dtype=torch.uint8)
        st["payload"] = payload.flatten()
        shape = (case["batch"], cols) if case["layout"] == "token" else (cols, case["batch"])
        st["x"] = torch.randn(shape, generator=gen, device="cuda").to(st["dtype"])
    else:
        x = 2.5 * torch.randn(case["rows"], case["vocab"], generator=gen, device="cuda")
        likely = torch.randint(0, case["vocab"], (case["rows"], 3), generator=gen, device="cuda")
        x.scatter_add_(1, likely, 6.0 + 6.0 * torch.rand(case["rows"], 3, generator=gen, device="cuda"))
        st["logits"] = x.to(st["dtype"])
        st["targets"] = torch.where(torch.rand(case["rows"], generator=gen, device="cuda") < 0.7, likely[:, 0],
                                    torch.randint(0, case["vocab"], (case["rows"],), generator=gen, device="cuda")).to(torch.int32)
    return st


def _whole(case, b):
    """The batch whose new tokens are all the tokens of every sequence."""
    lengths = b["length"]
    first = torch.zeros(case["seqs"] + 1, dtype=torch.int32, device="cuda")
    first[1:] = torch.cumsum(lengths, 0)
    return dict(b, first=first, tokens=int(first[-1]))


def _paged(st, which, codes, step, minimum):
    """Codes, steps and minima of all sequences' rows in pages, codes two a byte."""
    case, b = st["case"], st["batch"]
    lengths = _lengths(case)[0]
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), b["length"].to(torch.int64))
    start = torch.tensor([0] + list(np.cumsum(lengths)), device="cuda")
    pos = torch.arange(st["total"], device="cuda") - start[seq]
    slot = b["pages"][seq, pos // case["page"]].to(torch.int64) * case["page"] + pos % case["page"]
    c = codes.flatten(-2)
    for name, t in (("_codes", c[..., 0::2] | (c[..., 1::2] << 4)), ("_step", step), ("_min", minimum)):
        room = torch.zeros(b["n_pages"] * case["page"], *t.shape[1:], dtype=t.dtype, device="cuda")
        room[slot] = t
        st[which + name] = room.unflatten(0, (-1, case["page"]))


def prepare(case, seed):
    st = _inputs(case, seed)
    kind = case["kind"]
    if own:
        import cortexsdr_b200 as cs
        ctx, st["own_dtype"] = _context(), _own_dtype(case)
        if kind in ("append", "attend"):
            b = st["batch"]
            st["cache"] = cs.KVCache(b["n_pages"], case["page"], case["kv_heads"], case["head_dim"], rope_theta=THETA, ctx=ctx)
            st["own_batch"] = _own_batch(b, case["seqs"])
        if kind == "append":
            st["q_out"] = torch.empty(b["tokens"], case["q_heads"], case["head_dim"], dtype=st["dtype"], device="cuda")
            st["k_out"], st["v_out"] = (torch.empty(b["tokens"], case["kv_heads"], case["head_dim"], device="cuda") for _ in range(2))
        elif kind == "attend":
            st["out"] = torch.empty_like(st["q"])
            whole = _whole(case, b)
            torch.cuda.synchronize()
            st["cache"].append(_own_batch(whole, case["seqs"]), st["k"].data_ptr(), st["v"].data_ptr(), 1, rotate=False)
            ctx.synchronize()
        elif kind == "q4":
            st["weight"] = cs.Q4Weight.from_payload(st["payload"].cpu().numpy(), case["format"], case["rows"], case["cols"], ctx)
            token = case["layout"] == "token"
            st["y"] = torch.empty((case["batch"], case["rows"]) if token else (case["rows"], case["batch"]), device="cuda")
            st["own_layout"] = 1 if token else 0
        else:
            r, k = case["rows"], case["top"]
            st["out"] = {"logprob": torch.empty(r, device="cuda"), "entropy": torch.empty(r, device="cuda")}
            if k:
                st["out"] |= {"ids": torch.empty(r, k, dtype=torch.int32, device="cuda"), "top": torch.empty(r, k, device="cuda")}
        torch.cuda.synchronize()
    elif kind == "attend":
        _paged(st, "k", *_quantised(st["k"].to(torch.float64)))
        _paged(st, "v", *_quantised(st["v"].to(torch.float64)))
    if kind == "attend":
        del st["k"], st["v"]
    return st


def _own_append(st):
    case, q, k = st["case"], st["q"], st["k"]
    st["cache"].append(st["own_batch"], k.data_ptr(), st["v"].data_ptr(), st["own_dtype"], kv_stride=k.stride(0), q_ptr=q.data_ptr(),
                       q_stride=q.stride(0), q_heads=case["q_heads"], q_out_ptr=st["q_out"].data_ptr())
    st["cache"].read(st["own_batch"], st["k_out"].data_ptr(), st["v_out"].data_ptr())
    return {"q": st["q_out"], "k": st["k_out"], "v": st["v_out"]}


def _own_attend(st):
    st["cache"].attention(st["own_batch"], st["q"].data_ptr(), st["own_dtype"], st["case"]["q_heads"], st["out"].data_ptr())
    return st["out"]


def _own_q4(st):
    st["weight"].matmul_device(st["x"].data_ptr(), st["own_dtype"], st["own_layout"], st["case"]["batch"], st["y"].data_ptr(),
                               st["own_layout"])
    return st["y"]


def _own_logprob(st):
    import cortexsdr_b200 as cs
    case, out = st["case"], st["out"]
    top = (case["top"], out["ids"].data_ptr(), out["top"].data_ptr()) if case["top"] else ()
    cs.token_logprobs_device(st["logits"].data_ptr(), st["own_dtype"], case["rows"], case["vocab"], st["targets"].data_ptr(),
                             out["logprob"].data_ptr(), out["entropy"].data_ptr(), *top)
    return out


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "q4": _own_q4, "logprob": _own_logprob}[kind](state)
    return {"append": _plain_append, "attend": _plain_attend, "q4": _plain_q4, "logprob": _plain_logprob}[kind](state)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "q4":
        r, c, b = case["rows"], case["cols"], case["batch"]
        weight = r * c // 32 * 18 if case["format"] == "q4_0" else r * c // 256 * 144
        return dict(bytes=weight + b * c * es + b * r * 4, flops=2.0 * b * r * c)
    if case["kind"] == "logprob":
        r, n, k = case["rows"], case["vocab"], case["top"]
        return dict(bytes=r * n * es + r * 4 + r * 8 + r * k * 8, flops=5.0 * r * n)
    lengths, fresh = _lengths(case)
    qh, kvh, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    row = kvh * (d + d // GROUP * 8)      # a token's keys and values in the cache
    t = sum(fresh)
    if case["kind"] == "append":          # written to the cache and read back as 32-bit values
        return dict(bytes=t * ((2 * qh + 2 * kvh) * d * es + 2 * row + 2 * kvh * d * 4), flops=3.0 * t * (qh + kvh) * d + 6.0 * t * kvh * d)
    pairs = sum(n * length - n * (n - 1) // 2 for length, n in zip(lengths, fresh))
    read = sum(length for length, n in zip(lengths, fresh) if n)
    return dict(bytes=read * row + 2 * t * qh * d * es, flops=4.0 * d * qh * pairs)


# ---- from the definitions, in 64 bits ----

def _exact_group(x):
    """The values that rows of 64 numbers are held as."""
    lo, hi = x.min(dim=-1, keepdim=True).values, x.max(dim=-1, keepdim=True).values
    base = lo.float().half().double()
    delta = ((hi - lo) / 15).float().half().double()
    level = torch.floor((x - base) / delta)
    rest = (x - base) / delta - level
    odd = torch.remainder(level, 2) == 1
    level = level + ((rest > 0.5) | ((rest == 0.5) & odd)).double()
    level = torch.where(delta > 0, level.clamp(0, 15), torch.zeros_like(level))
    return base + torch.where(delta > 0, delta, torch.zeros_like(delta)) * level


def _exact_held(x):
    return _exact_group(x.double().reshape(-1, 64)).reshape(x.shape)


def _exact_turned(x, pos):
    d = x.shape[-1]
    z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], d // 2, 2).contiguous())
    rate = torch.exp(torch.arange(d // 2, dtype=torch.float64, device=x.device) * (-2.0 * math.log(THETA) / d))
    turn = torch.polar(torch.ones_like(rate)[None] * torch.ones_like(pos, dtype=torch.float64)[:, None], pos.double()[:, None] * rate)
    return torch.view_as_real(z * turn[:, None, :]).reshape(x.shape)


def _exact_attend(st):
    case, b = st["case"], st["batch"]
    lengths, fresh = _lengths(case)
    group, outs, row, base = case["q_heads"] // case["kv_heads"], [], 0, 0
    for length, n in zip(lengths, fresh):
        if n:
            k, v = (_exact_held(st[t][base:base + length]).repeat_interleave(group, dim=1) for t in ("k", "v"))
            q = st["q"][row:row + n].double()
            s = torch.einsum("thd,lhd->htl", q, k) * case["head_dim"] ** -0.5
            at = torch.arange(length, device="cuda")[None, :] > torch.arange(length - n, length, device="cuda")[:, None]
            s = s.masked_fill(at[None], -math.inf)
            w = torch.exp(s - torch.logsumexp(s, -1, keepdim=True))
            outs.append(torch.einsum("htl,lhd->thd", w, v))
        row, base = row + n, base + length
    return torch.cat(outs)


def exact(case, seed):
    st = _inputs(case, seed)
    if case["kind"] == "append":
        pos = st["batch"]["rows_pos"]
        return {"q": _exact_turned(st["q"], pos), "k": _exact_held(_exact_turned(st["k"], pos)), "v": _exact_held(st["v"])}
    if case["kind"] == "attend":
        return _exact_attend(st)
    if case["kind"] == "q4":
        w = _weights(st["payload"], case["rows"], case["cols"], case["format"], torch.float64)
        return st["x"].double() @ w.T if case["layout"] == "token" else w @ st["x"].double()
    parts = []
    for x, t in zip(st["logits"].split(256), st["targets"].split(256)):
        logp = torch.log_softmax(x.double(), -1)
        rows = {"logprob": logp.gather(1, t.long()[:, None])[:, 0], "entropy": -(logp.exp() * logp).sum(-1)}
        if case["top"]:
            rows["top"] = torch.topk(logp, case["top"], -1).values
        parts.append(rows)
    out = {n: torch.cat([p[n] for p in parts]) for n in parts[0]}
    return dict(out, ids=None) if case["top"] else out
