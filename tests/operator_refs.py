"""Plain 64-bit restatements of the operators that stand on their own (numpy), for the tests of the paged 4-bit cache,
the products with 4-bit weights and the log probabilities."""
import numpy as np

GROUP = 64


def rotate(x, pos, theta):
    """(T, heads, D), adjacent pairs turned by pos * theta^(-2i / D)."""
    d = x.shape[-1]
    a = np.asarray(pos, np.float64)[:, None] * theta ** (-np.arange(0, d, 2, dtype=np.float64) / d)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    x = np.asarray(x, np.float64)
    out = np.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    out[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
    return out


def held(x):
    """What a cache holds for rows of values: groups of 64, fp16 minimum and step, 4-bit codes."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        fine = np.isfinite(g).all(-1, keepdims=True)
        c = np.clip(g, -65504, 65504)
        lo, hi = c.min(-1, keepdims=True), c.max(-1, keepdims=True)
        mn = lo.astype(np.float32).astype(np.float16).astype(np.float64)
        st = ((hi - lo) / 15).astype(np.float32).astype(np.float16).astype(np.float64)
        code = np.where(st > 0, np.clip(np.rint((g - mn) / np.where(st > 0, st, 1)), 0, 15), 0)
        v = np.where(fine, mn + st * code, np.nan)
    return v.reshape(x.shape)


def attention(q, k, v, pos, scale):
    """q (T, QH, D); k, v (L, KVH, D) of one sequence; row t sees 0 .. pos[t]; `None` rows of k are not there."""
    group = q.shape[1] // k.shape[1]
    out = np.zeros(q.shape)
    for t in range(q.shape[0]):
        n = pos[t] + 1
        if n <= 0:
            continue
        kk, vv = (np.repeat(a[:n], group, axis=1) for a in (k, v))
        s = np.einsum("hd,lhd->hl", q[t].astype(np.float64), kk) * scale
        e = np.exp(s - s.max(1, keepdims=True))
        out[t] = np.einsum("hl,lhd->hd", e / e.sum(1, keepdims=True), vv)
    return out


def widened_bound(q, k, v, pos, scale):
    """What fp16 operands cost attention(): keys off by half a step each (2^-11 of themselves) move a score by at most
    d = 2^-11 |scale| sum |q k|, all weights together by a factor of e^(2 d) at most; values and weights are off by 2^-11 of
    themselves, weights under 2^-14 of the largest by 2^-25 of it (the largest is at least 1 before the division by a sum of at
    least that), where values are finite."""
    group = q.shape[1] // k.shape[1]
    out = np.zeros(q.shape)
    for t in range(q.shape[0]):
        n = pos[t] + 1
        if n <= 0:
            continue
        kk, vv = (np.repeat(a[:n], group, axis=1) for a in (k, v))
        s = np.einsum("hd,lhd->hl", q[t].astype(np.float64), kk) * scale
        d = 2.0 ** -11 * abs(scale) * np.einsum("hd,lhd->hl", np.abs(q[t]).astype(np.float64), np.abs(kk)).max(1)
        e = np.exp(s - s.max(1, keepdims=True))
        size = np.einsum("hl,lhd->hd", e / e.sum(1, keepdims=True), np.abs(vv))
        out[t] = np.expm1(2 * d + 2.0 ** -10)[:, None] * size + 2.0 ** -25 * np.abs(vv).sum(0)
    return out


def steps_bound(q, k, v, pos, scale):
    """What it costs attention() to round a weight times a step to fp16 (2^-11 of itself): an output is a sum of these times
    (code - 8), |code - 8| <= 8, and a group's fifteen steps are at most twice its largest value: 2^-11 16 / 15 of that, weighted.
    (Half as much again: a step is rounded up by 2^-11 at most, held values may lie inside the range.)"""
    group = q.shape[1] // k.shape[1]
    out = np.zeros(q.shape)
    most = np.abs(v.reshape(*v.shape[:2], -1, 64)).max(-1, keepdims=True)
    most = np.broadcast_to(most, (*most.shape[:3], 64)).reshape(v.shape)
    for t in range(q.shape[0]):
        n = pos[t] + 1
        if n <= 0:
            continue
        kk, mm = (np.repeat(a[:n], group, axis=1) for a in (k, most))
        s = np.einsum("hd,lhd->hl", q[t].astype(np.float64), kk) * scale
        e = np.exp(s - s.max(1, keepdims=True))
        out[t] = 1.5 * 2.0 ** -11 * 16 / 15 * np.einsum("hl,lhd->hd", e / e.sum(1, keepdims=True), mm)
    return out


def q4_pack(codes, steps, fmt, mins=None):
    """Blocks of a stored tensor. q4_0: codes (n, 32), steps (n,) fp16. q4_k: codes (n, 256), steps (n, 8) and mins (n, 8)
    6-bit, `steps[1]` is (n, 2) fp16 (d, dmin)."""
    codes = codes.astype(np.uint8)
    if fmt == "q4_0":
        out = np.empty((codes.shape[0], 18), np.uint8)
        out[:, :2] = steps.astype(np.float16).reshape(-1, 1).view(np.uint8)
        out[:, 2:] = codes[:, 0::2] | (codes[:, 1::2] << 4)
        return out
    sc, d = steps
    out = np.empty((codes.shape[0], 144), np.uint8)
    out[:, :4] = np.ascontiguousarray(d.astype(np.float16)).view(np.uint8)
    for j in range(4):
        out[:, 4 + j] = (sc[:, j] & 63) | ((sc[:, j + 4] >> 4) << 6)
        out[:, 8 + j] = (mins[:, j] & 63) | ((mins[:, j + 4] >> 4) << 6)
        out[:, 12 + j] = (sc[:, j + 4] & 15) | ((mins[:, j + 4] & 15) << 4)
    for g in range(4):
        out[:, 16 + 32 * g:48 + 32 * g] = codes[:, 64 * g:64 * g + 32] | (codes[:, 64 * g + 32:64 * g + 64] << 4)
    return out


def q4_weight(rng, rows, cols, fmt):
    """(payload bytes, the matrix in 64 bits)."""
    if fmt == "q4_0":
        n = rows * cols // 32
        codes, d = rng.integers(0, 16, (n, 32)), (0.02 * np.exp(rng.normal(0, 0.5, n))).astype(np.float16)
        d[rng.random(n) < 0.05] = 0
        w = (codes - 8.0) * d.astype(np.float64)[:, None]
        return q4_pack(codes, d, fmt), w.reshape(rows, cols)
    n = rows * cols // 256
    codes, sc, mn = rng.integers(0, 16, (n, 256)), rng.integers(0, 64, (n, 8)).astype(np.uint8), rng.integers(0, 64, (n, 8)).astype(np.uint8)
    d = (0.001 * np.exp(rng.normal(0, 0.5, (n, 2)))).astype(np.float16)
    df = d.astype(np.float64)
    w = codes.reshape(n, 8, 32) * (df[:, :1] * sc)[..., None] - (df[:, 1:] * mn)[..., None]
    return q4_pack(codes, (sc, d), fmt, mn), w.reshape(rows, cols)


def logprobs(x, targets, top):
    """(log probability, entropy, ids, their log probabilities) of rows of logits in 64 bits."""
    x = np.asarray(x, np.float64)
    m = x.max(1, keepdims=True)
    e = np.exp(x - m)
    s = e.sum(1, keepdims=True)
    lp = x - m - np.log(s)
    p = e / s
    ent = -(p * np.where(p > 0, lp, 0)).sum(1)
    ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return lp[np.arange(len(x)), targets], ent, ids, np.take_along_axis(lp, ids, 1)
