"""Plain numpy restatements, in 64 bits, of the operators that keep a paged
cache small: 4-bit quantisation, the decode that gives attention weights, and
the eviction plan. Used by the tests alone."""

import numpy as np

MAGNITUDES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def quantise(x):
    """fp16 values [..., D] -> codes [..., D/2] and scale bytes [..., 4] (uint8)."""
    x = np.asarray(x, dtype=np.float64)
    d = x.shape[-1]
    blocks = x.reshape(*x.shape[:-1], d // 32, 32)
    top = np.abs(blocks).max(-1)
    fine = np.isfinite(blocks).all(-1)
    _, e = np.frexp(np.where(fine & (top > 0), top, 2.0 ** -30))
    e = np.maximum(e - 3, -24)
    with np.errstate(invalid="ignore"):
        y = np.where(fine[..., None], blocks, 0.0) / np.ldexp(1.0, e)[..., None]
    # nearest magnitude; a tie (on a midpoint) goes to the even code
    a, mid = np.abs(y), (MAGNITUDES[:-1] + MAGNITUDES[1:]) / 2
    code = sum(((a > m) | ((a == m) & (i % 2 == 1))).astype(np.uint8) for i, m in enumerate(mid))
    code = code | (np.signbit(y).astype(np.uint8) << 3)
    code = np.where(fine[..., None], code, 0).reshape(x.shape).astype(np.uint8)
    scales = np.zeros((*x.shape[:-1], 4), dtype=np.uint8)
    scales[..., : d // 32] = np.where(fine, e + 127, 255)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def dequantise(codes, scales):
    """Codes [..., D/2] and scale rows [..., 4] -> float64 [..., D]."""
    d = 2 * codes.shape[-1]
    n = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], d)
    v = np.where(n & 8, -1.0, 1.0) * MAGNITUDES[n & 7]
    s = scales[..., : d // 32].astype(np.int64)
    f = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return (v.reshape(*codes.shape[:-1], d // 32, 32) * f[..., None]).reshape(v.shape)


def gather(cache, block_table_row, n):
    """The first n rows of a sequence: cache [P, ps, Hkv, X] -> [n, Hkv, X]."""
    ps = cache.shape[1]
    t = np.arange(n)
    return cache[block_table_row[t // ps], t % ps]


def decode(q, k, v, block_table, seq_lens, scale=None):
    """out [B, Hq, D] and, per sequence, the attention probabilities summed over
    the query heads of each KV head [n, Hkv], all in float64."""
    b, hq, d = q.shape
    hkv = k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out = np.zeros((b, hq, d))
    probs = []
    for i in range(b):
        n = int(seq_lens[i])
        if n == 0:
            probs.append(np.zeros((0, hkv)))
            continue
        kk, vv = gather(k, block_table[i], n).astype(np.float64), gather(v, block_table[i], n).astype(np.float64)
        s = np.einsum("hgd,thd->hgt", q[i].astype(np.float64).reshape(hkv, hq // hkv, d), kk) * scale
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[i] = np.einsum("hgt,thd->hgd", p, vv).reshape(hq, d)
        probs.append(p.sum(1).T)
    return out, probs


def accumulate(weights, probs, block_table, seq_lens, num_new):
    """weights [P, Hkv, ps] after the step (float64)."""
    w = weights.astype(np.float64).copy()
    ps = w.shape[2]
    for i, p in enumerate(probs):
        for t in range(int(seq_lens[i])):
            page, row = block_table[i, t // ps], t % ps
            old = 0.0 if t >= int(seq_lens[i]) - num_new else w[page, :, row]
            w[page, :, row] = old + p[t]
    return w


def evict_plan(weights, block_table, seq_lens, budget, recent=0, positions=None, total_lens=None):
    """(src, dst) lists per (sequence, head), and new lengths."""
    b, hkv, ps = len(seq_lens), weights.shape[1], weights.shape[2]
    src, dst = {}, {}
    for i in range(b):
        n = int(seq_lens[i])
        t = np.arange(n)
        for h in range(hkv):
            if n <= budget:
                src[i, h], dst[i, h] = [], []
                continue
            page, row = block_table[i, t // ps], t % ps
            w = weights[page, h, row].astype(np.float64) + 0.0
            cls = np.where(np.isnan(w), 1, 2)
            if recent > 0:
                cls = np.where(positions[page, h, row] >= int(total_lens[i]) - recent, 0, cls)
            w = np.where(cls == 2, w, 0.0)
            order = np.lexsort((t, -w, cls))
            keep = np.zeros(n, dtype=bool)
            keep[order[:budget]] = True
            dst[i, h] = [s for s in range(budget) if not keep[s]]
            src[i, h] = [s for s in range(budget, n) if keep[s]]
    return src, dst, np.minimum(np.asarray(seq_lens), budget)


def apply_moves(cache, block_table, src, dst, head_axis=2):
    """A copy of the cache ([P, ps, Hkv, X], or [P, Hkv, ps] with head_axis 1) after the moves."""
    out = cache.copy()
    ps = cache.shape[1 if head_axis == 2 else 2]
    for (i, h), ss in src.items():
        for s, d in zip(ss, dst[i, h]):
            a, z = (block_table[i, s // ps], s % ps), (block_table[i, d // ps], d % ps)
            if head_axis == 2:
                out[z[0], z[1], h] = cache[a[0], a[1], h]
            else:
                out[z[0], h, z[1]] = cache[a[0], h, a[1]]
    return out
