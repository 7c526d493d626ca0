"""What is measured of the operators that keep a paged KV cache small: decode
attention that accumulates each cached token's attention weight, the plan and
the moves of an eviction by that weight, and a cache in microscaled 4-bit
floating point (blocks of 32 values along the head dim, e2m1 codes two to a
byte with the lower dim in the low nibble, one power-of-two scale byte a
block) with its append, its read-back and the decode over it.

``own = False`` computes the plain forms with elementary torch operations;
``own = True`` calls the framework.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"


def api():
    """The framework's package, imported only where its operators are called."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paged-attention-decode_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import pad_b200

    return pad_b200


# ----------------------------------------------------------------------------- cases
def listed():
    heads = dict(hkv=2, g=6, d=128, ps=16)  # the 12-query-head, 2-KV-head shape of the batch sweep
    wide = dict(hkv=8, g=4, d=128, ps=16)   # the 32-query-head, 8-KV-head shape of the ragged batch
    return [
        # one request decoding while its cache is tracked for eviction: latency counts
        dict(name="weights_b1", op="weights", b=1, lo=4096, hi=4096, lens_seed=0, new=1, **heads),
        # the batch sweep's largest batch
        dict(name="weights_b64", op="weights", b=64, lo=4096, hi=4096, lens_seed=0, new=1, **heads),
        # a ragged serving batch, log-uniform lengths
        dict(name="weights_ragged256", op="weights", b=256, lo=128, hi=8192, lens_seed=1, new=1, **wide),
        # one long context over the 4-bit cache
        dict(name="fp4_b1_131072", op="fp4", b=1, lo=131072, hi=131072, lens_seed=0, track=False, new=1, hkv=2, g=6,
             d=128, ps=32),
        dict(name="fp4_b64", op="fp4", b=64, lo=4096, hi=4096, lens_seed=0, track=False, new=1, **heads),
        # 64 query heads over 8 KV heads, lengths 1024 to 16384, tracked for eviction as well
        dict(name="fp4_ragged64_tracked", op="fp4", b=64, lo=1024, hi=16384, lens_seed=2, track=True, new=1, hkv=8,
             g=8, d=128, ps=16),
        # one decoding step's new token of each sequence, written and read back (head dim 64)
        dict(name="append_step64", op="append", b=64, lo=1, hi=1, lens_seed=0, start=4095, hkv=2, g=6, d=64, ps=16),
        # prompts of eight requests written and read back, as a later chunk of the prompt needs them
        dict(name="append_prompt8", op="append", b=8, lo=1000, hi=8191, lens_seed=3, start=0, **wide),
        # steady state: a few tokens over the budget in every sequence
        dict(name="plan_step64", op="plan", b=64, lo=2049, hi=2112, lens_seed=4, budget=2048, recent=128, hkv=2, ps=16),
        # long prompts cut to an eighth once
        dict(name="plan_long4", op="plan", b=4, lo=100001, hi=131072, lens_seed=5, budget=16384, recent=256, hkv=8,
             ps=16),
        # the moves after halving every sequence's cache
        dict(name="move_fp16_b64", op="move", b=64, lo=4096, hi=4096, lens_seed=0, budget=2048, fp4=False, hkv=2,
             d=128, ps=16),
        # the same of a 4-bit cache cut to a quarter, ragged
        dict(name="move_fp4_b16", op="move", b=16, lo=8192, hi=16384, lens_seed=6, budget=4096, fp4=True, hkv=8,
             d=128, ps=16),
    ]


def draw(rng):
    lg = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["weights", "weights", "fp4", "fp4", "append", "plan", "move"])
    hkv, g = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 6, 8, 16])
    d = rng.choice([32, 64, 128, 128])
    ps = rng.choice([8, 16, 24, 32, 64])
    c = dict(op=op, lens_seed=rng.randrange(1 << 20), hkv=hkv, ps=ps)
    if op in ("weights", "fp4"):
        hi = lg(64, 131072)
        b = max(1, min(lg(1, 256), (7 << 19) // (hi * hkv)))  # at most the work of the largest listed case
        c.update(b=b, lo=max(1, int(hi * rng.uniform(0.05, 1.0))), hi=hi, g=g, d=d, new=rng.choice([1, 1, 2, 7]))
        if op == "fp4":
            c["track"] = rng.random() < 0.5
    elif op == "append":
        hi = lg(1, 8191)
        c.update(b=max(1, min(lg(1, 128), 32768 * 8 // (hi * hkv))), lo=max(1, int(hi * rng.uniform(0.1, 1.0))), hi=hi,
                 start=rng.randrange(0, 100), g=g, d=d)
    else:
        hi = lg(64, 65536)
        b = max(1, min(lg(1, 64), (1 << 21) // (hi * hkv)))
        budget = max(1, int(hi * rng.uniform(0.1, 0.9)))
        c.update(b=b, lo=max(1, int(hi * rng.uniform(0.3, 1.0))), hi=hi, budget=budget)
        if op == "plan":
            c["recent"] = rng.choice([0, 1, 64])
            c["recent"] = min(c["recent"], budget)
        else:
            c.update(fp4=rng.random() < 0.5, d=d)
    return c


def lengths(case):
    """seq_lens of a case, by the case alone (log-uniform, both ends possible)."""
    rng = np.random.default_rng(case["lens_seed"])
    u = rng.uniform(math.log(case["lo"]), math.log(case["hi"]), size=case["b"])
    return np.clip(np.exp(u).round(), case["lo"], case["hi"]).astype(np.int64)


def moves_of(case):
    """Rows that move for one (sequence, KV head): survivors spread evenly over the sequence."""
    n = lengths(case)
    m = case["budget"] * (n - case["budget"]) // np.maximum(n, 1)
    return np.where(n > case["budget"], np.minimum(m, n - case["budget"]), 0)


def work(case):
    n = lengths(case)
    b, hkv, op = case["b"], case["hkv"], case["op"]
    pages = int(((n + case["ps"] - 1) // case["ps"]).sum())
    t = int(n.sum())
    if op in ("weights", "fp4"):
        d, hq = case["d"], hkv * case["g"]
        row = 2 * (2 * d if op == "weights" else d // 2 + d // 32)
        by = t * hkv * row + 4 * b * hq * d + 4 * pages
        if op == "weights" or case["track"]:
            by += 8 * t * hkv
        return {"bytes": by, "flops": 4 * t * hq * d}
    if op == "append":  # values in, codes and scales out; codes and scales in, values out
        d = case["d"]
        return {"bytes": 2 * t * hkv * 2 * (2 * d + d // 2 + d // 32), "flops": 4 * t * hkv * d}
    width = max(0, min(case["budget"], table_width(case) * case["ps"] - case["budget"]))
    if op == "plan":
        return {"bytes": 8 * t * hkv + 4 * pages + 8 * b * hkv * width, "flops": t * hkv}
    d = case["d"]
    row = 2 * (d // 2 + d // 32 if case["fp4"] else 2 * d) + 8
    return {"bytes": int(moves_of(case).sum()) * hkv * 2 * row, "flops": 1}


# ----------------------------------------------------------------------------- inputs
def table_width(case):
    """Columns of the block table: what the longest sequence needs, and two more."""
    top = case["hi"] + case.get("start", 0)
    return -(-top // case["ps"]) + 2


def paging(case, seed):
    """A shuffled pool with spare pages, and every sequence's row of page ids."""
    n = lengths(case) + case.get("start", 0)
    need = -(-n // case["ps"])
    rng = np.random.default_rng(seed)
    total = int(need.sum()) + 5
    perm = rng.permutation(total).astype(np.int32)
    width = table_width(case)
    bt = np.zeros((case["b"], width), dtype=np.int32)
    cols = np.arange(width)[None, :] < need[:, None]
    bt[cols] = perm[: int(need.sum())]
    return torch.from_numpy(bt).to(DEV), torch.from_numpy(n.astype(np.int32)).to(DEV), total


def power(e):
    """2^e in 32 bits, exactly, for exponents of normal numbers."""
    return ((e.int() + 127) << 23).view(torch.float32)


def quantise(x):
    """Values [..., D] -> codes [..., D/2] and scale bytes [..., D/32], uint8, of the blocks of 32 along D."""
    y = x.float().unflatten(-1, (-1, 32))
    top = y.abs().amax(-1, keepdim=True)
    e = torch.frexp(top).exponent.clamp(min=-21) - 3
    a = y * power(-e)
    m = a.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5))
    code = code + 8 * torch.signbit(a).to(torch.uint8)
    fine = torch.isfinite(top)
    code = torch.where(fine, code, torch.zeros_like(code)).flatten(-2)
    scales = torch.where(fine, e + 127, torch.full_like(e, 255)).squeeze(-1).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def dequantise(codes, scales, d):
    """Codes [..., D/2] and scale bytes [..., 4] (D/32 of them used) -> values [..., D]."""
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    m = (both & 7).float()
    v = m * 0.5 + (m - 4).clamp(min=0) * 0.5 + (m - 6).clamp(min=0)  # 0 0.5 1 1.5 2 3 4 6
    v = torch.where(both > 7, -v, v)
    s = scales[..., : d // 32].int()
    f = torch.where(s == 255, torch.full_like(s, float("nan"), dtype=torch.float32), power(s - 127))
    return (v.unflatten(-1, (-1, 32)) * f.unsqueeze(-1)).flatten(-2)


def fp4_cache(gen, pages, ps, hkv, d):
    """A cache of quantised N(0, 1) values; scale rows are 4 bytes wide at every head dim."""
    codes = torch.empty((pages, ps, hkv, d // 2), dtype=torch.uint8, device=DEV)
    scales = torch.zeros((pages, ps, hkv, 4), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (ps * hkv * d))
    for p in range(0, pages, step):
        q = min(pages, p + step)
        x = torch.randn((q - p, ps, hkv, d), device=DEV, generator=gen).half()
        c, s = quantise(x)
        codes[p:q] = c
        scales[p:q, :, :, : d // 32] = s
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    bt, n, pages = paging(case, seed)
    b, hkv, ps, op = case["b"], case["hkv"], case["ps"], case["op"]
    st = dict(case=case, bt=bt, n=n, longest=int(case["hi"] + case.get("start", 0)))

    def tracked():
        # weights gathered over earlier steps (a few heavy tokens, a long tail), and each slot's token position
        st["weights"] = torch.rand((pages, hkv, ps), device=DEV, generator=gen) ** 8 * 10
        st["positions"] = torch.randint(0, 1 << 20, (pages, hkv, ps), device=DEV, generator=gen, dtype=torch.int32)
        st["total"] = n + 1000

    if op in ("weights", "fp4"):
        d = case["d"]
        st["q"] = torch.randn((b, hkv * case["g"], d), device=DEV, generator=gen).half()
        if op == "weights":
            st["k"] = torch.empty((pages, ps, hkv, d), dtype=torch.float16, device=DEV).normal_(generator=gen)
            st["v"] = torch.empty((pages, ps, hkv, d), dtype=torch.float16, device=DEV).normal_(generator=gen)
        else:
            st["k"], st["ks"] = fp4_cache(gen, pages, ps, hkv, d)
            st["v"], st["vs"] = fp4_cache(gen, pages, ps, hkv, d)
        if op == "weights" or case["track"]:
            tracked()
    elif op == "append":
        d = case["d"]
        lens = lengths(case)
        t = int(lens.sum())
        # keys and values of the new tokens, a different magnitude in every block of 32
        mag = torch.exp2(torch.randint(-6, 4, (2, t, hkv, d // 32, 1), device=DEV, generator=gen).float())
        x = (torch.randn((2, t, hkv, d // 32, 32), device=DEV, generator=gen) * mag).half().flatten(-2)
        st["k_new"], st["v_new"] = x[0], x[1]
        st["k"] = torch.zeros((pages, ps, hkv, d // 2), dtype=torch.uint8, device=DEV)
        st["v"] = torch.zeros_like(st["k"])
        st["ks"] = torch.zeros((pages, ps, hkv, 4), dtype=torch.uint8, device=DEV)
        st["vs"] = torch.zeros_like(st["ks"])
        ids = np.repeat(np.arange(b), lens)
        pos = np.arange(t) - np.repeat(np.cumsum(lens) - lens, lens) + case["start"]
        st["ids"] = torch.from_numpy(ids.astype(np.int32)).to(DEV)
        st["pos"] = torch.from_numpy(pos.astype(np.int32)).to(DEV)
    elif op == "plan":
        tracked()
        # weights with ties (a coarse grid) beside the long tail
        w = st["weights"]
        st["weights"] = torch.where(w < 0.05, (w * 1000).round() / 1000, w)
        # positions in the order of the slots, as before a first eviction
        st["total"] = n.clone()
        cols = torch.arange(bt.shape[1] * ps, device=DEV)
        page, row = bt[:, cols // ps].long(), cols % ps
        live = cols[None, :] < n[:, None]
        flat = (page[:, None, :] * hkv + torch.arange(hkv, device=DEV)[None, :, None]) * ps + row
        st["positions"].view(-1)[flat[live[:, None, :].expand(-1, hkv, -1)]] = (
            cols.to(torch.int32)[None, None, :].expand(b, hkv, -1)[live[:, None, :].expand(-1, hkv, -1)])
    else:
        d = case["d"]
        tracked()
        if case["fp4"]:
            st["k"], st["ks"] = fp4_cache(gen, pages, ps, hkv, d)
            st["v"], st["vs"] = fp4_cache(gen, pages, ps, hkv, d)
        else:
            st["k"] = torch.empty((pages, ps, hkv, d), dtype=torch.float16, device=DEV).normal_(generator=gen)
            st["v"] = torch.empty((pages, ps, hkv, d), dtype=torch.float16, device=DEV).normal_(generator=gen)
        # ascending holes below the budget, ascending survivors above it
        budget, m = case["budget"], torch.from_numpy(moves_of(case)).to(DEV)
        width = max(0, min(budget, bt.shape[1] * ps - budget))
        take = torch.arange(width, device=DEV)[None, None, :] < m[:, None, None]

        def choose(first, upto):
            slots = torch.arange(bt.shape[1] * ps, device=DEV)
            ok = (slots >= first) & (slots[None, :] < upto[:, None])
            r = torch.rand((b, hkv, slots.numel()), device=DEV, generator=gen)
            r = torch.where(ok[:, None, :], r, torch.full_like(r, 2.0))
            got = r.argsort(-1)[..., :width]
            got = torch.where(take, got, torch.full_like(got, 1 << 30)).sort(-1).values
            return torch.where(take, got, torch.full_like(got, -1)).to(torch.int32)

        st["src"] = choose(budget, n)
        st["dst"] = choose(0, torch.full_like(n, budget))
        st["counts"] = m[:, None].expand(b, hkv).to(torch.int32).contiguous()
    return st


# ----------------------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        pad = api()
        if op == "weights":
            out = pad.paged_attention_decode_weights(st["q"], st["k"], st["v"], st["bt"], st["n"], st["weights"],
                                                     num_new=case["new"], slot_positions=st["positions"],
                                                     total_lens=st["total"])
            return {"out": out, "weights": st["weights"], "positions": st["positions"]}
        if op == "fp4":
            if not case["track"]:
                return {"out": pad.paged_attention_decode_fp4(st["q"], st["k"], st["ks"], st["v"], st["vs"], st["bt"],
                                                              st["n"])}
            out = pad.paged_attention_decode_fp4(st["q"], st["k"], st["ks"], st["v"], st["vs"], st["bt"], st["n"],
                                                 weights=st["weights"], num_new=case["new"],
                                                 slot_positions=st["positions"], total_lens=st["total"])
            return {"out": out, "weights": st["weights"], "positions": st["positions"]}
        if op == "append":
            pad.paged_kv_append_fp4(st["k_new"], st["v_new"], st["k"], st["ks"], st["v"], st["vs"], st["bt"], st["pos"],
                                    st["ids"])
            k, v = pad.paged_kv_read_fp4(st["k"], st["ks"], st["v"], st["vs"], st["bt"], st["pos"], st["ids"])
            return {"k": k, "v": v}
        if op == "plan":
            src, dst, counts, lens = pad.paged_kv_evict_plan(st["weights"], st["bt"], st["n"], case["budget"],
                                                             case["recent"], slot_positions=st["positions"],
                                                             total_lens=st["total"])
            return {"src": src, "dst": dst, "counts": counts, "lens": lens}
        pad.paged_kv_move(caches_of(st), st["bt"], st["src"], st["dst"], st["counts"], weights=st["weights"],
                          slot_positions=st["positions"])
        return moved_values(st)
    if op in ("weights", "fp4"):
        return plain_decode(st)
    if op == "append":
        return plain_append(st)
    return plain_plan(st) if op == "plan" else plain_move(st)


def caches_of(st):
    return (st["k"], st["ks"], st["v"], st["vs"]) if st["case"]["fp4"] else (st["k"], st["v"])


def moved_values(st):
    """The caches after the moves. Rows of a 4-bit cache go as the words they are moved as (nothing is computed of them)."""
    got = {"weights": st["weights"], "positions": st["positions"]}
    if st["case"]["fp4"]:
        for name in ("k", "ks", "v", "vs"):
            got[name] = st[name].view(torch.int32)
    else:
        got.update(k=st["k"], v=st["v"])
    return got


def addresses(st, slots):
    """Page and row of slots [B, ...] of every sequence."""
    ps = st["case"]["ps"]
    b = torch.arange(slots.shape[0], device=slots.device).view(-1, *[1] * (slots.dim() - 1))
    return st["bt"][b, slots // ps].long(), slots % ps


def plain_decode(st):
    case = st["case"]
    b, hkv, g, d = case["b"], case["hkv"], case["g"], case["d"]
    slots = torch.arange(st["longest"], device=DEV)
    page, row = addresses(st, slots[None, :].expand(b, -1))
    live = slots[None, :] < st["n"][:, None]

    def rows(cache, scales):
        x = cache[page, row]
        x = x.float() if scales is None else dequantise(x, scales[page, row], d)
        return torch.where(live[:, :, None, None], x, torch.zeros_like(x)).transpose(1, 2)  # [B, Hkv, T, D]

    q = st["q"].float().view(b, hkv, g, d)
    s = (q @ rows(st["k"], st.get("ks")).transpose(2, 3)) / math.sqrt(d)
    s = torch.where(live[:, None, None, :], s, torch.full_like(s, -math.inf))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = (p @ rows(st["v"], st.get("vs"))).reshape(b, hkv * g, d).half()
    if "weights" not in st:
        return {"out": out}
    h = torch.arange(hkv, device=DEV)[None, :, None]
    flat = ((page[:, None, :] * hkv + h) * case["ps"] + row[:, None, :]).reshape(-1)
    fresh = (slots[None, :] >= st["n"][:, None] - case["new"])[:, None, :].expand(b, hkv, -1)
    on = live[:, None, :].expand(b, hkv, -1)
    w = st["weights"].view(-1)
    was = w[flat].view(b, hkv, -1)
    add = p.sum(2) - torch.where(fresh, was, torch.zeros_like(was))
    w.index_add_(0, flat, torch.where(on, add, torch.zeros_like(add)).reshape(-1))
    at = st["positions"].view(-1)
    said = (st["total"] - st["n"])[:, None, None] + slots.to(torch.int32)
    step = torch.where(on & fresh, said - at[flat].view(b, hkv, -1), torch.zeros_like(said))
    at.index_add_(0, flat, step.reshape(-1).to(torch.int32))
    return {"out": out, "weights": st["weights"], "positions": st["positions"]}


def plain_append(st):
    d, ps = st["case"]["d"], st["case"]["ps"]
    page, row = st["bt"][st["ids"].long(), st["pos"].long() // ps].long(), st["pos"].long() % ps
    got = {}
    for name in ("k", "v"):
        codes, scales = quantise(st[name + "_new"])
        st[name][page, row] = codes
        st[name + "s"][page, row] = torch.nn.functional.pad(scales, (0, 4 - d // 32))
        got[name] = dequantise(st[name][page, row], st[name + "s"][page, row], d).half()
    return got


def plain_plan(st):
    case = st["case"]
    b, hkv, budget = case["b"], case["hkv"], case["budget"]
    slots = torch.arange(st["longest"], device=DEV)
    page, row = addresses(st, slots[None, :].expand(b, -1))
    h = torch.arange(hkv, device=DEV)[None, :, None]
    w = st["weights"][page[:, None, :], h, row[:, None, :]].double()
    at = st["positions"][page[:, None, :], h, row[:, None, :]]
    n = st["n"].long()[:, None, None]
    live = slots < n
    key = torch.where(at >= st["total"][:, None, None] - case["recent"], torch.full_like(w, 1e300), w)
    key = torch.where(live, key, torch.full_like(w, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.zeros_like(order).scatter_(-1, order, slots.expand(b, hkv, -1).contiguous())
    keep = (rank < budget) & live
    hole = ~keep & live & (slots < budget) & (n > budget)
    mover = keep & (slots >= budget)
    width = max(0, min(budget, st["bt"].shape[1] * case["ps"] - budget))

    def as_list(on):
        to = torch.where(on, on.cumsum(-1) - 1, torch.full_like(order, width))
        got = torch.full((b, hkv, width + 1), -1, dtype=torch.int32, device=DEV)
        got.scatter_(-1, to, slots.to(torch.int32).expand(b, hkv, -1).contiguous())
        return got[..., :width].contiguous()

    return {"src": as_list(mover), "dst": as_list(hole), "counts": mover.sum(-1).to(torch.int32),
            "lens": st["n"].clamp(max=budget)}


def plain_move(st):
    valid = torch.arange(st["src"].shape[2], device=DEV) < st["counts"][:, :, None]
    # unused entries copy a row onto itself: the first source, which nothing overwrites, or slot 0 where nothing moves
    idle = torch.where(st["counts"][:, :, None] > 0, st["src"][:, :, :1], torch.zeros_like(st["src"][:, :, :1]))
    ps_, rs = addresses(st, torch.where(valid, st["src"], idle).long())
    pd, rd = addresses(st, torch.where(valid, st["dst"], idle).long())
    h = torch.arange(st["case"]["hkv"], device=DEV)[None, :, None].expand_as(ps_)
    for x in caches_of(st):
        x[pd, rd, h] = x[ps_, rs, h]
    for x in (st["weights"], st["positions"]):
        x[pd, h, rd] = x[ps_, h, rs]
    return moved_values(st)


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    op = case["op"]
    if op in ("plan", "move"):
        return None  # whole numbers and copies
    st = prepare(case, seed)
    if op == "append":
        return {"k": nearest(st["k_new"]), "v": nearest(st["v_new"])}
    b, hkv, g, d, ps = case["b"], case["hkv"], case["g"], case["d"], case["ps"]
    out = torch.zeros((b, hkv * g, d), dtype=torch.float64, device=DEV)
    w = st["weights"].double() if "weights" in st else None
    bt, lens = st["bt"].long(), lengths(case)
    for i in range(b):
        n = int(lens[i])
        pages = bt[i, : -(-n // ps)]

        def of(cache, scales):
            x = cache[pages].flatten(0, 1)[:n]
            if scales is None:
                return x.double()
            return values64(x, scales[pages].flatten(0, 1)[:n, :, : d // 32])

        k, v = of(st["k"], st.get("ks")), of(st["v"], st.get("vs"))
        q = st["q"][i].double().view(hkv, g, d)
        s = torch.einsum("hgd,thd->hgt", q, k) * d ** -0.5
        p = torch.softmax(s, -1)
        out[i] = torch.einsum("hgt,thd->hgd", p, v).reshape(hkv * g, d)
        if w is not None:
            t = torch.arange(n, device=DEV)
            page, row = pages[t // ps], t % ps
            old = w[page, :, row]
            old[max(0, n - case["new"]):] = 0
            w[page, :, row] = old + p.sum(1).t()
    return {"out": out} if w is None else {"out": out, "weights": w, "positions": None}


def values64(codes, scales):
    """What 4-bit codes stand for, from the format: sign, two exponent bits, one mantissa bit, times 2^(byte - 127)."""
    n = torch.stack((codes % 16, codes // 16), dim=-1).flatten(-2).double()
    sign = 1 - 2 * (n >= 8).double()
    n = n % 8
    e, m = torch.floor(n / 2), n % 2
    mag = torch.where(e == 0, m * 0.5, (1 + 0.5 * m) * power64(e - 1))
    return sign * mag * power64(scales.long() - 127).repeat_interleave(32, dim=-1)


def power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def nearest(x):
    """Every value's nearest code of its block's scale, ties to the even code, by distances."""
    blocks = x.double().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -27.0)
    for k in range(-24, 16):  # floor(log2(top)) - 2, by comparisons
        e += (top >= 2.0 ** k).double()
    e = e.clamp(min=-24)
    a = blocks * power64(-e)
    best, far = torch.zeros_like(a), a.abs().clone()
    for code, mag in ((2, 1.0), (4, 2.0), (6, 4.0), (1, 0.5), (3, 1.5), (5, 3.0), (7, 6.0)):  # even codes first: they keep ties
        off = (a.abs() - mag).abs()
        near = off < far
        best, far = torch.where(near, torch.full_like(a, mag), best), torch.where(near, off, far)
    return (torch.copysign(best, a) * power64(e)).flatten(-2)
