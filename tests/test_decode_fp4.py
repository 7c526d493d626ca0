"""Decode over the 4-bit cache, against float64 on what the codes stand for.

Tolerances: out has the parity bound of the other decode tests (gpu_utils);
weights the bound derived in test_decode_weights.py, with q.k summed block by
block (D / 32 more roundings, inside its D / 8 + 6)."""

import functools

import numpy as np
import pytest
import torch

import cache_oracle as co
import pad_b200
from gpu_utils import assert_parity
from pad_b200 import _lib
from pad_b200.cases import explicit_case
from test_decode_weights import check_weights, rel_bound, smax_of
from test_decode_weights import NEWS, by_sequence

gpu = pytest.mark.gpu


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _cuda(x, dt=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dt is None else t.to(dt)


def fp4_case(seqs, hkv, g, d, ps, seed):
    return _fp4_case(tuple(seqs), hkv, g, d, ps, seed)


@functools.lru_cache(maxsize=2)  # the same case over several num_splits
def _fp4_case(seqs, hkv, g, d, ps, seed):
    """q, the four cache arrays, what K and V stand for, block table, seq_lens (numpy)."""
    c = explicit_case(seqs, num_kv_heads=hkv, gqa_ratio=g, head_dim=d, page_size=ps, seed=seed)
    k, v = c.k_cache, c.v_cache
    rng = np.random.default_rng(seed + 1)  # a scale of its own for every block
    k = k * np.exp2(rng.integers(-5, 2, (*k.shape[:3], d // 32))).repeat(32, -1)
    v = v * np.exp2(rng.integers(-6, 1, (*v.shape[:3], d // 32))).repeat(32, -1)
    kc, ks = co.quantise(k.astype(np.float16))
    vc, vs = co.quantise(v.astype(np.float16))
    return c.q, (kc, ks, vc, vs), co.dequantise(kc, ks), co.dequantise(vc, vs), c.block_table, c.seq_lens


CASES = [
    # seq_lens, KV heads, G, D, page
    ([1], 1, 1, 128, 16),
    ([15, 16, 17, 31, 32, 33], 2, 6, 128, 16),
    ([4096], 2, 6, 128, 16),
    ([0, 1, 17, 300, 4000, 65, 0], 2, 6, 128, 16),
    ([5, 70, 333], 4, 4, 64, 4),
    ([129, 1000, 31], 8, 8, 128, 16),
    ([700, 64], 3, 5, 32, 24),
    ([900, 20], 4, 16, 128, 32),
    ([100, 257], 1, 12, 32, 1),
    ([640, 33], 5, 9, 64, 7),
    ([2000] * 8, 8, 4, 128, 16),
    ([20000], 8, 1, 64, 64),
    ([30, 1], 16, 3, 64, 16),
    ([1000] * 200, 1, 2, 64, 16),
]


@gpu
@pytest.mark.parametrize("num_splits", [None, 1, 3, 64])
@pytest.mark.parametrize("seqs,hkv,g,d,ps", CASES)
def test_decode_matches_float64(seqs, hkv, g, d, ps, num_splits):
    _need_cuda()
    pad_b200.read_error_flags()
    q, caches, k, v, bt, sl = fp4_case(seqs, hkv, g, d, ps, seed=d + g)
    ref, _ = co.decode(q, k, v, bt, sl)
    out = pad_b200.paged_attention_decode_fp4(_cuda(q, torch.float16), *map(_cuda, caches), _cuda(bt), _cuda(sl),
                                              num_splits)
    assert_parity(out.float().cpu().numpy(), ref)
    assert pad_b200.read_error_flags() == 0


@gpu
@pytest.mark.parametrize("num_splits", [None, 3])
@pytest.mark.parametrize("seqs,hkv,g,d,ps", [c for c in CASES if len(c[0]) < 100])
def test_weights_and_positions_match_float64(seqs, hkv, g, d, ps, num_splits):
    _need_cuda()
    q, caches, k, v, bt, sl = fp4_case(seqs, hkv, g, d, ps, seed=d + g + 1)
    ref, probs = co.decode(q, k, v, bt, sl)
    rng = np.random.default_rng(2)
    w0 = rng.random((k.shape[0], hkv, ps)).astype(np.float32)
    at0 = rng.integers(0, 99, w0.shape).astype(np.int32)
    total = np.asarray(seqs, np.int64) + 11
    qg, cg, btg, slg = _cuda(q, torch.float16), [_cuda(c) for c in caches], _cuda(bt), _cuda(sl)
    for num_new in (1, 4, 10 ** 6):
        w, at = _cuda(w0), _cuda(at0)
        out = pad_b200.paged_attention_decode_fp4(qg, *cg, btg, slg, num_splits, weights=w, num_new=num_new,
                                                  slot_positions=at, total_lens=_cuda(total))
        assert_parity(out.float().cpu().numpy(), ref)
        check_weights(w.cpu().numpy(), co.accumulate(w0, probs, bt, sl, num_new),
                      rel_bound(d, max(seqs), smax_of(q, k, d)))
        want = at0.copy()
        for i, n in enumerate(seqs):
            for t in range(max(0, n - num_new), n):
                want[bt[i, t // ps], :, t % ps] = total[i] - n + t
        np.testing.assert_array_equal(at.cpu().numpy(), want)
    plain = pad_b200.paged_attention_decode_fp4(qg, *cg, btg, slg, num_splits)
    assert torch.equal(out, plain)  # the weights change nothing of the output
    assert torch.equal(plain, pad_b200.paged_attention_decode_fp4(qg, *cg, btg, slg, num_splits))  # repeatable


@gpu
@pytest.mark.parametrize("tracked", [False, True])
def test_more_sequences_than_the_kernel_caches_lengths_of(tracked):
    _need_cuda()
    rng = np.random.default_rng(12)
    seqs = rng.integers(0, 90, 1300).tolist()
    seqs[0] = seqs[511] = seqs[512] = seqs[-1] = 0
    q, caches, k, v, bt, sl = fp4_case(seqs, 1, 2, 32, 16, seed=12)
    ref, probs = co.decode(q, k, v, bt, sl)
    w = torch.zeros(k.shape[0], 1, 16, device="cuda") if tracked else None
    out = pad_b200.paged_attention_decode_fp4(_cuda(q, torch.float16), *map(_cuda, caches), _cuda(bt), _cuda(sl),
                                              weights=w, num_new=100)
    assert_parity(out.float().cpu().numpy(), ref)
    if tracked:
        check_weights(w.cpu().numpy(), co.accumulate(np.zeros(tuple(w.shape)), probs, bt, sl, 100),
                      rel_bound(32, 90, smax_of(q, k, 32)))


@gpu
@pytest.mark.parametrize("d,ps", [(128, 1), (128, 5), (64, 16), (32, 48)])
def test_k_and_v_of_different_strides(d, ps):
    _need_cuda()
    q, caches, k, v, bt, sl = fp4_case([77, 300, 16], 3, 5, d, ps, seed=13)
    kc, ks, vc, vs = [_cuda(c) for c in caches]
    vc = _cuda(caches[2].transpose(0, 2, 1, 3)).permute(0, 2, 1, 3)  # V's pages head-major
    wide = torch.zeros(*vs.shape[:2], vs.shape[2] + 2, 4, dtype=torch.uint8, device="cuda")
    wide[:, :, : vs.shape[2]] = vs
    ref, _ = co.decode(q, k, v, bt, sl)
    out = pad_b200.paged_attention_decode_fp4(_cuda(q, torch.float16), kc, ks, vc, wide[:, :, : vs.shape[2]], _cuda(bt),
                                              _cuda(sl))
    assert_parity(out.float().cpu().numpy(), ref)


@gpu
def test_values_are_checked_when_asked_for(monkeypatch):
    """PAD_B200_CHECK: flags become the errors of the other entry points."""
    _need_cuda()
    from pad_b200 import kernel_cuda_v4

    monkeypatch.setattr(kernel_cuda_v4, "_CHECK_VALUES", True)
    caches = pad_b200.paged_kv_cache_fp4(4, 16, 2, 64)
    k16 = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda")
    q, new = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda"), torch.zeros(1, 2, 64, dtype=torch.float16, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    good, bad, w = i32([0, 1]), i32([0, 9]), torch.zeros(4, 2, 16, device="cuda")
    one, far = i32(20), i32(33)
    for call in (lambda bt, n: pad_b200.paged_attention_decode_fp4(q, *caches, bt, n),
                 lambda bt, n: pad_b200.paged_attention_decode_weights(q, k16, k16, bt, n, w),
                 lambda bt, n: pad_b200.paged_kv_evict_plan(w, bt, n, 4),
                 lambda bt, n: pad_b200.paged_kv_append_fp4(new, new, *caches, bt, n),
                 lambda bt, n: pad_b200.paged_kv_read_fp4(*caches, bt, n)):
        call(good, one)
        with pytest.raises(ValueError, match="page id"):
            call(bad, one)
        with pytest.raises(ValueError, match="seq_lens"):
            call(good, far)
    with pytest.raises(ValueError, match="seq_ids"):
        pad_b200.paged_kv_append_fp4(new, new, *caches, good, one, i32(1))
    many = torch.arange(4, dtype=torch.int32, device="cuda").repeat(40, 40)
    with pytest.raises(ValueError, match="share pages"):
        pad_b200.paged_attention_decode_fp4(q.expand(40, 4, 64).contiguous(), *caches, many,
                                            torch.full((40,), 640, dtype=torch.int32, device="cuda"), weights=w)


@gpu
def test_long_context_and_wide_table():
    _need_cuda()
    q, caches, k, v, bt, sl = fp4_case([70001, 50], 2, 6, 128, 32, seed=3)
    ref, _ = co.decode(q, k, v, bt, sl)
    wide = np.full((2, bt.shape[1] + 500), 10 ** 6, np.int32)  # ids behind the sequences are never read
    wide[:, : bt.shape[1]] = bt
    wide[1, 2:] = -5
    pad_b200.read_error_flags()
    out = pad_b200.paged_attention_decode_fp4(_cuda(q, torch.float16), *map(_cuda, caches), _cuda(wide), _cuda(sl))
    assert_parity(out.float().cpu().numpy(), ref)
    assert pad_b200.read_error_flags() == 0


@gpu
def test_large_scores_and_scales():
    """Scores of hundreds (one token takes all), V from 2^-24 to the largest block."""
    _need_cuda()
    rng = np.random.default_rng(4)
    d, ps, n = 128, 16, 200
    k = (rng.standard_normal((13, ps, 1, d)) * 30).astype(np.float16)
    v = np.zeros((13, ps, 1, d), np.float16)
    v[..., :32] = rng.standard_normal((13, ps, 1, 32)) * 6e-6  # scale at its least
    v[..., 32:64] = rng.standard_normal((13, ps, 1, 32)) * 10000
    v[..., 64:96] = rng.standard_normal((13, ps, 1, 32)) * 0.01
    (kc, ks), (vc, vs) = co.quantise(k), co.quantise(v)
    q = (rng.standard_normal((1, 4, d)) * 3).astype(np.float16)
    bt, sl = np.arange(13, dtype=np.int32)[None], np.array([n], np.int32)
    ref, _ = co.decode(q, co.dequantise(kc, ks), co.dequantise(vc, vs), bt, sl)
    out = pad_b200.paged_attention_decode_fp4(_cuda(q), _cuda(kc), _cuda(ks), _cuda(vc), _cuda(vs), _cuda(bt), _cuda(sl))
    got = out.double().cpu().numpy()
    # half a step of fp16, and the probabilities' own error: scores of up to 2^10 in log2 units off by
    # (D / 8 + 6) 2^-24 of it, so e^x by 1e-3; below 2^-14 fp16 has steps of 2^-24
    s = smax_of(q, co.dequantise(kc, ks), d)
    tol = np.abs(ref) * (2.0 ** -11 + 1e-5) + 2.0 ** -25 + rel_bound(d, n, s) * np.abs(co.dequantise(vc, vs)).max(0).max(0)
    assert np.all(np.abs(got - ref) <= tol)


@gpu
def test_garbage_behind_the_sequences_is_not_seen():
    _need_cuda()
    seqs = [1, 30, 100, 47]
    q, caches, k, v, bt, sl = fp4_case(seqs, 2, 4, 64, 16, seed=5)
    used = np.zeros(k.shape[:2], bool)
    for i, n in enumerate(seqs):
        t = np.arange(n)
        used[bt[i, t // 16], t % 16] = True
    kc, ks, vc, vs = [c.copy() for c in caches]
    ks[~used], vs[~used], kc[~used], vc[~used] = 255, 255, 0x7F, 0xF7  # NaN scales, codes of 6
    ref, _ = co.decode(q, k, v, bt, sl)
    out = pad_b200.paged_attention_decode_fp4(_cuda(q, torch.float16), _cuda(kc), _cuda(ks), _cuda(vc), _cuda(vs),
                                              _cuda(bt), _cuda(sl))
    assert_parity(out.float().cpu().numpy(), ref)


@gpu
@pytest.mark.parametrize("where", ["k", "v"])
def test_a_nan_block_reaches_its_sequence_alone(where):
    _need_cuda()
    q, caches, k, v, bt, sl = fp4_case([100, 50], 2, 2, 64, 16, seed=6)
    kc, ks, vc, vs = [c.copy() for c in caches]
    (ks if where == "k" else vs)[bt[0, 2], 3, 0, 1] = 255
    out = pad_b200.paged_attention_decode_fp4(_cuda(q, torch.float16), _cuda(kc), _cuda(ks), _cuda(vc), _cuda(vs),
                                              _cuda(bt), _cuda(sl))
    ref, _ = co.decode(q, k, v, bt, sl)
    got = out.float().cpu().numpy()
    if where == "k":
        assert np.isnan(got[0, :2]).all()
    else:  # the block's dims alone
        assert np.isnan(got[0, :2, 32:]).all()
        assert_parity(got[0, :2, :32], ref[0, :2, :32])
    assert_parity(got[0, 2:], ref[0, 2:])  # the other KV head
    assert_parity(got[1], ref[1])


@gpu
def test_strides_streams_and_graph():
    _need_cuda()
    seqs = [300, 77]
    q, caches, k, v, bt, sl = fp4_case(seqs, 3, 4, 64, 16, seed=7)
    ref, _ = co.decode(q, k, v, bt, sl, scale=0.2)
    qg = torch.zeros(2, 12, 80, dtype=torch.float16, device="cuda")
    qg[..., :64] = _cuda(q, torch.float16)
    cg = [_cuda(c.transpose(0, 2, 1, 3)).permute(0, 2, 1, 3) for c in caches]  # head-major pages
    out = torch.zeros(2, 12, 66, dtype=torch.float16, device="cuda")[..., :64]
    wide = torch.zeros(2, bt.shape[1] + 3, dtype=torch.int64, device="cuda")
    wide[:, : bt.shape[1]] = _cuda(bt)
    got = pad_b200.paged_attention_decode_fp4(qg[..., :64], *cg, wide, _cuda(sl).long(), scale=0.2, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert_parity(out.float().cpu().numpy(), ref)
    unaligned = torch.zeros(q.size + 1, dtype=torch.float16, device="cuda")[1:].view(2, 12, 64)
    unaligned.copy_(_cuda(q))
    btg, slg = _cuda(bt), _cuda(sl)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = pad_b200.paged_attention_decode_fp4(unaligned, *cg, btg, slg, scale=0.2)
    side.synchronize()
    # (a narrower table may split the sequences otherwise, so not bit for bit)
    assert_parity(a.float().cpu().numpy(), ref)
    graph = torch.cuda.CUDAGraph()
    w = torch.zeros(k.shape[0], 3, 16, device="cuda")
    pad_b200.paged_attention_decode_fp4(unaligned, *cg, btg, slg, scale=0.2, weights=w)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        b = pad_b200.paged_attention_decode_fp4(unaligned, *cg, btg, slg, scale=0.2, weights=w, num_new=10 ** 6)
    for lens in ([300, 77], [1, 16], [0, 64]):
        slg.copy_(torch.tensor(lens, dtype=torch.int32))
        w.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        ref, probs = co.decode(q, k, v, bt, lens, scale=0.2)
        assert_parity(b.float().cpu().numpy(), ref)
        want = co.accumulate(np.full(tuple(w.shape), 5.0), probs, bt, lens, 10 ** 6)
        check_weights(w.cpu().numpy(), want, rel_bound(64, 300, smax_of(q, k, 64)))


@gpu
def test_bad_pages_and_lengths_are_flagged():
    _need_cuda()
    pad_b200.read_error_flags()
    caches = pad_b200.paged_kv_cache_fp4(4, 16, 2, 64)
    q = torch.randn(2, 4, 64, device="cuda").half()
    bt = torch.tensor([[0, 9], [1, -1]], dtype=torch.int32, device="cuda")
    sl = torch.tensor([32, 16], dtype=torch.int32, device="cuda")
    for weights in (None, torch.zeros(4, 2, 16, device="cuda")):
        pad_b200.paged_attention_decode_fp4(q, *caches, bt, sl, weights=weights)
        assert pad_b200.read_error_flags() == _lib.PAD_FLAG_BAD_PAGE_ID
        pad_b200.paged_attention_decode_fp4(q, *caches, bt[:, :1], sl, weights=weights)
        assert pad_b200.read_error_flags() == _lib.PAD_FLAG_SEQ_LEN_RANGE
        pad_b200.paged_attention_decode_fp4(q, *caches, bt[:, :1], sl - 33, weights=weights)
        assert pad_b200.read_error_flags() == _lib.PAD_FLAG_SEQ_LEN_RANGE


@gpu
def test_offsets_past_32_bits():
    _need_cuda()
    q, caches, k, v, bt, sl = fp4_case([40], 1, 4, 64, 16, seed=8)
    far = []
    big = torch.zeros((11 << 29,), dtype=torch.uint8, device="cuda")
    for i, c in enumerate(caches):
        t = big[(i << 20):].as_strided(c.shape, (1 << 30, *_cuda(c).stride()[1:]))
        t.copy_(_cuda(c))
        far.append(t)
    assert far[0].shape[0] <= 6
    ref, _ = co.decode(q, k, v, bt, sl)
    out = pad_b200.paged_attention_decode_fp4(_cuda(q, torch.float16), *far, _cuda(bt), _cuda(sl))
    assert_parity(out.float().cpu().numpy(), ref)


@gpu
def test_empty_batch_and_refusals():
    _need_cuda()
    caches = pad_b200.paged_kv_cache_fp4(4, 16, 2, 64)
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")
    bt, sl = torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert pad_b200.paged_attention_decode_fp4(q[:0], *caches, bt[:0], sl[:0]).shape == (0, 4, 64)
    assert pad_b200.paged_attention_decode_fp4(q, *caches, bt, sl).eq(0).all()
    out = torch.full_like(q, 3.0)
    pad_b200.paged_attention_decode_fp4(q, *caches, bt[:, :0], sl, out=out)  # a table without columns: empty sequences
    assert out.eq(0).all()
    with pytest.raises(AssertionError):
        pad_b200.paged_attention_decode_fp4(q.float(), *caches, bt, sl)
    with pytest.raises(AssertionError):
        pad_b200.paged_attention_decode_fp4(q[:, :3], *caches, bt, sl)
    with pytest.raises(AssertionError):
        pad_b200.paged_attention_decode_fp4(q, *caches, bt, sl, slot_positions=sl)
    with pytest.raises(RuntimeError):
        pad_b200.paged_attention_decode_fp4(q, *caches, bt, torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError):
        pad_b200.paged_attention_decode_fp4(q, caches[0], caches[0], *caches[2:], bt, sl)
    with pytest.raises(RuntimeError):
        pad_b200.paged_attention_decode_fp4(torch.zeros(1, 34, 64, dtype=torch.float16, device="cuda"), *caches, bt, sl)
    with pytest.raises(RuntimeError):
        pad_b200.paged_attention_decode_fp4(q, *caches, bt, sl, weights=torch.zeros(4, 16, 2, device="cuda"))


def test_refusals_without_a_device():
    lib, p, a = _lib.load(), 1 << 20, _lib.i64_array

    def call(**over):
        kw = dict(q=p, k=p, ks=p, out=p, w=0, sp=0, tl=0, new=1, b=2, hq=12, hkv=2, d=128, ps=16, maxp=4,
                  qs=[1536, 128, 1], kst=[2048, 128, 64, 1], kss=[128, 8, 4, 1], bts=4, os=[1536, 128, 1], scale=0.1)
        kw.update(over)
        return lib.pad_paged_attention_decode_fp4(
            kw["q"], kw["k"], kw["ks"], p, p, p, p, kw["out"], kw["w"], kw["sp"], kw["tl"], kw["new"], kw["b"],
            kw["hq"], kw["hkv"], kw["d"], 10, kw["ps"], kw["maxp"], a(kw["qs"]), a(kw["kst"]), a(kw["kss"]),
            a([2048, 128, 64, 1]), a([128, 8, 4, 1]), kw["bts"], a(kw["os"]), None, None, kw["scale"], 0, 0, 0, 0, 0)

    inv, uns = _lib.PAD_ERR_INVALID_ARGUMENT, _lib.PAD_ERR_UNSUPPORTED
    for over, status, text in [
            (dict(b=-1), inv, b"size"), (dict(ps=0), inv, b"size"), (dict(d=16), uns, b"head_dim"),
            (dict(hq=11), inv, b"divisible"), (dict(hq=34), uns, b"gqa_ratio"), (dict(scale=float("nan")), inv, b"scale"),
            (dict(new=-1), inv, b"num_new"), (dict(k=0), inv, b"null"), (dict(w=p), inv, b"null"),
            (dict(sp=p), inv, b"null"), (dict(qs=[1536, 128, 2]), uns, b"contiguous"),
            (dict(kst=[2048, 120, 64, 1]), uns, b"16 bytes"), (dict(kss=[128, 6, 4, 1]), uns, b"scale strides"),
            (dict(q=p + 2), uns, b"q must be"), (dict(out=p + 2), uns, b"out must be"), (dict(k=p + 4), uns, b"aligned"),
            (dict(bts=3), inv, b"stride"), (dict(ps=1 << 30), uns, b"32-bit")]:
        assert call(**over) == status, over
        assert b"decode_fp4" in lib.pad_last_error() and text in lib.pad_last_error(), over
    assert call(b=0) == _lib.PAD_OK


def _foreign(rng, seqs, hkv, g, d, ps):
    """A cache that another writer filled: random codes and scale bytes (K's near 2^-2, V's 2^-4 to 2^2)."""
    need = [-(-n // ps) for n in seqs]
    pages = sum(need) + 1
    perm = rng.permutation(pages).astype(np.int32)
    bt = np.zeros((len(seqs), max(max(need), 1)), np.int32)
    at = 0
    for i, n in enumerate(need):
        bt[i, :n] = perm[at:at + n]
        at += n
    codes = lambda: rng.integers(0, 256, (pages, ps, hkv, d // 2)).astype(np.uint8)  # noqa: E731
    scales = lambda lo, hi: rng.integers(lo, hi, (pages, ps, hkv, 4)).astype(np.uint8)  # noqa: E731
    q = (rng.standard_normal((len(seqs), hkv * g, d)) * 0.3).astype(np.float16)
    return q, codes(), scales(124, 127), codes(), scales(123, 130), bt, np.asarray(seqs, np.int32)


def _check_foreign(q, kc, ks, vc, vs, bt, sl, num_splits=None, weights=False, off_v=0.0):
    """Half a step of fp16 on the result; each probability off by its bound (test_decode_weights.py) and by the 2^-25 that
    P's two fp16 terms resolve (the largest P is at least 1); every value off by off_v."""
    k, v = co.dequantise(kc, ks), co.dequantise(vc, vs)
    ref, probs = co.decode(q, k, v, bt, sl)
    w = torch.zeros(k.shape[0], k.shape[2], k.shape[1], device="cuda") if weights else None
    out = pad_b200.paged_attention_decode_fp4(*map(_cuda, (q, kc, ks, vc, vs, bt, sl)), num_splits, weights=w)
    got = out.double().cpu().numpy()
    hkv, d = k.shape[2], k.shape[3]
    bound = rel_bound(d, int(max(sl)), smax_of(q.astype(np.float64), k, d))
    for i, n in enumerate(sl):
        vv = np.abs(co.gather(v, bt[i], int(n)))  # [n, Hkv, D]
        terms = bound * np.einsum("th,thd->hd", probs[i], vv) + 2.0 ** -25 * vv.sum(0)
        want = ref[i].reshape(hkv, -1, d)
        tol = np.abs(want) * 2.0 ** -11 + 2.0 ** -25 + terms[:, None] + off_v
        off = np.abs(got[i].reshape(want.shape) - want)
        assert np.all(off <= tol), f"sequence {i}: off by {np.nanmax(off / tol):.3g} of the tolerance"
    if weights:
        check_weights(w.cpu().numpy(), co.accumulate(np.zeros(tuple(w.shape)), probs, bt, sl, 1), bound)


@gpu
@pytest.mark.parametrize("byte", [140, 139, 103, 102, 95, 3, 0])
@pytest.mark.parametrize("d,g", [(128, 2), (64, 12), (32, 5)])
def test_v_scales_at_the_ends_of_fp16(byte, d, g):
    """Up to 2^13 exact; below 2^-24 a scale counts as 0, so a value (6 x 2^-25 at most) is off by itself. At 2^-24 the
    codes 0.5 and 1.5 lie between two fp16 values (no append writes them there): half a step of 2^-24."""
    _need_cuda()
    pad_b200.read_error_flags()
    rng = np.random.default_rng(byte + d)
    q, kc, ks, vc, vs, bt, sl = _foreign(rng, [1, 40, 200], 2, g, d, 16)
    if byte > 127:  # a few tokens of them, in some blocks
        vs[rng.random(vs.shape) < 0.1] = byte
    else:
        vs[:] = byte
    for num_splits, weights in ((None, False), (3, True)):
        _check_foreign(q, kc, ks, vc, vs, bt, sl, num_splits, weights,
                       off_v=6 * 2.0 ** -25 if byte < 103 else 2.0 ** -25 if byte == 103 else 0.0)
    assert pad_b200.read_error_flags() == 0


@gpu
@pytest.mark.parametrize("byte", [141, 142, 200, 254, 255])
@pytest.mark.parametrize("d,g", [(128, 2), (64, 12), (32, 5)])
def test_v_scales_above_the_largest_are_flagged(byte, d, g, monkeypatch):
    """In a block that a sequence attends to, wherever its token lies; NaN (255) is none of them."""
    _need_cuda()
    from pad_b200 import kernel_cuda_v4

    pad_b200.read_error_flags()
    rng = np.random.default_rng(byte)
    q, kc, ks, vc, vs, bt, sl = _foreign(rng, [300, 40, 200], 2, g, d, 16)
    vs -= 3  # values below 4, where the parity bound holds fp16's half step
    flag = 0 if byte == 255 else _lib.PAD_FLAG_SCALE_RANGE
    qg, kcg, ksg, vcg, btg, slg = map(_cuda, (q, kc, ks, vc, bt, sl))
    run = lambda x, **kw: pad_b200.paged_attention_decode_fp4(qg, kcg, ksg, vcg, _cuda(x), btg, slg, **kw)  # noqa: E731
    ref, _ = co.decode(q, co.dequantise(kc, ks), co.dequantise(vc, vs), bt, sl)
    for i, t, blk in [(0, 0, 0), (0, 299, d // 32 - 1), (0, 150, 0), (1, 39, d // 32 - 1)]:
        bad = vs.copy()
        bad[bt[i, t // 16], t % 16, 1, blk] = byte
        for kw in ({}, dict(num_splits=3), dict(weights=torch.zeros(kc.shape[0], 2, 16, device="cuda"))):
            out = run(bad, **kw).float().cpu().numpy()
            assert pad_b200.read_error_flags() == flag
            for j in range(3):  # the other sequences, and the other head
                assert_parity(out[j, : g if j == i else 2 * g], ref[j, : g if j == i else 2 * g])
    if flag:
        monkeypatch.setattr(kernel_cuda_v4, "_CHECK_VALUES", True)
        with pytest.raises(ValueError, match="v_scales"):
            run(bad)
        run(vs)
        monkeypatch.setattr(kernel_cuda_v4, "_CHECK_VALUES", False)
    # behind a sequence, in a page of none, and in the unused bytes of a row: never looked at
    bad = vs.copy()
    bad[..., d // 32:] = byte
    for i, n in enumerate(sl):
        bad[bt[i, n // 16], n % 16:] = byte  # (no length is a multiple of the page)
    bad[sorted(set(range(len(bad))) - {int(x) for i, n in enumerate(sl) for x in bt[i, : -(-n // 16)]})] = byte
    assert_parity(run(bad).float().cpu().numpy(), ref)
    assert pad_b200.read_error_flags() == 0


@gpu
@pytest.mark.parametrize("n", [1, 100])
@pytest.mark.parametrize("num_splits", [None, 3])
def test_scores_far_below_zero(n, num_splits):
    """Every score below -1e31: the largest of them still takes all."""
    _need_cuda()
    caches = pad_b200.paged_kv_cache_fp4(7, 16, 1, 64)
    caches[0].fill_(0xFF)  # keys of -6 ...
    caches[0][(n - 1) // 16, (n - 1) % 16] = 0x99  # ... and, in the last token, of -0.5
    caches[1].fill_(127)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    v = torch.randint(0, 256, caches[2].shape, device="cuda", generator=gen).to(torch.uint8)
    caches[2].copy_(v), caches[3].fill_(127)
    q = torch.ones(1, 2, 64, dtype=torch.float16, device="cuda")
    bt, sl = torch.arange(7, dtype=torch.int32, device="cuda").view(1, 7), torch.tensor([n], dtype=torch.int32, device="cuda")
    w = torch.zeros(7, 1, 16, device="cuda")
    out = pad_b200.paged_attention_decode_fp4(q, *caches, bt, sl, num_splits, scale=1e32, weights=w, num_new=10 ** 6)
    want = co.dequantise(caches[2].cpu().numpy(), caches[3].cpu().numpy())[(n - 1) // 16, (n - 1) % 16, 0]
    np.testing.assert_array_equal(out[0].double().cpu().numpy(), np.stack([want, want]))
    got = w[:, 0].flatten()
    assert got[n - 1].item() == 2.0 and got.sum().item() == 2.0


@gpu
@pytest.mark.parametrize("hkv,g,d,ps", [(2, 6, 128, 16), (3, 12, 32, 7)])
@pytest.mark.parametrize("num_splits", [None, 3])
def test_new_tokens_of_each_sequence(hkv, g, d, ps, num_splits):
    _need_cuda()
    seqs = [0, 1, 17, 300, 4000, 65, 64]
    q, caches, k, v, bt, sl = fp4_case(seqs, hkv, g, d, ps, seed=22)
    rng = np.random.default_rng(22)
    w0 = rng.random((k.shape[0], hkv, ps)).astype(np.float32)
    at0 = rng.integers(0, 99, w0.shape).astype(np.int32)
    total = np.asarray(seqs, np.int64) + 7
    ref, probs = co.decode(q, k, v, bt, sl)
    want_w, want_at = by_sequence(w0, at0, probs, bt, seqs, total, NEWS)
    w, at = _cuda(w0), _cuda(at0)
    out = pad_b200.paged_attention_decode_fp4(_cuda(q, torch.float16), *map(_cuda, caches), _cuda(bt), _cuda(sl),
                                              num_splits, weights=w, num_new=torch.tensor(NEWS, device="cuda"),
                                              slot_positions=at, total_lens=_cuda(total))
    assert_parity(out.float().cpu().numpy(), ref)
    check_weights(w.cpu().numpy(), want_w, rel_bound(d, 4000, smax_of(q, k, d)))
    np.testing.assert_array_equal(at.cpu().numpy(), want_at)
    with pytest.raises(RuntimeError, match="num_new"):
        pad_b200.paged_attention_decode_fp4(_cuda(q, torch.float16), *map(_cuda, caches), _cuda(bt), _cuda(sl),
                                            weights=w, num_new=torch.ones(6, dtype=torch.int32, device="cuda"))


def test_new_tokens_by_sequence_refusals_without_a_device():
    lib, p, a = _lib.load(), 1 << 20, _lib.i64_array
    call = lambda new, b, hq=12: lib.pad_paged_attention_decode_fp4_by_seq(  # noqa: E731
        p, p, p, p, p, p, p, p, p, 0, 0, new, b, hq, 2, 128, 10, 16, 4, a([1536, 128, 1]), a([2048, 128, 64, 1]),
        a([128, 8, 4, 1]), a([2048, 128, 64, 1]), a([128, 8, 4, 1]), 4, a([1536, 128, 1]), a([32, 16, 1]), None, 0.1, 0,
        0, 0, 0, 0)
    for new, hq, text in [(0, 12, b"num_new"), (p, 11, b"divisible")]:
        assert call(new, 2, hq) == _lib.PAD_ERR_INVALID_ARGUMENT and text in lib.pad_last_error()
    assert call(0, 0) == _lib.PAD_OK


@gpu
@pytest.mark.parametrize("alike", [True, False])
@pytest.mark.parametrize("bad_id", [-1, 10 ** 6])
def test_a_bad_page_reads_as_zero_rows(alike, bad_id):
    """Page 0 and the pages read before hold no zeros, so that anything read in a bad page's place shows."""
    _need_cuda()
    pad_b200.read_error_flags()
    q, caches, k, v, bt, sl = fp4_case([100, 64, 90], 2, 4, 64, 16, seed=31)
    (kc, ks), (vc, vs) = [[c.copy() for c in x] for x in (caches[:2], caches[2:])]
    kc[0], vc[0], ks[0], vs[0] = 0x77, 0x77, 126, 126  # values of 3
    pages = k.shape[0]
    bt = bt.copy()
    bt[0, 1] = bt[2, 0] = bad_id
    zeros = lambda c: np.concatenate([c, np.zeros_like(c[:1])])  # noqa: E731  (one more page, of zeros)
    good = np.where(bt == bad_id, pages, bt)
    ref, probs = co.decode(q, co.dequantise(zeros(kc), zeros(ks)), co.dequantise(zeros(vc), zeros(vs)), good, sl)
    cg = [_cuda(c) for c in (kc, ks, vc, vs)]
    if not alike:
        cg[2] = _cuda(vc.transpose(0, 2, 1, 3)).permute(0, 2, 1, 3)
    w = torch.zeros(pages, 2, 16, device="cuda")
    for weights in (None, w):
        out = pad_b200.paged_attention_decode_fp4(_cuda(q, torch.float16), *cg, _cuda(bt), _cuda(sl), weights=weights,
                                                  num_new=10 ** 6)
        assert_parity(out.float().cpu().numpy(), ref)
        assert pad_b200.read_error_flags() == _lib.PAD_FLAG_BAD_PAGE_ID
    want = co.accumulate(np.zeros((pages + 1, 2, 16)), probs, good, sl, 10 ** 6)[:pages]
    check_weights(w.cpu().numpy(), want, rel_bound(64, 100, smax_of(q, co.dequantise(kc, ks), 64)))
