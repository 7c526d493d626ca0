"""Decode that accumulates attention weights, against float64.

Tolerances. out: the parity bound of the other decode tests (gpu_utils), and
for these inputs (|v| < 8) the fp16 rounding 2^-11 |out| is far inside it.
weights (fp32): the score in log2 units, |s| <= S, carries fp32 rounding of the
dot product and of two multiplications, at most (D / 16 + 3) steps of 2^-24 S
(a dot product of D terms goes through D / 16 tensor-core steps, each rounded
once or truncated, 2^-23), the exponential 2^-22, the sums l and over G heads
under (T / 16 + 150 + G) 2^-24; a probability's relative error is below
    (D / 8 + 6) 2^-24 S ln 2 + 2^-22 + (T / 16 + 170) 2^-24,
and each addition to an old weight adds 2^-24 of it. Absolute: the same times
the row's probabilities' sum G <= 16, never needed below 1e-7."""

import numpy as np
import pytest
import torch

import cache_oracle as co
import pad_b200
from gpu_utils import assert_parity
from pad_b200 import _lib
from pad_b200.cases import explicit_case

gpu = pytest.mark.gpu


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _cuda(x, dt=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dt is None else t.to(dt)


def rel_bound(d, longest, smax):
    return (d / 8 + 6) * 2.0 ** -24 * smax * np.log(2) + 2.0 ** -22 + (longest / 16 + 170) * 2.0 ** -24


def smax_of(q, k, d):
    """Largest |score| in log2 units that these inputs can give."""
    return float(np.linalg.norm(q, axis=-1).max() * np.linalg.norm(k, axis=-1).max() / np.sqrt(d) * np.log2(np.e))


def check_weights(got, want, bound):
    err = np.abs(got.astype(np.float64) - want)
    tol = bound * np.abs(want) + 1e-7
    assert np.all(err <= tol), f"weights off by {np.max(err / tol):.2f} of the tolerance"


def _case_inputs(c):
    return (_cuda(c.q, torch.float16), _cuda(c.k_cache, torch.float16), _cuda(c.v_cache, torch.float16),
            _cuda(c.block_table), _cuda(c.seq_lens))


CASES = [
    # seq_lens, heads, G, D, page
    ([1], 1, 1, 128, 16),
    ([4096], 2, 6, 128, 16),
    ([0, 1, 17, 300, 4000, 65, 0], 2, 6, 128, 16),
    ([5, 70, 333], 4, 4, 64, 4),
    ([129, 1000, 31], 8, 8, 128, 16),
    ([700, 64], 3, 5, 32, 24),
    ([900, 20], 4, 16, 128, 32),
    ([100, 257], 1, 12, 16, 1),
    ([2000] * 8, 8, 4, 128, 16),
    ([20000], 8, 1, 64, 64),
]


@gpu
@pytest.mark.parametrize("seqs,hkv,g,d,ps", CASES)
@pytest.mark.parametrize("num_splits", [None, 1, 3])
def test_weights_and_positions_match_float64(seqs, hkv, g, d, ps, num_splits):
    _need_cuda()
    pad_b200.read_error_flags()
    c = explicit_case(seqs, num_kv_heads=hkv, gqa_ratio=g, head_dim=d, page_size=ps, seed=d + g)
    rng = np.random.default_rng(1)
    pages = c.k_cache.shape[0]
    w0 = rng.random((pages, hkv, ps)).astype(np.float32)
    at0 = rng.integers(0, 99, (pages, hkv, ps)).astype(np.int32)
    total = np.asarray(seqs, np.int64) + 7
    ref, probs = co.decode(c.q, c.k_cache, c.v_cache, c.block_table, c.seq_lens)
    bound = rel_bound(d, max(seqs), smax_of(c.q, c.k_cache, d))
    q, k, v, bt, sl = _case_inputs(c)
    for num_new in (1, 0, 5, 2 ** 31 - 1):
        w, at = _cuda(w0), _cuda(at0)
        out = pad_b200.paged_attention_decode_weights(q, k, v, bt, sl, w, num_new, num_splits, slot_positions=at,
                                                      total_lens=_cuda(total))
        assert_parity(out.float().cpu().numpy(), ref)
        want = co.accumulate(w0, probs, c.block_table, c.seq_lens, num_new)
        check_weights(w.cpu().numpy(), want, bound)
        want_at = at0.copy()
        for i, n in enumerate(seqs):
            for t in range(max(0, n - num_new), n):
                want_at[c.block_table[i, t // ps], :, t % ps] = total[i] - n + t
        np.testing.assert_array_equal(at.cpu().numpy(), want_at)
    assert pad_b200.read_error_flags() == 0


@gpu
def test_more_sequences_than_the_kernel_caches_lengths_of():
    _need_cuda()
    rng = np.random.default_rng(13)
    seqs = rng.integers(0, 40, 1500).tolist()
    c = explicit_case(seqs, num_kv_heads=1, gqa_ratio=2, head_dim=16, page_size=8, seed=13)
    ref, probs = co.decode(c.q, c.k_cache, c.v_cache, c.block_table, c.seq_lens)
    q, k, v, bt, sl = _case_inputs(c)
    w = torch.zeros(k.shape[0], 1, 8, device="cuda")
    out = pad_b200.paged_attention_decode_weights(q, k, v, bt, sl, w, num_new=40)
    assert_parity(out.float().cpu().numpy(), ref)
    check_weights(w.cpu().numpy(), co.accumulate(np.zeros(tuple(w.shape)), probs, c.block_table, c.seq_lens, 40),
                  rel_bound(16, 40, smax_of(c.q, c.k_cache, 16)))


@gpu
def test_out_is_the_decode_without_weights_bit_for_bit():
    _need_cuda()
    c = explicit_case([3000, 17, 900], num_kv_heads=2, gqa_ratio=6, head_dim=128, page_size=16, seed=3)
    q, k, v, bt, sl = _case_inputs(c)
    w = torch.zeros(k.shape[0], 2, 16, device="cuda")
    a = pad_b200.paged_attention_decode_weights(q, k, v, bt, sl, w)
    b = pad_b200.paged_attention_decode_cuda_v4(q, k, v, bt, sl)
    assert torch.equal(a, b)
    first = w.clone()
    w.zero_()
    pad_b200.paged_attention_decode_weights(q, k, v, bt, sl, w)
    assert torch.equal(w, first)  # repeatable


@gpu
def test_weights_sum_to_the_query_heads_and_add_up_over_steps():
    """Each head group's probabilities sum to G; repeated calls add."""
    _need_cuda()
    seqs, hkv, g, ps = [5000, 333], 4, 5, 16
    c = explicit_case(seqs, num_kv_heads=hkv, gqa_ratio=g, head_dim=64, page_size=ps, seed=4)
    q, k, v, bt, sl = _case_inputs(c)
    w = torch.full((k.shape[0], hkv, ps), 3.0, device="cuda")
    pad_b200.paged_attention_decode_weights(q, k, v, bt, sl, w, num_new=10 ** 6)
    one = w.double().cpu()
    for i, n in enumerate(seqs):
        pages = c.block_table[i, : -(-n // ps)]
        s = one[pages].permute(1, 0, 2).reshape(hkv, -1)[:, :n].sum(1)
        # G sums of n terms, each within the bound above (T = 5000, |s| < 40)
        assert torch.allclose(s, torch.full_like(s, g), rtol=rel_bound(64, 5000, 40), atol=0)
    used = torch.zeros(k.shape[0], ps, dtype=torch.bool)
    for i, n in enumerate(seqs):
        t = np.arange(n)
        used[c.block_table[i, t // ps], t % ps] = True
    assert (one.permute(0, 2, 1)[~used] == 3.0).all()  # slots behind the sequences stay
    pad_b200.paged_attention_decode_weights(q, k, v, bt, sl, w, num_new=0)
    two = w.double().cpu()
    both = used[:, None, :].expand_as(two)
    assert torch.allclose(two[both], 2 * one[both], rtol=2.0 ** -23, atol=0)


@gpu
def test_garbage_behind_the_sequences_and_in_other_pages_is_not_seen():
    _need_cuda()
    seqs = [1, 30, 100]
    c = explicit_case(seqs, num_kv_heads=2, gqa_ratio=4, head_dim=64, page_size=16, seed=5)
    k, v = c.k_cache.copy(), c.v_cache.copy()
    used = np.zeros(k.shape[:2], bool)
    for i, n in enumerate(seqs):
        t = np.arange(n)
        used[c.block_table[i, t // 16], t % 16] = True
    k[~used], v[~used] = np.nan, np.inf
    w0 = np.full((k.shape[0], 2, 16), np.nan, np.float32)
    w = _cuda(w0)
    q, kg, vg = _cuda(c.q, torch.float16), _cuda(k, torch.float16), _cuda(v, torch.float16)
    pad_b200.paged_attention_decode_weights(q, kg, vg, _cuda(c.block_table), _cuda(c.seq_lens), w, num_new=200)
    _, probs = co.decode(c.q, c.k_cache, c.v_cache, c.block_table, c.seq_lens)
    got = w.cpu().numpy()
    assert np.isnan(got.transpose(0, 2, 1)[~used]).all()
    want = co.accumulate(np.zeros_like(w0), probs, c.block_table, c.seq_lens, 200)
    check_weights(np.where(np.isnan(got), 0, got), want, rel_bound(64, 100, smax_of(c.q, c.k_cache, 64)))


@gpu
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_a_nan_or_infinite_key_reaches_its_sequence_alone(value):
    _need_cuda()
    c = explicit_case([100, 50], num_kv_heads=1, gqa_ratio=2, head_dim=64, page_size=16, seed=6)
    k = c.k_cache.copy()
    k[c.block_table[0, 2], 3, 0, :] = value  # inf - inf in the dot product, or NaN: every weight of sequence 0
    w = torch.zeros(k.shape[0], 1, 16, device="cuda")
    out = pad_b200.paged_attention_decode_weights(_cuda(c.q, torch.float16), _cuda(k, torch.float16),
                                                  _cuda(c.v_cache, torch.float16), _cuda(c.block_table),
                                                  _cuda(c.seq_lens), w)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()
    row = w[c.block_table[0, :7]].flatten()[:100]
    assert torch.isnan(row).all()
    assert torch.isfinite(w[c.block_table[1, :4]]).all()


@gpu
def test_strides_out_and_scale():
    _need_cuda()
    seqs, hkv, g, d, ps = [300, 77], 2, 4, 64, 16
    c = explicit_case(seqs, num_kv_heads=hkv, gqa_ratio=g, head_dim=d, page_size=ps, seed=7)
    q, k, v, bt, sl = _case_inputs(c)
    pages = k.shape[0]
    w = torch.zeros(ps, pages, hkv, device="cuda").permute(1, 2, 0)  # any strides
    at = torch.zeros(pages, hkv, 2 * ps, dtype=torch.int32, device="cuda")[:, :, ::2]
    out = torch.full_like(q, 7.0)
    wide = torch.zeros(2, bt.shape[1] + 9, dtype=torch.int64, device="cuda")
    wide[:, : bt.shape[1]] = bt
    got = pad_b200.paged_attention_decode_weights(q, k, v, wide, sl.long(), w, 400, scale=0.3, slot_positions=at, out=out)
    assert got.data_ptr() == out.data_ptr()
    ref, probs = co.decode(c.q, c.k_cache, c.v_cache, c.block_table, c.seq_lens, scale=0.3)
    assert_parity(out.float().cpu().numpy(), ref)
    want = co.accumulate(np.zeros((pages, hkv, ps)), probs, c.block_table, c.seq_lens, 400)
    check_weights(w.cpu().numpy(), want, rel_bound(d, 300, smax_of(c.q, c.k_cache, d) * 0.3 * 8))
    want_at = np.zeros((pages, hkv, ps), np.int32)
    for i, n in enumerate(seqs):  # total_lens defaults to seq_lens: positions are the slots
        for t in range(n):
            want_at[c.block_table[i, t // ps], :, t % ps] = t
    np.testing.assert_array_equal(at.cpu().numpy(), want_at)


@gpu
def test_bad_pages_lengths_and_shared_pages_are_flagged():
    _need_cuda()
    pad_b200.read_error_flags()
    q = torch.randn(2, 4, 64, device="cuda").half()
    k = torch.randn(4, 16, 2, 64, device="cuda").half()
    w = torch.zeros(4, 2, 16, device="cuda")
    sl = torch.tensor([32, 32], device="cuda")
    bt = torch.tensor([[0, 9], [1, 2]], dtype=torch.int32, device="cuda")
    pad_b200.paged_attention_decode_weights(q, k, k, bt, sl, w)
    assert pad_b200.read_error_flags() == _lib.PAD_FLAG_BAD_PAGE_ID
    assert w[3].eq(0).all()
    bt[0, 1] = 3
    pad_b200.paged_attention_decode_weights(q, k, k, bt, sl + 1, w)
    assert pad_b200.read_error_flags() == _lib.PAD_FLAG_SEQ_LEN_RANGE
    # 40 sequences over the same 4 pages: more tokens than the pool holds
    q, bt = torch.randn(40, 4, 64, device="cuda").half(), torch.arange(4, device="cuda").repeat(40, 40)
    out = pad_b200.paged_attention_decode_weights(q, k, k, bt, torch.full((40,), 640, device="cuda"), w)
    assert pad_b200.read_error_flags() == _lib.PAD_FLAG_SHARED_PAGE
    assert torch.equal(out, pad_b200.paged_attention_decode_cuda_v4(q, k, k, bt, torch.full((40,), 640, device="cuda")))


@gpu
def test_two_streams_and_two_graphs_keep_their_own_workspaces():
    _need_cuda()
    cases = [explicit_case([2500, 40], num_kv_heads=2, gqa_ratio=6, head_dim=128, page_size=16, seed=s) for s in (8, 9)]
    ins = [_case_inputs(c) for c in cases]
    ws = [torch.zeros(i[1].shape[0], 2, 16, device="cuda") for i in ins]
    want = []
    for i, w in zip(ins, ws):
        out = pad_b200.paged_attention_decode_weights(*i, w, 10 ** 6)
        want.append((out.clone(), w.clone()))
        w.zero_()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i, w in zip(ins, ws):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pad_b200.paged_attention_decode_weights(*i, w, 10 ** 6))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w, (wo, ww) in zip(outs, ws, want):
        assert torch.equal(o, wo) and torch.equal(w, ww)


def test_refusals_without_a_device():
    lib = _lib.load()
    p = 1 << 20
    a = _lib.i64_array

    def call(**over):
        kw = dict(w=p, sp=0, tl=0, new=1, ws=a([32, 16, 1]), pst=a([32, 16, 1]), hq=12)
        kw.update(over)
        return lib.pad_paged_attention_decode_weights(
            p, p, p, p, p, p, kw["w"], kw["sp"], kw["tl"], kw["new"], 2, kw["hq"], 2, 128, 10, 16, 4,
            a([1536, 128, 1]), a([4096, 256, 128, 1]), a([4096, 256, 128, 1]), 4, a([1536, 128, 1]), kw["ws"],
            kw["pst"], 0.088, 0, 0, 0, 0, 0)

    for over, text in [(dict(w=0), b"weights"), (dict(ws=None), b"weights"), (dict(new=-1), b"num_new"),
                       (dict(sp=p), b"total_lens"), (dict(sp=p, tl=p, pst=None), b"position_strides"),
                       (dict(hq=11), b"divisible")]:
        assert call(**over) == _lib.PAD_ERR_INVALID_ARGUMENT, over
        assert text in lib.pad_last_error()
    q = torch.zeros(1, 12, 128, dtype=torch.float16)
    k = torch.zeros(4, 16, 2, 128, dtype=torch.float16)
    with pytest.raises(AssertionError):
        pad_b200.paged_attention_decode_weights(q, k, k, torch.zeros(1, 4, dtype=torch.int32),
                                                torch.ones(1, dtype=torch.int32), torch.zeros(4, 2, 16))


@gpu
def test_wrong_weights_are_refused():
    _need_cuda()
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda")
    bt, sl = torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    w = torch.zeros(4, 2, 16, device="cuda")
    for bad in (w.half(), w[:3], w.transpose(1, 2), w.cpu()):
        with pytest.raises((RuntimeError, NotImplementedError)):
            pad_b200.paged_attention_decode_weights(q, k, k, bt, sl, bad)
    with pytest.raises(RuntimeError):
        pad_b200.paged_attention_decode_weights(q, k, k, bt, sl, w, slot_positions=w)
    with pytest.raises(AssertionError):
        pad_b200.paged_attention_decode_weights(q, k, k, bt, sl, w, num_new=-1)
    with pytest.raises(AssertionError):
        pad_b200.paged_attention_decode_weights(q, k, k, bt, sl, w, total_lens=sl)


NEWS = [1, 10 ** 6, 0, 7, 1, -3, 65]  # one of each of the sequences [0, 1, 17, 300, 4000, 65, 64]


def by_sequence(w0, at0, probs, bt, seqs, total, news):
    """weights and slot_positions after a step with a number of new tokens for each sequence."""
    w, at, ps = w0.astype(np.float64), at0.copy(), w0.shape[2]
    for i, n in enumerate(seqs):
        new = min(max(news[i], 0), n)
        w = co.accumulate(w, [probs[i]], bt[i:i + 1], seqs[i:i + 1], new)
        for t in range(n - new, n):
            at[bt[i, t // ps], :, t % ps] = total[i] - n + t
    return w, at


@gpu
@pytest.mark.parametrize("hkv,g,d,ps", [(2, 6, 128, 16), (3, 12, 16, 7)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.int16])
def test_new_tokens_of_each_sequence(hkv, g, d, ps, dtype):
    _need_cuda()
    seqs = [0, 1, 17, 300, 4000, 65, 64]
    c = explicit_case(seqs, num_kv_heads=hkv, gqa_ratio=g, head_dim=d, page_size=ps, seed=21)
    rng = np.random.default_rng(21)
    w0 = rng.random((c.k_cache.shape[0], hkv, ps)).astype(np.float32)
    at0 = rng.integers(0, 99, w0.shape).astype(np.int32)
    total = np.asarray(seqs, np.int64) + 7
    ref, probs = co.decode(c.q, c.k_cache, c.v_cache, c.block_table, c.seq_lens)
    want_w, want_at = by_sequence(w0, at0, probs, c.block_table, seqs, total, NEWS)
    q, k, v, bt, sl = _case_inputs(c)
    news = torch.tensor([min(n, torch.iinfo(dtype).max) for n in NEWS], dtype=dtype, device="cuda")
    if dtype == torch.int64:
        news[1] = 2 ** 40  # past 32 bits: all of the sequence
    w, at = _cuda(w0), _cuda(at0)
    out = pad_b200.paged_attention_decode_weights(q, k, v, bt, sl, w, news, slot_positions=at, total_lens=_cuda(total))
    assert_parity(out.float().cpu().numpy(), ref)
    check_weights(w.cpu().numpy(), want_w, rel_bound(d, 4000, smax_of(c.q, c.k_cache, d)))
    np.testing.assert_array_equal(at.cpu().numpy(), want_at)


@gpu
def test_wrong_numbers_of_new_tokens_are_refused():
    _need_cuda()
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda")
    bt, sl = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    w = torch.zeros(4, 2, 16, device="cuda")
    for bad in (sl[:1], sl.float(), sl.view(2, 1), sl.bool()):
        with pytest.raises(RuntimeError, match="num_new"):
            pad_b200.paged_attention_decode_weights(q, k, k, bt, sl, w, bad)


def test_new_tokens_by_sequence_refusals_without_a_device():
    lib, p, a = _lib.load(), 1 << 20, _lib.i64_array

    def call(**over):
        kw = dict(w=p, new=p, b=2, hq=12)
        kw.update(over)
        return lib.pad_paged_attention_decode_weights_by_seq(
            p, p, p, p, p, p, kw["w"], 0, 0, kw["new"], kw["b"], kw["hq"], 2, 128, 10, 16, 4, a([1536, 128, 1]),
            a([4096, 256, 128, 1]), a([4096, 256, 128, 1]), 4, a([1536, 128, 1]), a([32, 16, 1]), None, 0.088, 0, 0, 0,
            0, 0)

    for over, text in [(dict(new=0), b"num_new"), (dict(w=0), b"weights"), (dict(hq=11), b"divisible")]:
        assert call(**over) == _lib.PAD_ERR_INVALID_ARGUMENT, over
        assert text in lib.pad_last_error()
    assert call(b=0, new=0) == _lib.PAD_OK
