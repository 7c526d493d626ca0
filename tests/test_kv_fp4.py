"""The 4-bit paged cache: append and read-back against a numpy quantiser, bit
for bit (the format has one rounding, so there is nothing to tolerate)."""

import numpy as np
import pytest
import torch

import cache_oracle as co
import pad_b200
from pad_b200 import _lib


def _values(rng, shape):
    """fp16 values of very different magnitudes, blocks of zeros, subnormals and ties among them."""
    x = rng.standard_normal(shape) * np.exp2(rng.integers(-24, 14, size=(*shape[:-1], 1)))
    x = np.clip(x, -65504, 65504).astype(np.float16)
    flat = x.reshape(-1, 32)
    flat[0] = 0
    flat[1] = np.float16(-0.0)
    flat[2] = np.tile(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0], np.float16), 4)  # ties, saturation
    flat[3] = -np.tile(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], np.float16), 4)
    flat[4] = np.arange(32) * np.float16(2.0 ** -24)  # subnormals
    flat[5] = np.float16(65504)
    return x


def _paging(rng, batch, width, spare=3):
    perm = rng.permutation(batch * width + spare).astype(np.int32)
    return perm[: batch * width].reshape(batch, width), batch * width + spare


def test_oracle_quantiser_holds_fp16_exactly_on_its_grid():
    """What the codes stand for is always an fp16 value, and nearest to the input among the codes."""
    rng = np.random.default_rng(0)
    x = _values(rng, (64, 128))
    c, s = co.quantise(x)
    v = co.dequantise(c, s)
    assert np.array_equal(v, v.astype(np.float16).astype(np.float64))
    assert s[..., :4].min() >= 103
    step = np.ldexp(1.0, s.astype(np.int64) - 127).repeat(32, -1)
    # e2m1 steps are at most 2 below 6, and values above 6 (below 8) saturate
    assert np.all(np.abs(v - x.astype(np.float64)) <= np.where(np.abs(x) > 6 * step, 2 * step, step))


def test_wrapper_refusals_on_cpu_tensors():
    k = torch.zeros(2, 2, 64, dtype=torch.float16)
    caches = pad_b200.paged_kv_cache_fp4(4, 16, 2, 64, device="cpu")
    assert [tuple(c.shape) for c in caches] == [(4, 16, 2, 32), (4, 16, 2, 4)] * 2
    bt, pos = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError):
        pad_b200.paged_kv_append_fp4(k, k, *caches, bt, pos)
    with pytest.raises(AssertionError):
        pad_b200.paged_kv_read_fp4(*caches, bt, pos)
    with pytest.raises(AssertionError):
        pad_b200.paged_kv_cache_fp4(4, 16, 2, 48, device="cpu")


def _abi_append(**over):
    lib = _lib.load()
    p = 1 << 20
    kw = dict(kn=p, vn=p, k=p, ks=p, v=p, vs=p, bt=p, pos=p, ids=0, tokens=2, batch=2, hkv=2, d=128, pages=10, ps=16,
              maxp=4, kns=[256, 128, 1], vns=[256, 128, 1], kst=[2048, 128, 64, 1], kss=[128, 8, 4, 1],
              vst=[2048, 128, 64, 1], vss=[128, 8, 4, 1], bts=4)
    kw.update(over)
    a = lambda x: None if x is None else _lib.i64_array(x)  # noqa: E731
    return lib.pad_paged_kv_append_fp4(
        kw["kn"], kw["vn"], kw["k"], kw["ks"], kw["v"], kw["vs"], kw["bt"], kw["pos"], kw["ids"], kw["tokens"],
        kw["batch"], kw["hkv"], kw["d"], kw["pages"], kw["ps"], kw["maxp"], a(kw["kns"]), a(kw["vns"]), a(kw["kst"]),
        a(kw["kss"]), a(kw["vst"]), a(kw["vss"]), kw["bts"], 0, 0)


@pytest.mark.parametrize("over,status,text", [
    (dict(tokens=-1), _lib.PAD_ERR_INVALID_ARGUMENT, b"size"),
    (dict(ps=0), _lib.PAD_ERR_INVALID_ARGUMENT, b"size"),
    (dict(d=48), _lib.PAD_ERR_UNSUPPORTED, b"head_dim"),
    (dict(d=16), _lib.PAD_ERR_UNSUPPORTED, b"head_dim"),
    (dict(k=0), _lib.PAD_ERR_INVALID_ARGUMENT, b"null"),
    (dict(vst=None), _lib.PAD_ERR_INVALID_ARGUMENT, b"null"),
    (dict(tokens=3), _lib.PAD_ERR_INVALID_ARGUMENT, b"seq_ids"),
    (dict(bts=3), _lib.PAD_ERR_INVALID_ARGUMENT, b"stride"),
    (dict(kns=[256, 128, 2]), _lib.PAD_ERR_UNSUPPORTED, b"contiguous"),
    (dict(kst=[2048, 128, 65, 1]), _lib.PAD_ERR_UNSUPPORTED, b"16 bytes"),
    (dict(kss=[128, 8, 5, 1]), _lib.PAD_ERR_UNSUPPORTED, b"scale strides"),
    (dict(k=(1 << 20) + 8), _lib.PAD_ERR_UNSUPPORTED, b"aligned"),
    (dict(vs=(1 << 20) + 2), _lib.PAD_ERR_UNSUPPORTED, b"aligned"),
])
def test_append_refusals_without_a_device(over, status, text):
    assert _abi_append(**over) == status
    assert b"kv_append_fp4" in _lib.load().pad_last_error() and text in _lib.load().pad_last_error()


def test_append_of_nothing_is_ok_without_a_device():
    assert _abi_append(tokens=0) == _lib.PAD_OK
    assert _abi_append(batch=0, tokens=0) == _lib.PAD_OK


gpu = pytest.mark.gpu


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _expect(caches, k, v, bt, pos, ids, ps):
    """The four cache arrays after the append (numpy)."""
    kc, ks, vc, vs = [c.copy() for c in caches]
    for (c, s), x in (((kc, ks), k), ((vc, vs), v)):
        codes, scales = co.quantise(x)
        for t, (p, i) in enumerate(zip(pos, ids)):
            if p >= 0:
                c[bt[i, p // ps], p % ps] = codes[t]
                s[bt[i, p // ps], p % ps] = scales[t]
    return kc, ks, vc, vs


@gpu
@pytest.mark.parametrize("d,ps,hkv", [(128, 16, 2), (64, 16, 8), (32, 1, 3), (128, 24, 1), (64, 7, 5), (128, 256, 8)])
def test_append_and_read_bit_for_bit(d, ps, hkv):
    _need_cuda()
    rng = np.random.default_rng(d + ps)
    batch, width = 3, 200 // ps + 2
    bt, pages = _paging(rng, batch, width)
    tokens = [(i, p) for i in range(batch) for p in range(150) if rng.random() < 0.5]
    rng.shuffle(tokens)
    ids, pos = np.array([t[0] for t in tokens], np.int32), np.array([t[1] for t in tokens], np.int32)
    pos[5] = -1  # skipped
    k, v = _values(rng, (len(pos), hkv, d)), _values(rng, (len(pos), hkv, d))
    k[7, 0, 3], v[8, hkv - 1, d - 1], v[9, 0, 0] = np.inf, np.nan, -np.inf
    before = [np.full((pages, ps, hkv, n), 0xA5, np.uint8) for n in (d // 2, 4, d // 2, 4)]
    caches = [_cuda(c) for c in before]
    pad_b200.paged_kv_append_fp4(_cuda(k), _cuda(v), *caches, _cuda(bt), _cuda(pos), _cuda(ids))
    want = _expect(before, k, v, bt, pos, ids, ps)
    for got, ref in zip(caches, want):  # rows that no token names stay as they were
        np.testing.assert_array_equal(got.cpu().numpy(), ref)
    ko, vo = pad_b200.paged_kv_read_fp4(*caches, _cuda(bt), _cuda(pos), _cuda(ids))
    for got, x in ((ko, k), (vo, v)):
        ref = co.dequantise(*co.quantise(x))
        ref[5] = 0
        np.testing.assert_array_equal(got.cpu().numpy().astype(np.float64), ref)


@gpu
def test_one_token_of_each_sequence_without_seq_ids():
    _need_cuda()
    rng = np.random.default_rng(1)
    bt, pages = _paging(rng, 5, 4)
    pos = np.array([0, 63, 17, -1, 32], np.int64)  # int64 is cast, as for paged_kv_append
    k, v = _values(rng, (5, 2, 64)), _values(rng, (5, 2, 64))
    caches = list(pad_b200.paged_kv_cache_fp4(pages, 16, 2, 64))
    pad_b200.paged_kv_append_fp4(_cuda(k), _cuda(v), *caches, _cuda(bt.astype(np.int64)), _cuda(pos))
    want = _expect([np.zeros(c.shape, np.uint8) for c in caches], k, v, bt, pos, range(5), 16)
    for got, ref in zip(caches, want):
        np.testing.assert_array_equal(got.cpu().numpy(), ref)


@gpu
@pytest.mark.parametrize("kind", ["sliced", "unaligned", "head_major_cache", "inner_stride"])
def test_strides_and_alignment(kind):
    _need_cuda()
    rng = np.random.default_rng(2)
    d, ps, hkv, n = 64, 16, 3, 40
    bt, pages = _paging(rng, 1, 4)
    pos, ids = np.arange(n, dtype=np.int32), np.zeros(n, np.int32)
    k, v = _values(rng, (n, hkv, d)), _values(rng, (n, hkv, d))
    kt, vt = _cuda(k), _cuda(v)
    caches = list(pad_b200.paged_kv_cache_fp4(pages, ps, hkv, d))
    if kind == "sliced":  # rows of one fused projection
        both = torch.cat([kt, vt], 1)
        kt, vt = both[:, :hkv], both[:, hkv:]
    elif kind == "unaligned":
        flat = torch.zeros(kt.numel() + 1, dtype=torch.float16, device="cuda")
        flat[1:] = kt.flatten()
        kt = flat[1:].view(n, hkv, d)
    elif kind == "head_major_cache":
        caches = [c.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for c in caches]
    else:
        kt = kt.transpose(0, 2).contiguous().transpose(0, 2)
    pad_b200.paged_kv_append_fp4(kt, vt, *caches, _cuda(bt), _cuda(pos), _cuda(ids))
    want = _expect([np.zeros(c.shape, np.uint8) for c in caches], k, v, bt, pos, ids, ps)
    for got, ref in zip(caches, want):
        np.testing.assert_array_equal(got.cpu().numpy(), ref)
    ko, vo = pad_b200.paged_kv_read_fp4(*caches, _cuda(bt), _cuda(pos), _cuda(ids))
    np.testing.assert_array_equal(ko.cpu().numpy().astype(np.float64), co.dequantise(*co.quantise(k)))
    np.testing.assert_array_equal(vo.cpu().numpy().astype(np.float64), co.dequantise(*co.quantise(v)))


@gpu
def test_bad_pages_positions_and_sequences_are_flagged_and_not_written():
    _need_cuda()
    pad_b200.read_error_flags()
    k = torch.ones(4, 2, 32, dtype=torch.float16, device="cuda")
    bt = torch.tensor([[0, 7], [1, -1]], dtype=torch.int32, device="cuda")
    cases = [([16, 0], [0, 0], _lib.PAD_FLAG_BAD_PAGE_ID), ([16, 0], [1, 0], _lib.PAD_FLAG_BAD_PAGE_ID),
             ([32, 0], [0, 0], _lib.PAD_FLAG_SEQ_LEN_RANGE), ([0, 0], [2, 0], _lib.PAD_FLAG_BAD_SEQ_ID),
             ([0, 0], [-1, 0], _lib.PAD_FLAG_BAD_SEQ_ID), ([-1, 0], [9, 0], 0)]
    for pos, ids, flag in cases:
        caches = pad_b200.paged_kv_cache_fp4(2, 16, 2, 32)
        p, i = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (pos, ids))
        pad_b200.paged_kv_append_fp4(k[:2], k[:2], *caches, bt, p, i)
        assert pad_b200.read_error_flags() == flag
        written = caches[1].flatten(0, 1)[:, :, 0].ne(0).nonzero()[:, 0].unique().tolist()
        assert written == [0]  # the good token alone
        ko, vo = pad_b200.paged_kv_read_fp4(*caches, bt, p, i)
        assert pad_b200.read_error_flags() == flag
        assert ko[0].eq(0).all() and vo[0].eq(0).all() and ko[1].eq(1).all()


@gpu
def test_read_of_any_scale_byte():
    """Scale bytes that the append never writes read as what they stand for, rounded once to fp16."""
    _need_cuda()
    caches = pad_b200.paged_kv_cache_fp4(16, 16, 1, 32)
    scales = torch.arange(256, dtype=torch.uint8, device="cuda").view(16, 16, 1, 1)
    caches[1][..., :1] = scales
    caches[3][..., :1] = scales
    codes = torch.arange(256, device="cuda").to(torch.uint8).view(16, 16)
    caches[0][:] = codes.view(1, 16, 1, 16)[:, :, :, :]
    caches[2][:] = codes.view(1, 16, 1, 16)
    bt = torch.arange(16, dtype=torch.int32, device="cuda").view(1, 16)
    pos, ids = torch.arange(256, dtype=torch.int32, device="cuda"), torch.zeros(256, dtype=torch.int32, device="cuda")
    ko, _ = pad_b200.paged_kv_read_fp4(*caches, bt, pos, ids)
    with np.errstate(over="ignore"):
        ref = co.dequantise(caches[0].cpu().numpy(), caches[1].cpu().numpy()).reshape(256, 1, 32).astype(np.float16)
    np.testing.assert_array_equal(ko.cpu().numpy(), ref)


@gpu
def test_offsets_past_32_bits():
    _need_cuda()
    rng = np.random.default_rng(3)
    d, ps, hkv = 64, 2, 1
    big = torch.zeros((5 << 30,), dtype=torch.uint8, device="cuda")
    far = lambda off, n: big[off:].as_strided((2, ps, hkv, n), ((9 << 29), 64, 32, 1))  # noqa: E731
    caches = [far(0, d // 2), far(1 << 12, 4), far(1 << 13, d // 2), far(1 << 14, 4)]
    bt = np.array([[1, 0]], np.int32)
    pos, ids = np.arange(4, dtype=np.int32), np.zeros(4, np.int32)
    k, v = rng.standard_normal((4, 1, d)).astype(np.float16), rng.standard_normal((4, 1, d)).astype(np.float16)
    pad_b200.paged_kv_append_fp4(_cuda(k), _cuda(v), *caches, _cuda(bt), _cuda(pos), _cuda(ids))
    ko, vo = pad_b200.paged_kv_read_fp4(*caches, _cuda(bt), _cuda(pos), _cuda(ids))
    np.testing.assert_array_equal(ko.cpu().numpy().astype(np.float64), co.dequantise(*co.quantise(k)))
    np.testing.assert_array_equal(vo.cpu().numpy().astype(np.float64), co.dequantise(*co.quantise(v)))
    assert int(big[: 9 << 29].ne(0).sum()) > 0 and int(big[9 << 29:].ne(0).sum()) > 0


@gpu
def test_wrong_types_and_shapes_are_refused():
    _need_cuda()
    caches = pad_b200.paged_kv_cache_fp4(4, 16, 2, 64)
    k = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    bt, pos = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(AssertionError):
        pad_b200.paged_kv_append_fp4(k.float(), k, *caches, bt, pos)
    with pytest.raises(RuntimeError):
        pad_b200.paged_kv_append_fp4(k[:, :1], k[:, :1], *caches, bt, pos)
    with pytest.raises(RuntimeError):
        pad_b200.paged_kv_append_fp4(k, k, caches[0], caches[0], caches[2], caches[3], bt, pos)
    with pytest.raises(RuntimeError):
        pad_b200.paged_kv_append_fp4(k, k, *caches, bt, pos[:1])
    with pytest.raises(RuntimeError):
        pad_b200.paged_kv_read_fp4(caches[0].to(torch.int32), *caches[1:], bt, pos)
    with pytest.raises(AssertionError):
        pad_b200.paged_kv_append_fp4(k, k, *caches, bt[:1], pos)


@gpu
def test_append_and_read_in_a_graph_on_another_stream():
    _need_cuda()
    rng = np.random.default_rng(4)
    bt, pages = _paging(rng, 2, 4)
    btg = _cuda(bt)
    caches = pad_b200.paged_kv_cache_fp4(pages, 16, 2, 128)
    k = torch.zeros(2, 2, 128, dtype=torch.float16, device="cuda")
    v, pos = torch.zeros_like(k), torch.zeros(2, dtype=torch.int32, device="cuda")
    pad_b200.paged_kv_append_fp4(k, v, *caches, btg, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pad_b200.paged_kv_append_fp4(k, v, *caches, btg, pos)
        ko, vo = pad_b200.paged_kv_read_fp4(*caches, btg, pos)
    for step in range(3):
        x = rng.standard_normal((2, 2, 2, 128)).astype(np.float16)
        k.copy_(_cuda(x[0])), v.copy_(_cuda(x[1])), pos.copy_(_cuda(np.array([step, 30 + step], np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(ko.cpu().numpy().astype(np.float64), co.dequantise(*co.quantise(x[0])))
        np.testing.assert_array_equal(vo.cpu().numpy().astype(np.float64), co.dequantise(*co.quantise(x[1])))


@gpu
def test_a_pool_or_a_table_of_nothing():
    """Tokens that cannot have a place are flagged, as in any other pool; they read as zeros."""
    _need_cuda()
    pad_b200.read_error_flags()
    k = torch.ones(2, 2, 64, dtype=torch.float16, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    none, some = pad_b200.paged_kv_cache_fp4(0, 16, 2, 64), pad_b200.paged_kv_cache_fp4(3, 16, 2, 64)
    table = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    for caches, bt, flag in [(none, table, _lib.PAD_FLAG_BAD_PAGE_ID), (some, table[:, :0], _lib.PAD_FLAG_SEQ_LEN_RANGE),
                             (none, table[:, :0], _lib.PAD_FLAG_SEQ_LEN_RANGE)]:
        for pos, ids, want in [(i32(3, 0), None, flag), (i32(-1, -1), None, 0), (i32(0, 0), i32(1, 1), flag)]:
            pad_b200.paged_kv_append_fp4(k, k, *caches, bt, pos, ids)
            assert pad_b200.read_error_flags() == want
            for got in pad_b200.paged_kv_read_fp4(*caches, bt, pos, ids):
                assert got.shape == (2, 2, 64) and got.eq(0).all()
            assert pad_b200.read_error_flags() == want
    nobody = table[:0]
    pad_b200.paged_kv_append_fp4(k, k, *some, nobody, i32(0, 0), i32(0, 0))
    assert pad_b200.read_error_flags() == _lib.PAD_FLAG_BAD_SEQ_ID
    assert pad_b200.paged_kv_read_fp4(*some, nobody, i32(0, 0), i32(0, 0))[0].eq(0).all()
    assert pad_b200.read_error_flags() == _lib.PAD_FLAG_BAD_SEQ_ID
    assert all(c.eq(0).all() for c in some)
