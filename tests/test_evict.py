"""Eviction by accumulated attention weight: plans against a numpy ranking and
moves against numpy copies, all exact."""

import numpy as np
import pytest
import torch

import cache_oracle as co
import pad_b200
from pad_b200 import _lib


def _paging(rng, lens, ps, width=None, spare=2):
    need = [-(-int(n) // ps) for n in lens]
    width = max(max(need), 1) + 1 if width is None else width
    perm = rng.permutation(sum(need) + spare).astype(np.int32)
    bt = np.zeros((len(lens), width), np.int32)
    at = 0
    for i, n in enumerate(need):
        bt[i, :n] = perm[at:at + n]
        at += n
    return bt, sum(need) + spare


def _weights(rng, shape, kind):
    if kind == "tail":
        return (rng.random(shape) ** 8).astype(np.float32)
    if kind == "ties":
        return rng.integers(0, 3, shape).astype(np.float32)
    if kind == "equal":
        return np.zeros(shape, np.float32)
    w = rng.standard_normal(shape).astype(np.float32) * np.float32(1e-30)  # "odd": every kind of value
    pick = rng.integers(0, 12, shape)
    for i, x in enumerate([np.nan, np.inf, -np.inf, 0.0, -0.0, 3.4e38, -3.4e38, 1e-45]):
        w[pick == i] = x
    w[pick == 8] = -np.float32(np.nan)
    return w


def _plan_lists(src, dst, counts):
    src, dst, counts = src.cpu().numpy(), dst.cpu().numpy(), counts.cpu().numpy()
    ss, dd = {}, {}
    for i in range(src.shape[0]):
        for h in range(src.shape[1]):
            n = counts[i, h]
            assert 0 <= n <= src.shape[2]
            ss[i, h], dd[i, h] = src[i, h, :n].tolist(), dst[i, h, :n].tolist()
            assert (src[i, h, n:] == -1).all() and (dst[i, h, n:] == -1).all()
    return ss, dd


# ------------------------------------------------------------------ without a device
def _abi_plan(**over):
    lib = _lib.load()
    p = 1 << 20
    kw = dict(w=p, sp=0, bt=p, sl=p, tl=0, src=p, dst=p, cnt=p, nl=p, b=2, h=2, pages=10, ps=16, maxp=4, budget=10,
              recent=0, ws=[32, 16, 1], ps_=[32, 16, 1], bts=4)
    kw.update(over)
    a = lambda x: None if x is None else _lib.i64_array(x)  # noqa: E731
    return lib.pad_paged_kv_evict_plan(kw["w"], kw["sp"], kw["bt"], kw["sl"], kw["tl"], kw["src"], kw["dst"], kw["cnt"],
                                       kw["nl"], kw["b"], kw["h"], kw["pages"], kw["ps"], kw["maxp"], kw["budget"],
                                       kw["recent"], a(kw["ws"]), a(kw["ps_"]), kw["bts"], 0, 0)


@pytest.mark.parametrize("over,status,text", [
    (dict(b=-1), _lib.PAD_ERR_INVALID_ARGUMENT, b"size"),
    (dict(budget=0), _lib.PAD_ERR_INVALID_ARGUMENT, b"budget"),
    (dict(recent=11), _lib.PAD_ERR_INVALID_ARGUMENT, b"recent"),
    (dict(recent=1), _lib.PAD_ERR_INVALID_ARGUMENT, b"slot_positions"),
    (dict(w=0), _lib.PAD_ERR_INVALID_ARGUMENT, b"null"),
    (dict(sp=1 << 20, tl=0), _lib.PAD_ERR_INVALID_ARGUMENT, b"null"),
    (dict(bts=3), _lib.PAD_ERR_INVALID_ARGUMENT, b"stride"),
    (dict(ps=1 << 29, maxp=4), _lib.PAD_ERR_UNSUPPORTED, b"32-bit"),
])
def test_plan_refusals_without_a_device(over, status, text):
    assert _abi_plan(**over) == status
    assert b"evict_plan" in _lib.load().pad_last_error() and text in _lib.load().pad_last_error()


def test_max_moves_and_empty_batch():
    lib = _lib.load()
    got = _lib.ctypes.c_int64(-1)
    for budget, ps, maxp, want in [(10, 16, 4, 10), (60, 16, 4, 4), (64, 16, 4, 0), (100, 16, 4, 0), (1, 1, 1, 0)]:
        assert lib.pad_evict_max_moves(budget, ps, maxp, _lib.ctypes.byref(got)) == _lib.PAD_OK
        assert got.value == want
    assert lib.pad_evict_max_moves(0, 16, 4, _lib.ctypes.byref(got)) == _lib.PAD_ERR_INVALID_ARGUMENT
    assert _abi_plan(b=0) == _lib.PAD_OK


def test_wrapper_refusals_on_cpu_tensors():
    w = torch.zeros(4, 2, 16)
    bt, sl = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(AssertionError):
        pad_b200.paged_kv_evict_plan(w, bt, sl, 10)
    with pytest.raises(AssertionError):
        pad_b200.paged_kv_move([w], bt, sl, sl, sl)


def _abi_move(**over):
    lib = _lib.load()
    p = 1 << 20
    kw = dict(n=1, c=[p], rb=[64], cs=[2048, 128, 64], bt=p, src=p, dst=p, cnt=p, b=2, h=2, pages=10, ps=16, maxp=4,
              moves=5, bts=4)
    kw.update(over)
    arr = (_lib.ctypes.c_void_p * len(kw["c"]))(*kw["c"])
    return lib.pad_paged_kv_move(kw["n"], arr, _lib.i64_array(kw["rb"]), _lib.i64_array(kw["cs"]), kw["bt"], kw["src"],
                                 kw["dst"], kw["cnt"], 0, 0, kw["b"], kw["h"], kw["pages"], kw["ps"], kw["maxp"],
                                 kw["moves"], None, None, kw["bts"], 0, 0)


@pytest.mark.parametrize("over,text", [
    (dict(n=0), b"caches"), (dict(n=5), b"caches"), (dict(c=[0]), b"null"), (dict(rb=[0]), b"row"),
    (dict(moves=-1), b"size"), (dict(src=0), b"null"), (dict(bts=1), b"stride")])
def test_move_refusals_without_a_device(over, text):
    assert _abi_move(**over) == _lib.PAD_ERR_INVALID_ARGUMENT
    assert text in _lib.load().pad_last_error()
    assert _abi_move(moves=0) == _lib.PAD_OK


# ------------------------------------------------------------------ on the GPU
gpu = pytest.mark.gpu


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


PLAN_CASES = [
    # lens, budget, recent, page size, heads, kind, table width
    ([0, 1, 40, 41, 64, 500], 40, 0, 16, 2, "tail", None),
    ([500, 333], 1, 0, 16, 3, "ties", None),
    ([500, 333], 332, 5, 7, 1, "ties", None),
    ([130], 129, 129, 1, 2, "equal", None),
    ([1024, 1025, 1023], 1024, 64, 32, 2, "odd", None),
    ([777, 2000], 300, 0, 24, 5, "odd", None),
    ([2000, 60, 1999], 512, 100, 16, 2, "equal", 4096),      # a table far wider than the sequences (clusters)
    ([8192, 8193, 16385], 4096, 128, 16, 1, "tail", None),   # up to a cluster of 4
    ([9000, 3], 8990, 2, 8, 2, "odd", None),                 # a cluster of 2
    ([70001], 9999, 200, 64, 2, "ties", None),               # a cluster of 8
    ([70000, 69999], 1, 0, 16, 1, "equal", None),
    ([450000], 100000, 0, 64, 1, "odd", None),               # more keys than the cluster's shared memory
]


@gpu
@pytest.mark.parametrize("lens,budget,recent,ps,hkv,kind,width", PLAN_CASES)
def test_plan_matches_ranking(lens, budget, recent, ps, hkv, kind, width):
    _need_cuda()
    pad_b200.read_error_flags()
    rng = np.random.default_rng(budget + ps)
    bt, pages = _paging(rng, lens, ps, width)
    w = _weights(rng, (pages, hkv, ps), kind)
    at = rng.integers(0, max(lens) + 50, (pages, hkv, ps)).astype(np.int32)
    total = np.asarray(lens) + 50
    src, dst, counts, new = pad_b200.paged_kv_evict_plan(
        _cuda(w), _cuda(bt), _cuda(np.asarray(lens, np.int64)), budget, recent,
        slot_positions=_cuda(at) if recent else None, total_lens=_cuda(total) if recent else None)
    ss, dd, want_new = co.evict_plan(w, bt, lens, budget, recent, at, total)
    assert new.cpu().tolist() == want_new.tolist()
    got_s, got_d = _plan_lists(src, dst, counts)
    assert got_s == ss and got_d == dd
    assert pad_b200.read_error_flags() == 0


@gpu
def test_plan_strides_and_repeatability():
    _need_cuda()
    rng = np.random.default_rng(9)
    lens, ps, hkv = [300, 290], 16, 4
    bt, pages = _paging(rng, lens, ps)
    w = _weights(rng, (pages, hkv, ps), "ties")
    wt = _cuda(w.transpose(2, 0, 1)).permute(1, 2, 0)  # row-major last
    btw = torch.zeros(2, bt.shape[1] + 5, dtype=torch.int32, device="cuda")
    btw[:, : bt.shape[1]] = _cuda(bt)
    at = rng.integers(0, 400, (pages, hkv, ps)).astype(np.int32)
    atw = torch.zeros(pages, 2 * hkv, ps, dtype=torch.int32, device="cuda")
    atw[:, ::2] = _cuda(at)  # every other head of a wider array
    ss, dd, _ = co.evict_plan(w, bt, lens, 100, 30, at, lens)
    for _ in range(3):
        got = pad_b200.paged_kv_evict_plan(wt, btw[:, : bt.shape[1]], _cuda(np.array(lens, np.int32)), 100, 30,
                                           slot_positions=atw[:, ::2])
        assert _plan_lists(*got[:3]) == (ss, dd)


@gpu
def test_plan_flags_bad_pages_and_lengths():
    _need_cuda()
    pad_b200.read_error_flags()
    w = torch.rand(4, 1, 16, device="cuda")
    bt = torch.tensor([[0, 1, 9]], dtype=torch.int32, device="cuda")
    src, dst, counts, new = pad_b200.paged_kv_evict_plan(w, bt, torch.tensor([40], device="cuda"), 8)
    assert pad_b200.read_error_flags() == _lib.PAD_FLAG_BAD_PAGE_ID
    assert src.max() < 32  # slots of a bad page weigh nothing
    pad_b200.paged_kv_evict_plan(w, bt[:, :2], torch.tensor([33], device="cuda"), 8)
    assert pad_b200.read_error_flags() == _lib.PAD_FLAG_SEQ_LEN_RANGE
    _, _, counts, new = pad_b200.paged_kv_evict_plan(w, bt[:, :2], torch.tensor([-1], device="cuda"), 8)
    assert pad_b200.read_error_flags() == _lib.PAD_FLAG_SEQ_LEN_RANGE
    assert new.item() == 0 and counts.item() == 0


MOVE_ROWS = [("fp16", [(torch.float16, 128)] * 2), ("fp4", [(torch.uint8, 64), (torch.uint8, 4)] * 2),
             ("long", [(torch.float32, 256)]), ("odd", [(torch.uint8, 7), (torch.float16, 3), (torch.float32, 5)]),
             ("small", [(torch.float16, 16), (torch.uint8, 1)])]


@gpu
@pytest.mark.parametrize("name,rows", MOVE_ROWS, ids=[r[0] for r in MOVE_ROWS])
@pytest.mark.parametrize("tracked", [True, False])
def test_moves_and_evict(name, rows, tracked):
    _need_cuda()
    pad_b200.read_error_flags()
    rng = np.random.default_rng(len(rows))
    lens, ps, hkv, budget, recent = [700, 90, 333, 0], 24, 3, 100, 10
    bt, pages = _paging(rng, lens, ps)
    w = _weights(rng, (pages, hkv, ps), "tail")
    at = np.zeros((pages, hkv, ps), np.int32)
    for i, n in enumerate(lens):
        for t in range(n):
            at[bt[i, t // ps], :, t % ps] = t
    caches = [torch.randint(0, 100, (pages, ps, hkv, n), device="cuda").to(dt) for dt, n in rows]
    before = [c.cpu().numpy() for c in caches]
    ss, dd, new = co.evict_plan(w, bt, lens, budget, recent if tracked else 0, at, lens)
    wg, atg, sl = _cuda(w), _cuda(at), _cuda(np.array(lens, np.int32))
    if tracked:
        got = pad_b200.paged_kv_evict(caches, wg, _cuda(bt), sl, budget, recent, slot_positions=atg, total_lens=sl)
    else:
        src, dst, counts, got = pad_b200.paged_kv_evict_plan(wg, _cuda(bt), sl, budget)
        pad_b200.paged_kv_move(caches, _cuda(bt), src, dst, counts)
    assert got.tolist() == new.tolist()
    for c, x in zip(caches, before):  # everything that no move names stays as it was
        np.testing.assert_array_equal(c.cpu().numpy(), co.apply_moves(x, bt, ss, dd))
    if tracked:
        np.testing.assert_array_equal(wg.cpu().numpy(), co.apply_moves(w, bt, ss, dd, 1))
        np.testing.assert_array_equal(atg.cpu().numpy(), co.apply_moves(at, bt, ss, dd, 1))
    else:
        np.testing.assert_array_equal(wg.cpu().numpy(), w)
    assert pad_b200.read_error_flags() == 0


@gpu
def test_moves_of_bad_entries_are_flagged_and_skipped():
    _need_cuda()
    pad_b200.read_error_flags()
    cache = torch.arange(4 * 16 * 1 * 8, device="cuda", dtype=torch.float16).view(4, 16, 1, 8)
    was = cache.clone()
    bt = torch.tensor([[0, 1, 9]], dtype=torch.int32, device="cuda")
    lists = lambda x: torch.tensor([[x]], dtype=torch.int32, device="cuda")  # noqa: E731
    for src, dst, flag in [([48], [0], _lib.PAD_FLAG_SEQ_LEN_RANGE), ([20], [-1], _lib.PAD_FLAG_SEQ_LEN_RANGE),
                           ([40], [0], _lib.PAD_FLAG_BAD_PAGE_ID), ([20], [33], _lib.PAD_FLAG_BAD_PAGE_ID)]:
        pad_b200.paged_kv_move([cache], bt, lists(src), lists(dst), lists(1).view(1, 1))
        assert pad_b200.read_error_flags() == flag and torch.equal(cache, was)
    # a count past the list is cut to it
    pad_b200.paged_kv_move([cache], bt, lists([20]), lists([3]), lists(9).view(1, 1))
    was[0, 3] = was[1, 4]
    assert torch.equal(cache, was) and pad_b200.read_error_flags() == 0


@gpu
def test_move_refusals_and_unaligned_views():
    _need_cuda()
    cache = torch.zeros(4, 16, 2, 8, device="cuda")
    bt = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    lists, counts = torch.zeros(1, 2, 3, dtype=torch.int32, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError):
        pad_b200.paged_kv_move([cache] * 5, bt, lists, lists, counts)
    with pytest.raises(RuntimeError):
        pad_b200.paged_kv_move([cache, cache[:, :8]], bt, lists, lists, counts)
    with pytest.raises(RuntimeError):
        pad_b200.paged_kv_move([cache], bt, lists.long(), lists, counts)
    with pytest.raises(RuntimeError):
        pad_b200.paged_kv_move([cache], bt, lists, lists, counts, weights=cache)
    with pytest.raises(RuntimeError):
        pad_b200.paged_kv_evict_plan(torch.zeros(4, 2, 16, device="cuda"), bt, counts[0], 4)  # seq_lens of 2, table of 1
    odd = torch.arange(4 * 16 * 2 * 9 + 1, device="cuda", dtype=torch.float16)[1:].view(4, 16, 2, 9)[..., :8]
    src, dst = lists.clone(), lists.clone()
    src[0, :, 0], dst[0, :, 0] = 50, 2
    counts[:] = 1
    want = odd.clone()
    btg = torch.tensor([[3, 2, 1, 0]], dtype=torch.int32, device="cuda")
    want[3, 2] = odd[0, 2]
    pad_b200.paged_kv_move([odd], btg, src, dst, counts)
    assert torch.equal(odd, want)


@gpu
def test_evict_in_a_graph_replayed_on_new_contents():
    _need_cuda()
    rng = np.random.default_rng(11)
    lens, ps, hkv, budget = [300, 120], 16, 2, 100
    bt, pages = _paging(rng, lens, ps)
    btg, sl = _cuda(bt), _cuda(np.array(lens, np.int32))
    w = torch.zeros(pages, hkv, ps, device="cuda")
    cache = torch.zeros(pages, ps, hkv, 64, dtype=torch.float16, device="cuda")
    pad_b200.paged_kv_evict([cache], w, btg, sl, budget)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = pad_b200.paged_kv_evict([cache], w, btg, sl, budget)
    for _ in range(3):
        wn = _weights(rng, (pages, hkv, ps), "ties")
        cn = rng.standard_normal((pages, ps, hkv, 64)).astype(np.float16)
        w.copy_(_cuda(wn)), cache.copy_(_cuda(cn))
        graph.replay()
        torch.cuda.synchronize()
        ss, dd, want = co.evict_plan(wn, bt, lens, budget)
        assert new.tolist() == want.tolist()
        np.testing.assert_array_equal(cache.cpu().numpy(), co.apply_moves(cn, bt, ss, dd))
        np.testing.assert_array_equal(w.cpu().numpy(), co.apply_moves(wn, bt, ss, dd, 1))


@gpu
def test_plan_and_evict_of_an_empty_pool():
    _need_cuda()
    pad_b200.read_error_flags()
    w, at = torch.zeros(0, 2, 16, device="cuda"), torch.zeros(0, 2, 16, dtype=torch.int32, device="cuda")
    bt, sl = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for kw in ({}, dict(recent=2, slot_positions=at, total_lens=sl)):
        src, dst, counts, lens = pad_b200.paged_kv_evict_plan(w, bt, sl, 8, **kw)
        assert src.eq(-1).all() and dst.eq(-1).all() and counts.eq(0).all() and lens.eq(0).all()
        cache = torch.zeros(0, 16, 2, 64, dtype=torch.float16, device="cuda")
        assert pad_b200.paged_kv_evict([cache], w, bt, sl, 8, **kw).eq(0).all()
    assert pad_b200.read_error_flags() == 0
    # sequences that claim slots of a pool without pages are flagged
    src, dst, counts, lens = pad_b200.paged_kv_evict_plan(w, bt, sl + 40, 8)
    assert pad_b200.read_error_flags() == _lib.PAD_FLAG_BAD_PAGE_ID and lens.eq(8).all()


@gpu
def test_shared_pages_and_unsound_moves_are_refused_when_asked_for(monkeypatch):
    """PAD_B200_CHECK: nothing is written where two sequences name a page, or a move's target is named twice."""
    _need_cuda()
    from pad_b200 import kernel_cuda_v4

    monkeypatch.setattr(kernel_cuda_v4, "_CHECK_VALUES", True)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pages, ps, hkv, d = 50, 16, 2, 64  # a pool far larger than the batch: no flag tells
    q = torch.randn(3, 4, d, device="cuda").half()
    k = torch.randn(pages, ps, hkv, d, device="cuda").half()
    fp4 = pad_b200.paged_kv_cache_fp4(pages, ps, hkv, d)
    w = torch.rand(pages, hkv, ps, device="cuda")
    was, k_was = w.clone(), k.clone()
    calls = [lambda bt, n: pad_b200.paged_attention_decode_weights(q, k, k, bt, n, w),
             lambda bt, n: pad_b200.paged_attention_decode_fp4(q, *fp4, bt, n, weights=w),
             lambda bt, n: pad_b200.paged_kv_evict_plan(w, bt, n, 20),
             lambda bt, n: pad_b200.paged_kv_evict([k], w, bt, n, 20)]
    shared = [([[0, 1, 2], [0, 3, 4], [5, 6, 7]], [40, 40, 40]),  # a common first page
              ([[0, 1, 2], [3, 4, 5], [6, 7, 6]], [40, 40, 33]),  # one sequence names a page twice
              ([[0, 1, 2], [3, 4, 5], [6, 7, 2]], [33, 48, 40])]
    for bt, n in shared:
        for call in calls:
            with pytest.raises(ValueError, match="share pages"):
                call(i32(bt), torch.tensor(n, device="cuda"))
    assert torch.equal(w, was) and torch.equal(k, k_was)
    # ids behind the sequences, of empty ones and of none are no sharing; the decode without weights may share
    for bt, n in [([[0, 1, 2], [3, 4, 2], [0, 0, 0]], [40, 32, 0]), ([[0, 1, 1], [3, 4, 5], [6, 6, 6]], [17, 48, 16])]:
        for call in calls:
            call(i32(bt), torch.tensor(n, device="cuda"))
    pad_b200.paged_attention_decode_fp4(q, *fp4, i32(shared[0][0]), i32(shared[0][1]))
    # moves given by hand
    bt, cache = i32([[0, 1, 2], [3, 4, 0]]), torch.arange(pages * ps * 8, device="cuda").view(pages, ps, 1, 8)
    was = cache.clone()
    lists = lambda a, b: torch.tensor([[a], [b]], dtype=torch.int32, device="cuda")  # noqa: E731
    for src, dst, n in [(lists([40, 41], [40, 41]), lists([3, 3], [1, 2]), [2, 0]),        # a target twice
                        (lists([40, 20], [40, 41]), lists([20, 3], [1, 2]), [2, 0]),       # a target that is a source
                        (lists([40, 41], [20, 21]), lists([5, 6], [37, 38]), [2, 2]),      # by way of page 0
                        (lists([40, 41], [37, 21]), lists([5, 6], [2, 3]), [2, 1])]:
        with pytest.raises(ValueError, match="target"):
            pad_b200.paged_kv_move([cache], bt, src, dst, i32(n).view(2, 1))
    assert torch.equal(cache, was)
    pad_b200.paged_kv_move([cache], bt, lists([40, 41], [20, 21]), lists([5, 5], [2, 3]), i32([1, 2]).view(2, 1))
    for (p, r), (p2, r2) in {(0, 5): (2, 8), (3, 2): (4, 4), (3, 3): (4, 5)}.items():
        was[p, r] = was[p2, r2]
    assert torch.equal(cache, was)
