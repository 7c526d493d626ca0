"""The operators that keep a cache small, run together as a serving loop runs
them: prompt in, then steps of append, decode with weights, and eviction once a
sequence is over its budget -- on the fp16 and on the 4-bit cache, eagerly and as
one captured graph."""

import numpy as np
import pytest
import torch

import cache_oracle as co
import pad_b200
from gpu_utils import assert_parity
from test_decode_weights import check_weights, rel_bound, smax_of
from test_decode_weights import by_sequence

gpu = pytest.mark.gpu


def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


class Loop:
    """A batch's cache and the steps of its decoding loop."""

    def __init__(self, fp4, prompts, budget, recent, hkv=2, g=4, d=64, ps=16, seed=0):
        self.fp4, self.budget, self.recent, self.hkv, self.g, self.d, self.ps = fp4, budget, recent, hkv, g, d, ps
        self.b = len(prompts)
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.rand = lambda *s: torch.randn(*s, device="cuda", generator=gen).half()
        width = -(-(max(max(prompts), budget) + 40) // ps)
        self.pages = self.b * width
        perm = torch.randperm(self.pages, device="cuda", generator=gen).to(torch.int32)
        self.bt = perm.view(self.b, width)
        if fp4:
            self.caches = list(pad_b200.paged_kv_cache_fp4(self.pages, ps, hkv, d))
        else:
            self.caches = [torch.zeros(self.pages, ps, hkv, d, dtype=torch.float16, device="cuda") for _ in range(2)]
        self.w = torch.full((self.pages, hkv, ps), 9.0, device="cuda")  # left by former owners of the pages
        self.at = torch.full((self.pages, hkv, ps), 10 ** 6, dtype=torch.int32, device="cuda")
        self.lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
        self.total = self.lens.clone()
        ids = torch.repeat_interleave(torch.arange(self.b, device="cuda"), self.lens).to(torch.int32)
        pos = torch.cat([torch.arange(n, device="cuda") for n in prompts]).to(torch.int32)
        k, v = self.rand(len(ids), hkv, d), self.rand(len(ids), hkv, d)
        if fp4:
            pad_b200.paged_kv_append_fp4(k, v, *self.caches, self.bt, pos, ids)
        else:
            page, row = self.bt[ids.long(), pos.long() // ps].long(), pos.long() % ps
            self.caches[0][page, row], self.caches[1][page, row] = k, v

    def append(self, k, v):
        if self.fp4:
            pad_b200.paged_kv_append_fp4(k, v, *self.caches, self.bt, self.lens)
        else:
            pad_b200.paged_kv_append(k, v, *self.caches, self.bt, self.lens)
        self.lens.add_(1)
        self.total.add_(1)

    def decode(self, q, num_new):
        f = pad_b200.paged_attention_decode_fp4 if self.fp4 else pad_b200.paged_attention_decode_weights
        kw = dict(num_new=num_new, slot_positions=self.at, total_lens=self.total)
        if self.fp4:
            return f(q, *self.caches, self.bt, self.lens, weights=self.w, **kw)
        return f(q, *self.caches, self.bt, self.lens, self.w, **kw)

    def evict(self):
        self.lens.copy_(pad_b200.paged_kv_evict(self.caches, self.w, self.bt, self.lens, self.budget, self.recent,
                                                slot_positions=self.at, total_lens=self.total))

    def values(self):
        c = [x.cpu().numpy() for x in self.caches]
        if self.fp4:
            return co.dequantise(c[0], c[1]), co.dequantise(c[2], c[3])
        return c[0].astype(np.float64), c[1].astype(np.float64)


@gpu
@pytest.mark.parametrize("fp4", [False, True])
def test_every_step_against_float64(fp4):
    """Each step is checked on the state the GPU itself left, so that no near-tie of two weights decides the test."""
    _need_cuda()
    pad_b200.read_error_flags()
    prompts = [150, 40, 97, 1]
    lp = Loop(fp4, prompts, budget=64, recent=8, seed=int(fp4))
    bt = lp.bt.cpu().numpy()
    for step in range(12):
        k, v, q = lp.rand(lp.b, lp.hkv, lp.d), lp.rand(lp.b, lp.hkv, lp.d), lp.rand(lp.b, lp.hkv * lp.g, lp.d)
        num_new = 10 ** 6 if step == 0 else 1  # the first step takes the prompts' weights and positions too
        lp.append(k, v)
        w0, at0 = lp.w.cpu().numpy(), lp.at.cpu().numpy()
        out = lp.decode(q, num_new)
        lens, total = lp.lens.cpu().numpy(), lp.total.cpu().numpy()
        kk, vv = lp.values()
        ref, probs = co.decode(q.cpu().numpy(), kk, vv, bt, lens)
        assert_parity(out.float().cpu().numpy(), ref, f"step {step}")
        w1, at1 = lp.w.cpu().numpy(), lp.at.cpu().numpy()
        check_weights(w1, co.accumulate(w0, probs, bt, lens, num_new), rel_bound(lp.d, int(lens.max()), smax_of(q.cpu().numpy().astype(np.float64), kk, lp.d)))
        for i, n in enumerate(lens):
            for t in range(max(0, n - num_new), n):
                at0[bt[i, t // lp.ps], :, t % lp.ps] = total[i] - n + t
        np.testing.assert_array_equal(at1, at0)
        before = [c.cpu().numpy() for c in lp.caches]
        lp.evict()
        ss, dd, new = co.evict_plan(w1, bt, lens, lp.budget, lp.recent, at1, total)
        assert lp.lens.cpu().tolist() == new.tolist()
        for c, x in zip(lp.caches, before):
            np.testing.assert_array_equal(c.cpu().numpy(), co.apply_moves(x, bt, ss, dd))
        np.testing.assert_array_equal(lp.w.cpu().numpy(), co.apply_moves(w1, bt, ss, dd, 1))
        at2 = lp.at.cpu().numpy()
        np.testing.assert_array_equal(at2, co.apply_moves(at1, bt, ss, dd, 1))
        for i, n in enumerate(new):  # what is kept: distinct positions, the recent ones among them
            t = np.arange(n)
            for h in range(lp.hkv):
                kept = at2[bt[i, t // lp.ps], h, t % lp.ps]
                assert len(set(kept.tolist())) == n and kept.max() == total[i] - 1
                assert set(range(max(0, total[i] - lp.recent), total[i])) <= set(kept.tolist())
    assert lp.lens.cpu().tolist() == [64, 52, 64, 13]
    assert pad_b200.read_error_flags() == 0


@gpu
@pytest.mark.parametrize("fp4", [False, True])
def test_a_captured_step_equals_the_eager_loop(fp4):
    _need_cuda()
    prompts = [70, 33, 64]
    eager, replayed = (Loop(fp4, prompts, budget=64, recent=4, seed=7) for _ in range(2))
    k, v, q = (torch.zeros(3, h, 64, dtype=torch.float16, device="cuda") for h in (2, 2, 8))

    def step(loop):
        loop.append(k, v)
        out = loop.decode(q, 1)
        loop.evict()
        return out

    steps = [(eager.rand(3, 2, 64), eager.rand(3, 2, 64), eager.rand(3, 8, 64)) for _ in range(6)]
    for lp in (eager, replayed):  # the prompts' weights and positions; also warms up what the capture uses
        q.copy_(steps[0][2])
        lp.decode(q, 10 ** 6)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(replayed)
    for a, b, c in steps:
        k.copy_(a), v.copy_(b), q.copy_(c)
        want = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        for x, y in zip([*eager.caches, eager.w, eager.at, eager.lens], [*replayed.caches, replayed.w, replayed.at, replayed.lens]):
            assert torch.equal(x, y)


@gpu
def test_without_eviction_the_weights_are_those_of_all_steps():
    """A budget nothing reaches: weights and positions add up as if written out, and both caches' loops agree with it."""
    _need_cuda()
    lp = Loop(False, [30, 5], budget=100, recent=0, seed=3)
    want = np.zeros((2, 2, 40))
    bt = lp.bt.cpu().numpy()
    worst = 0.0
    for s in range(5):
        k, v, q = lp.rand(2, 2, 64), lp.rand(2, 2, 64), lp.rand(2, 8, 64)
        lp.append(k, v)
        lp.decode(q, 10 ** 6 if s == 0 else 1)
        lp.evict()
        kk, vv = lp.values()
        _, probs = co.decode(q.cpu().numpy(), kk, vv, bt, lp.lens.cpu().numpy())
        worst = max(worst, smax_of(q.cpu().numpy().astype(np.float64), kk, 64))
        for i, p in enumerate(probs):
            want[i, :, : len(p)] += p.T
    w = lp.w.cpu().numpy()
    for i, n in enumerate([35, 10]):
        t = np.arange(n)
        got = w[bt[i, t // 16], :, t % 16].T
        # five additions round by 2^-24 each, on top of each probability's own bound
        assert np.all(np.abs(got - want[i, :, :n]) <= (rel_bound(64, 35, worst) + 5 * 2.0 ** -24) * want[i, :, :n] + 1e-7)
    assert lp.lens.cpu().tolist() == [35, 10]


@gpu
@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("captured", [False, True])
def test_a_sequence_joins_the_others_with_its_prompt(fp4, captured):
    """Sequence 2 is empty for three steps, then has a prompt of 90 tokens on pages that others have used, and is
    evicted by the weights and positions of this step's decode; the others add one token a step all along."""
    _need_cuda()
    pad_b200.read_error_flags()
    lp = Loop(fp4, [70, 33, 0], budget=64, recent=4, seed=9)
    bt = lp.bt.cpu().numpy()
    k, v, q = lp.rand(3, lp.hkv, lp.d), lp.rand(3, lp.hkv, lp.d), lp.rand(3, lp.hkv * lp.g, lp.d)
    news = torch.zeros(3, dtype=torch.int32, device="cuda")
    q.copy_(lp.rand(*q.shape))
    lp.decode(q, 10 ** 6)  # the first prompts' weights and positions
    graph = None
    for step in range(6):
        if step == 3:  # the prompt, all but its last token, which this step appends
            pk, pv = lp.rand(89, lp.hkv, lp.d), lp.rand(89, lp.hkv, lp.d)
            pos = torch.arange(89, dtype=torch.int32, device="cuda")
            if fp4:
                pad_b200.paged_kv_append_fp4(pk, pv, *lp.caches, lp.bt, pos, torch.full_like(pos, 2))
            else:
                page, row = lp.bt[2, pos.long() // lp.ps].long(), pos.long() % lp.ps
                lp.caches[0][page, row], lp.caches[1][page, row] = pk, pv
            lp.lens[2] = lp.total[2] = 89
        live = [0, 1] if step < 3 else [0, 1, 2]
        news.copy_(torch.tensor([1, 1, 0 if step < 3 else 90 if step == 3 else 1]))
        k.copy_(lp.rand(*k.shape)), v.copy_(lp.rand(*v.shape)), q.copy_(lp.rand(*q.shape))
        f, kw = (pad_b200.paged_attention_decode_fp4, dict(weights=lp.w)) if fp4 else (pad_b200.paged_attention_decode_weights, {})

        def decode():
            args = (q, *lp.caches, lp.bt, lp.lens) + (() if fp4 else (lp.w,))
            return f(*args, num_new=news, slot_positions=lp.at, total_lens=lp.total, **kw)

        lens = lp.lens.clone()
        lens[2] = -1 if step < 3 else lens[2]  # (a position below 0 appends nothing)
        (pad_b200.paged_kv_append_fp4 if fp4 else pad_b200.paged_kv_append)(k, v, *lp.caches, lp.bt, lens)
        lp.lens[live] += 1
        lp.total[live] += 1
        w0, at0 = lp.w.cpu().numpy(), lp.at.cpu().numpy()
        if not captured:
            out = decode()
            lp.evict_lens = pad_b200.paged_kv_evict_plan(lp.w, lp.bt, lp.lens, lp.budget, lp.recent, slot_positions=lp.at,
                                                         total_lens=lp.total)
        else:
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    out = decode()
                    lp.evict_lens = pad_b200.paged_kv_evict_plan(lp.w, lp.bt, lp.lens, lp.budget, lp.recent,
                                                                 slot_positions=lp.at, total_lens=lp.total)
            graph.replay()
        torch.cuda.synchronize()
        seqs, total = lp.lens.tolist(), lp.total.cpu().numpy()
        kk, vv = lp.values()
        ref, probs = co.decode(q.cpu().numpy(), kk, vv, bt, seqs)
        assert_parity(out.float().cpu().numpy(), ref, f"step {step}")
        w1, at1 = lp.w.cpu().numpy(), lp.at.cpu().numpy()
        want_w, want_at = by_sequence(w0, at0, probs, bt, seqs, total, news.tolist())
        check_weights(w1, want_w, rel_bound(lp.d, max(seqs), smax_of(q.cpu().numpy().astype(np.float64), kk, lp.d)))
        np.testing.assert_array_equal(at1, want_at)
        src, dst, counts, new = lp.evict_lens
        ss, dd, want_new = co.evict_plan(w1, bt, seqs, lp.budget, lp.recent, at1, total)
        assert new.tolist() == want_new.tolist()
        for (i, h), x in ss.items():
            n = int(counts[i, h])
            assert src[i, h, :n].tolist() == x and dst[i, h, :n].tolist() == dd[i, h]
        pad_b200.paged_kv_move(lp.caches, lp.bt, src, dst, counts, weights=lp.w, slot_positions=lp.at)
        lp.lens.copy_(new)
        if step == 3:  # the newcomer keeps its own last tokens
            at2 = lp.at.cpu().numpy()
            t = np.arange(64)
            for h in range(lp.hkv):
                assert {86, 87, 88, 89} <= set(at2[bt[2, t // lp.ps], h, t % lp.ps].tolist())
    assert lp.lens.tolist() == [64, 39, 64]
    assert pad_b200.read_error_flags() == 0


@gpu
@pytest.mark.parametrize("fp4", [False, True])
def test_lengths_left_out_after_an_eviction_are_refused_when_asked_for(fp4, monkeypatch):
    """total_lens may be left out until a first eviction; afterwards positions would be given twice and the window of
    recent tokens be too wide."""
    _need_cuda()
    from pad_b200 import kernel_cuda_v4

    monkeypatch.setattr(kernel_cuda_v4, "_CHECK_VALUES", True)
    lp = Loop(fp4, [100, 20], budget=64, recent=8, seed=4)
    q = lp.rand(2, lp.hkv * lp.g, lp.d)
    decode = lambda new, **kw: (pad_b200.paged_attention_decode_fp4(  # noqa: E731
        q, *lp.caches, lp.bt, lp.lens, weights=lp.w, num_new=new, slot_positions=lp.at, **kw) if fp4 else
        pad_b200.paged_attention_decode_weights(q, *lp.caches, lp.bt, lp.lens, lp.w, new, slot_positions=lp.at, **kw))
    evict = lambda **kw: pad_b200.paged_kv_evict(lp.caches, lp.w, lp.bt, lp.lens, lp.budget, lp.recent,  # noqa: E731
                                                 slot_positions=lp.at, **kw)
    decode(10 ** 6)
    decode(0)
    decode(torch.tensor([-5, 0], device="cuda"))  # nothing new, and the slots behind the sequences are nobody's
    for wrong in (torch.tensor(1, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")):
        with pytest.raises(RuntimeError, match="num_new"):
            decode(wrong)
    lp.append(lp.rand(2, lp.hkv, lp.d), lp.rand(2, lp.hkv, lp.d))
    decode(torch.tensor([1, 1], device="cuda"))
    lp.lens.copy_(evict())
    lp.append(lp.rand(2, lp.hkv, lp.d), lp.rand(2, lp.hkv, lp.d))
    was = lp.at.clone()
    for new in (1, torch.ones(2, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError, match="total_lens"):
            decode(new)
    assert torch.equal(lp.at, was)
    decode(1, total_lens=lp.total)
    with pytest.raises(ValueError, match="total_lens"):
        evict()
    lp.lens.copy_(evict(total_lens=lp.total))
    assert lp.lens.tolist() == [64, 22] and lp.at.max().item() == 10 ** 6  # (left by former owners, never looked at)
