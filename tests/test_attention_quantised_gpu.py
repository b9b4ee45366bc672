"""Attention over the 8-bit cache against the definition in 64 bits, with bounds that count the roundings (plain_quantised.attention)."""
import math

import pytest
import torch

import plain_quantised as plain

pytestmark = pytest.mark.gpu


def kernels():
    from mini_llama_cpp_release_b200 import kernels as k
    return k


class Case:
    """Sequences (cached, new) over pages in no order; whatever no sequence's key owns is bytes of every kind, NaN codes and the scale of
    a row that is not finite among them."""

    def __init__(self, H, KV, hd, seqs, seed=0, entries=2, entry=1, shared=False, q_size=1.5, v_spread=0, k_rows=None, v_rows=None, tail=0):
        dev = "cuda"
        g = torch.Generator(device=dev).manual_seed(seed)
        self.H, self.KV, self.hd, self.seqs = H, KV, hd, seqs
        lens = [c + n for c, n in seqs]
        n_pages = sum((t + 63) // 64 for t in lens) + 2
        width = max(1, max((t + 63) // 64 for t in lens))
        order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = torch.full((len(seqs), width), -1, dtype=torch.int32)
        shape = (entries, n_pages, KV, 64, hd)
        self.codes = [torch.randint(0, 256, shape, generator=g, device=dev).to(torch.uint8) for _ in range(1 if shared else 2)]
        self.scales = [torch.randint(0, 256, shape[:4], generator=g, device=dev).to(torch.uint8) for _ in range(1 if shared else 2)]
        for t in self.codes:
            t[:, :, :, ::5] = 0x7f
        for t in self.scales:
            t[:, :, :, ::7] = 255
        self.k, self.v = [], []
        for b, t in enumerate(lens):
            pages = [order.pop() for _ in range((t + 63) // 64)]
            self.table[b, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            k = torch.randn(t, KV, hd, generator=g, device=dev) if k_rows is None else k_rows(b, t, g)
            v = torch.randn(t, KV, hd, generator=g, device=dev) if v_rows is None else v_rows(b, t, g)
            if v_spread:
                v = v * torch.exp2(torch.randint(-v_spread, v_spread + 1, (t, KV, 1), generator=g, device=dev).float())
            kept = []
            for i, x in enumerate((k,) if shared else (k, v)):
                codes, byte = plain.quantise(x)
                kept.append(plain.values(codes, byte))
                for p, page in enumerate(pages):
                    n = min(64, t - 64 * p)
                    self.codes[i][entry, page, :, :n] = codes[64 * p:64 * p + n].transpose(0, 1)
                    self.scales[i][entry, page, :, :n] = byte[64 * p:64 * p + n].T
            self.k.append(kept[0])
            self.v.append(kept[-1])
        self.n = sum(n for _, n in seqs)
        self.tail = tail
        self.q = (torch.randn(self.n + tail, H * hd, generator=g, device=dev) * q_size).bfloat16()
        self.cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).int().to(dev)
        self.start = torch.tensor([c for c, _ in seqs], dtype=torch.int32, device=dev)
        self.sinks = torch.randn(H, generator=g, device=dev)
        self.entry, self.shared = entry, shared

    def view(self, table=None):
        e4 = torch.float8_e4m3fn
        k, ks = self.codes[0].view(e4), self.scales[0]
        v, vs = (k, ks) if self.shared else (self.codes[1].view(e4), self.scales[1])
        return kernels().QuantisedKVView(k, v, ks, vs, self.entry * self.codes[0][0].numel(), (self.table if table is None else table).cuda(), 64,
                                         self.KV, self.hd)

    def run(self, scale=None, window=0, keep_first=0, chunk=0, softcap=0.0, sinks=False, table=None, out=None, max_kv=None):
        out = torch.full_like(self.q, 7.0) if out is None else out
        kernels().attention_quantised(self.q, out, self.cu, self.start, len(self.seqs), max(n for _, n in self.seqs),
                                      max(c + n for c, n in self.seqs) if max_kv is None else max_kv, self.H, self.view(table),
                                      self.hd ** -0.5 if scale is None else scale, window, sinks=self.sinks if sinks else None,
                                      keep_first=keep_first, chunk=chunk, softcap=softcap)
        return out

    def check(self, out, scale=None, window=0, keep_first=0, chunk=0, softcap=0.0, sinks=False, gone=()):
        """`gone`: (sequence, page index) whose page is missing."""
        at = 0
        for b, (c, n) in enumerate(self.seqs):
            if n == 0:
                continue
            seen = plain.visible(torch.arange(c, c + n, device="cuda"), c + n, window, keep_first, chunk)
            for s, p in gone:
                if s == b:
                    seen[:, 64 * p:64 * p + 64] = False
            q = self.q[at:at + n].view(n, self.H, self.hd)
            want, bound = plain.attention(q, self.k[b], self.v[b], seen, self.hd ** -0.5 if scale is None else scale,
                                          self.sinks if sinks else None, softcap)
            got = out[at:at + n].view(n, self.H, self.hd).double()
            assert torch.isfinite(got).all(), f"sequence {b}"
            worst = ((got - want).abs() / bound).max()
            assert worst <= 1.0, f"sequence {b}: {float(worst):.3g} of the bound"
            at += n
        if self.tail:
            assert (out[self.n:] == 7.0).all(), "rows behind the last sequence"
        kernels().check_gemm_status(torch.device("cuda", 0))


LAYOUTS = [(14, 2, 64), (12, 2, 128), (4, 4, 16), (6, 2, 48), (8, 1, 256), (40, 2, 64)]
SINGLES = [
    [(0, 1)],
    [(62, 1)], [(63, 1)], [(64, 1)],
    [(0, 1), (1, 1), (64, 1), (999, 1), (127, 1)],
    [(5000, 1), (3, 1)],
]


@pytest.mark.parametrize("H,KV,hd", LAYOUTS)
@pytest.mark.parametrize("seqs", SINGLES, ids=[str(i) for i in range(len(SINGLES))])
def test_single_tokens(H, KV, hd, seqs):
    c = Case(H, KV, hd, seqs, tail=2)
    c.check(c.run())


MASKS = [
    dict(window=1), dict(window=64), dict(window=100, keep_first=4), dict(window=3, keep_first=130), dict(window=2000, keep_first=1),
    dict(chunk=1), dict(chunk=100), dict(softcap=5.0), dict(sinks=True), dict(window=70, keep_first=65, sinks=True, softcap=3.0),
]


@pytest.mark.parametrize("mask", MASKS, ids=[str(m) for m in MASKS])
@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (12, 2, 128), (6, 2, 48)])
def test_single_tokens_with_masks(H, KV, hd, mask):
    c = Case(H, KV, hd, [(700, 1), (0, 1), (99, 1), (100, 1), (63, 1), (1500, 1)], seed=3)
    c.check(c.run(**mask), **mask)


CHUNKS = [
    [(0, 2)],
    [(0, 64)], [(0, 65)], [(63, 2), (0, 1), (64, 64)],
    [(300, 129), (0, 1), (1000, 17), (5, 300)],
    [(0, 700), (2500, 90)],
]


@pytest.mark.parametrize("H,KV,hd", LAYOUTS)
@pytest.mark.parametrize("seqs", CHUNKS, ids=[str(i) for i in range(len(CHUNKS))])
def test_chunks(H, KV, hd, seqs):
    c = Case(H, KV, hd, seqs, seed=1, tail=3)
    c.check(c.run())


@pytest.mark.parametrize("mask", MASKS, ids=[str(m) for m in MASKS])
@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (12, 2, 128), (6, 2, 48)])
def test_chunks_with_masks(H, KV, hd, mask):
    c = Case(H, KV, hd, [(700, 150), (0, 1), (0, 260), (100, 5), (1500, 40)], seed=4)
    c.check(c.run(**mask), **mask)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("seqs", [[(4000, 1)], [(800, 200)]], ids=["single", "chunk"])
def test_values_whose_rows_differ_by_many_binades(hd, seqs):
    c = Case(14, 2, hd, seqs, seed=5, v_spread=20)
    c.check(c.run())


@pytest.mark.parametrize("seqs", [[(900, 1)], [(300, 200)]], ids=["single", "chunk"])
def test_values_of_zeros_count_in_the_denominator(seqs):
    """Rows of zeros have the lowest scale; rows far larger than the others must not push them out of the sum."""
    def rows(b, t, g):
        v = torch.zeros(t, 2, 64, device="cuda")
        v[::50] = 2.0 ** 22 * torch.randn(v[::50].shape, generator=g, device="cuda")
        return v
    c = Case(14, 2, 64, seqs, seed=6, v_rows=rows)
    c.check(c.run())


@pytest.mark.parametrize("seqs", [[(500, 1), (20, 1)], [(300, 200)]], ids=["single", "chunk"])
def test_values_read_out_of_the_key_rows(seqs):
    c = Case(14, 1, 128, seqs, seed=7, shared=True)
    c.check(c.run())


@pytest.mark.parametrize("exponent", [-60, 60])
@pytest.mark.parametrize("seqs", [[(500, 1)], [(300, 200)]], ids=["single", "chunk"])
def test_large_queries_on_small_keys(exponent, seqs):
    def rows(b, t, g):
        return torch.randn(t, 2, 64, generator=g, device="cuda") * 2.0 ** -exponent
    c = Case(14, 2, 64, seqs, seed=8, q_size=2.0 ** exponent, k_rows=rows)
    c.check(c.run())


@pytest.mark.parametrize("seqs", [[(900, 1), (64, 1)], [(300, 200), (0, 70)]], ids=["single", "chunk"])
@pytest.mark.parametrize("value", [-1, 10 ** 6], ids=["negative", "beyond the pool"])
def test_missing_pages(seqs, value):
    c = Case(14, 2, 64, seqs, seed=9)
    table = c.table.clone()
    table[0, 2] = value
    table[1, 0] = value
    c.check(c.run(table=table), gone=[(0, 2), (1, 0)])


@pytest.mark.parametrize("seqs", [[(30, 1), (100, 1)], [(0, 40), (60, 130)]], ids=["single", "chunk"])
@pytest.mark.parametrize("sinks", [False, True])
def test_rows_that_see_no_key_are_zeros(seqs, sinks):
    c = Case(14, 2, 64, seqs, seed=10)
    table = c.table.clone()
    table[0, :] = -1
    out = c.run(table=table, sinks=sinks)
    assert not out[:seqs[0][1]].any()
    c.check(out, gone=[(0, p) for p in range(c.table.shape[1])], sinks=sinks)


@pytest.mark.parametrize("seqs,window", [([(200, 1), (200, 1)], 100), ([(130, 100), (130, 100)], 50)], ids=["single", "chunk"])
@pytest.mark.parametrize("which", [0, 1], ids=["keys", "values"])
def test_a_row_that_is_not_finite_reaches_those_that_see_it_only(seqs, window, which):
    c = Case(14, 2, 64, seqs, seed=11)
    clean = c.run(window=window)
    spoilt = 140                                   # of sequence 0, kv head 1
    c.codes[which][1, c.table[0, spoilt // 64], 1, spoilt % 64] = 0
    c.scales[which][1, c.table[0, spoilt // 64], 1, spoilt % 64] = 255
    out = c.run(window=window).view(-1, 14, 64)
    clean = clean.view(-1, 14, 64)
    n = seqs[0][1]
    p = torch.arange(seqs[0][0], seqs[0][0] + n, device="cuda")
    sees = (spoilt <= p) & (p - spoilt < window)
    hit = torch.zeros(out.shape[0], 14, dtype=torch.bool, device="cuda")
    hit[:n, 7:] = sees[:, None]
    assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


def test_a_window_whose_pages_were_given_back():
    c = Case(14, 2, 64, [(1000, 1), (900, 30)], seed=12)
    table = c.table.clone()
    for b, first in ((0, 1000 - 100 + 1), (1, 900 - 100 + 1)):
        table[b, 1:first // 64] = -1
    c.check(c.run(window=100, keep_first=4, table=table), window=100, keep_first=4)


def test_empty_sequences_and_bounds_that_are_too_large_or_too_small():
    c = Case(14, 2, 64, [(10, 0), (200, 3), (0, 0), (64, 1), (5, 0)], seed=13, tail=1)
    c.check(c.run())
    c.check(c.run(max_kv=30000))
    c.check(c.run(max_kv=1))                       # a bound that is too small costs time, not keys


@pytest.mark.parametrize("seqs", [[(2000, 1)] * 3, [(500, 100), (0, 300)]], ids=["single", "chunk"])
def test_captured_on_another_stream_and_two_graphs_at_once(seqs):
    a, b = Case(14, 2, 64, seqs, seed=14), Case(14, 2, 64, seqs, seed=15)
    outs = [torch.zeros_like(a.q), torch.zeros_like(b.q)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    views = [a.view(), b.view()]
    graphs = []

    def call(i):
        c = (a, b)[i]
        kernels().attention_quantised(c.q, outs[i], c.cu, c.start, len(seqs), max(n for _, n in seqs), max(x + n for x, n in seqs), 14, views[i], 0.125)

    for i in range(2):
        streams[i].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[i]):
            call(i)
        streams[i].synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            call(i)
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        a.check(outs[0])
        b.check(outs[1])


def test_the_same_call_twice_gives_the_same_bits():
    for seqs in ([(3000, 1), (17, 1)], [(300, 200)]):
        c = Case(14, 2, 64, seqs, seed=16)
        assert torch.equal(c.run(), c.run())


def test_refusals():
    import dataclasses
    K = kernels()
    c = Case(14, 2, 64, [(10, 1)], seed=17)
    kv = c.view()
    ok = dict(q=c.q, out=torch.empty_like(c.q), cu=c.cu, start=c.start, n_seqs=1, H=14, kv=kv, scale=0.1, more={})
    bad = [dict(q=c.q.float()), dict(out=c.q.float()), dict(H=13), dict(H=28), dict(n_seqs=2), dict(cu=c.cu.long()), dict(scale=0.0), dict(scale=math.nan),
           dict(more=dict(window=-1)), dict(more=dict(window=4, chunk=4)), dict(more=dict(softcap=-1.0)), dict(more=dict(softcap=math.nan)),
           dict(more=dict(keep_first=-1)), dict(more=dict(sinks=c.sinks[:3])), dict(more=dict(sinks=c.sinks.double())),
           dict(kv=dataclasses.replace(kv, page_size=32)), dict(q=c.q.cpu()), dict(out=torch.empty(1, 14 * 64 * 2, device="cuda", dtype=torch.bfloat16)[:, ::2])]
    for change in bad:
        a = {**ok, **change}
        with pytest.raises(K.KernelError):
            K.attention_quantised(a["q"], a["out"], a["cu"], a["start"], a["n_seqs"], 1, 11, a["H"], a["kv"], a["scale"], **a["more"])


@pytest.mark.parametrize("which", [0, 1], ids=["keys", "values"])
@pytest.mark.parametrize("seqs,window", [([(200, 1), (200, 1)], 100), ([(130, 100), (130, 100)], 50)], ids=["single", "chunk"])
def test_a_capped_score_that_is_not_finite_reaches_no_neighbour(seqs, window, which):
    """Row 190 of the chunk sees key 141 and not key 140 beside it, which is not finite."""
    c = Case(14, 2, 64, seqs, seed=31)
    clean = c.run(window=window, softcap=4.0).view(-1, 14, 64)
    c.codes[which][1, c.table[0, 2], 1, 12] = 0
    c.scales[which][1, c.table[0, 2], 1, 12] = 255
    out = c.run(window=window, softcap=4.0).view(-1, 14, 64)
    p = torch.arange(seqs[0][0], seqs[0][0] + seqs[0][1], device="cuda")
    hit = torch.zeros(out.shape[0], 14, dtype=torch.bool, device="cuda")
    hit[:seqs[0][1], 7:] = ((140 <= p) & (p - 140 < window))[:, None]
    assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (12, 2, 128), (6, 2, 48)])
@pytest.mark.parametrize("softcap,size", [(0.5, 40.0), (30.0, 60.0), (2.0, 300.0), (50.0, 0.01)])
@pytest.mark.parametrize("seqs", [[(150, 1), (63, 1)], [(70, 90), (0, 129)]], ids=["single", "chunk"])
def test_capped_scores_far_past_the_cap_and_near_zero(H, KV, hd, softcap, size, seqs):
    c = Case(H, KV, hd, seqs, seed=32, q_size=size)
    c.check(c.run(softcap=softcap), softcap=softcap)


@pytest.mark.parametrize("bound", [2048, 16384, 1 << 20])
@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (12, 2, 128), (8, 1, 256)])
@pytest.mark.parametrize("seqs", [[(0, 1)], [(70, 1), (0, 1), (1300, 1)], [(600, 3), (64, 1)]], ids=["one", "three", "few"])
def test_a_bound_far_above_the_lengths(H, KV, hd, seqs, bound):
    c = Case(H, KV, hd, seqs, seed=33)
    c.check(c.run(max_kv=bound))
    c.check(c.run(max_kv=bound, window=100, keep_first=3, sinks=True), window=100, keep_first=3, sinks=True)


@pytest.mark.parametrize("n_splits,split_tiles", [(2, 1), (5, 3), (16, 8)])
@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("mask", [dict(), dict(sinks=True, softcap=5.0), dict(window=70, keep_first=65, sinks=True), dict(chunk=100)],
                         ids=["all", "sinks", "window", "chunk"])
def test_first_row_tiles_shared_out_and_the_others_whole(monkeypatch, H, KV, hd, n_splits, split_tiles, mask):
    """Sequences shorter than the split rows, one without new tokens, a page that is missing, and rows behind the last sequence's."""
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    monkeypatch.setattr(bindings, "_attention_q8_form", lambda *sizes: (n_splits, min(split_tiles, -(-150 // (128 // (H // KV))))))
    empty = torch.empty

    def spoilt(*a, **k):
        t = empty(*a, **k)
        return t.fill_(float("nan")) if t.is_floating_point() else t

    monkeypatch.setattr(bindings.torch, "empty", spoilt)
    c = Case(H, KV, hd, [(70, 90), (0, 150), (500, 3), (10, 0), (700, 20)], seed=34, tail=3)
    c.check(c.run(**mask), **mask)
    table = c.table.clone()
    table[0, 0] = table[4, 3] = -1
    c.check(c.run(table=table, **mask), gone=[(0, 0), (4, 3)], **mask)


@pytest.mark.parametrize("H,KV,hd,new,cached", [(28, 4, 128, 700, 3000), (14, 2, 64, 1400, 9000)])
def test_a_partial_wave_behind_whole_ones(H, KV, hd, new, cached):
    plan = kernels().attention_q8_tcgen05_plan(new, 1, new + cached, H, KV, hd, torch.cuda.get_device_properties(0).multi_processor_count)
    assert plan[0] > 1 and 0 < plan[1] < -(-new // (128 // (H // KV)))
    c = Case(H, KV, hd, [(cached, new)], seed=35, tail=1)
    c.check(c.run())
    again = c.run()
    assert torch.equal(again, c.run())


@pytest.mark.parametrize("H,KV,hd,seqs", [(12, 4, 48, [(6000, 300)]), (8, 1, 256, [(6100, 140), (20, 200)])], ids=["48", "256"])
def test_long_chunks_of_other_head_sizes_in_two_shares(H, KV, hd, seqs):
    plan = kernels().attention_q8_plan(max(n for _, n in seqs), len(seqs), max(c + n for c, n in seqs), H, KV, hd,
                                       torch.cuda.get_device_properties(0).multi_processor_count)
    assert plan[0] == 64 and plan[1] >= 2
    c = Case(H, KV, hd, seqs, seed=36, tail=1)
    c.check(c.run())
    c.check(c.run(sinks=True, softcap=9.0), sinks=True, softcap=9.0)


@pytest.mark.parametrize("form", [(5, 3), (8, 0, "few")], ids=["first row tiles", "equal shares"])
def test_two_captured_graphs_with_splits_and_other_lengths_at_replay(monkeypatch, form):
    """Partial results are each graph's own, and shares follow the lengths that the replay finds."""
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    seqs = [(70, 90), (500, 130)] if len(form) == 2 else [(700, 1), (90, 1), (1500, 1)]
    monkeypatch.setattr(bindings, "_attention_q8_form", lambda *sizes: form if len(form) == 2 else (8, 8, 0, False))
    cases = [Case(14, 2, 64, seqs, seed=40 + i, tail=1) for i in range(2)]
    streams, graphs, outs, views = [torch.cuda.Stream() for _ in cases], [], [torch.full_like(c.q, 7.0) for c in cases], [c.view() for c in cases]

    def call(i):
        c = cases[i]
        kernels().attention_quantised(c.q, outs[i], c.cu, c.start, len(seqs), max(n for _, n in seqs), 4096, 14, views[i], 0.125)

    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call(i)
        s.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=s):
            call(i)
    for cut in (0, 33, 37):
        for i, c in enumerate(cases):
            c.start -= cut
            c.seqs = [(cached - cut, n) for cached, n in c.seqs]
            c.k, c.v = [k[:len(k) - cut] for k in c.k], [v[:len(v) - cut] for v in c.v]
            outs[i].fill_(7.0)
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i, c in enumerate(cases):
            c.check(outs[i])


@pytest.mark.parametrize("form", [(8, 5, 0, False), (8, 4, 0, True), (8, 3, 5, False), (64, 2, 0, False), (3, 1), (1, 0)], ids=str)
def test_rows_before_the_first_sequence_are_left_as_they_are(monkeypatch, form):
    """Whatever lies in fresh memory, the joining of key splits writes the sequences' rows only."""
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    monkeypatch.setattr(bindings, "_attention_q8_form", lambda *sizes: form)
    empty = torch.empty
    monkeypatch.setattr(bindings.torch, "empty", lambda *a, **k: (lambda t: t.fill_(3.0) if t.is_floating_point() else t)(empty(*a, **k)))
    c = Case(14, 2, 64, [(900, 1), (70, 1)] if form[0] == 8 else [(900, 9), (70, 2)], seed=50, tail=2)
    before = 3
    q, cu = c.q, c.cu
    c.q = torch.cat([q[:before], q])
    c.cu = cu + before
    out = c.run()
    assert (out[:before] == 7.0).all()
    c.q, c.cu = q, cu
    c.check(out[before:])


@pytest.mark.parametrize("mask", [dict(window=100), dict(window=64, keep_first=65), dict(chunk=100)], ids=str)
def test_pages_written_out_follow_the_mask_and_not_the_page_list(mask):
    """A few new tokens far into long sequences whose layer has a mask: scratch for the pages that they see."""
    c = Case(14, 2, 64, [(9000, 40), (30, 70), (6000, 1)], seed=51, tail=1)
    out = torch.full_like(c.q, 7.0)
    view = c.view()
    c.run(out=out, **mask)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    kernels().attention_quantised(c.q, out, c.cu, c.start, 3, 70, 9040, 14, view, 0.125, **mask)
    torch.cuda.synchronize()
    # keys and values, 2 kv heads of 64 in bfloat16, at most 7 pages of each sequence (100 keys, 72 rows in whole blocks of 18 tokens, two kept pages)
    assert kernels().attention_q8_tcgen05_plan(70, 3, 9040, 14, 2, 64, 148, **mask) == (1, 0)
    assert torch.cuda.max_memory_allocated() - before <= 3 * 7 * 64 * 2 * 2 * 64 * 2 + 4096
    c.check(out, **mask)


class Spy:
    """A library of attention kernels that notes which entry point a call went through."""

    def __init__(self, lib):
        self.lib, self.calls = lib, []

    def __getattr__(self, name):
        f = getattr(self.lib, name)
        return lambda *a: (self.calls.append(name), f(*a))[1]


def spied(monkeypatch, hd):
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    spy = Spy(kernels().attention_q8_library(hd))
    monkeypatch.setitem(bindings._attn_q8_libs, hd, spy)
    return spy


GROUPS = [(70, 90), (0, 150), (500, 3), (10, 0), (700, 20), (64, 64), (0, 1)]


@pytest.mark.parametrize("at_once", [1, 2, 3, 6])
@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("mask", [dict(), dict(sinks=True, softcap=5.0), dict(window=70, keep_first=65, sinks=True), dict(chunk=100)],
                         ids=["all", "sinks", "window", "chunk"])
def test_as_many_sequences_at_a_time_as_scratch_memory_holds(monkeypatch, H, KV, hd, mask, at_once):
    """The sequences' pages are written out in groups: every sequence as in one call for all, one without new tokens, a missing page and rows behind the last among them."""
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    spy = spied(monkeypatch, hd)
    c = Case(H, KV, hd, GROUPS, seed=52, tail=3)
    places = kernels().attention_q8_places(150, c.table.shape[1], H, KV, mask.get("window", 0), mask.get("keep_first", 0), mask.get("chunk", 0))
    per_seq = KV * places * 64 * hd * 2 * 2
    monkeypatch.setattr(bindings, "EXPANDED_AT_ONCE", at_once * per_seq + per_seq // 2)
    monkeypatch.setattr(bindings, "EXPANDED_BYTES", per_seq)
    c.check(c.run(**mask), **mask)
    assert spy.calls == ["mlc_attention_q8_tcgen05"] * -(-len(GROUPS) // at_once)
    table = c.table.clone()
    table[0, 0] = table[4, 3] = -1
    c.check(c.run(table=table, **mask), gone=[(0, 0), (4, 3)], **mask)


def test_scratch_memory_that_is_short_halves_the_groups(monkeypatch):
    """Where several sequences' pages find no room, fewer at a time are tried, down to one, before the form without is taken."""
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    spy = spied(monkeypatch, 64)
    c = Case(14, 2, 64, GROUPS, seed=53, tail=1)
    per_seq = 2 * c.table.shape[1] * 128 * 64
    empty = torch.empty

    def short(n, *a, **k):
        if k.get("dtype") == torch.bfloat16 and n > room:
            raise torch.OutOfMemoryError("no room")
        return empty(n, *a, **k)

    monkeypatch.setattr(bindings.torch, "empty", short)
    for room, calls in ((3 * per_seq, 3), (per_seq, 7)):
        del spy.calls[:]
        c.check(c.run(out=torch.full_like(c.q, 7.0)))
        assert spy.calls == ["mlc_attention_q8_tcgen05"] * calls
    room = per_seq - 1
    del spy.calls[:]
    c.check(c.run(out=torch.full_like(c.q, 7.0)))
    assert spy.calls == ["mlc_attention_q8"]


@pytest.fixture(params=[(14, 2, 64), (12, 2, 128), (28, 4, 128), (5, 1, 64)], ids=str)
def without_scratch(request, monkeypatch):
    """Layouts whose many-token calls run in the form without scratch pages, 64 rows a block, because there is no room for them; that they do is checked."""
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    monkeypatch.setattr(bindings, "EXPANDED_BYTES", 0)
    spy = spied(monkeypatch, request.param[2])
    yield request.param
    assert spy.calls and set(spy.calls) == {"mlc_attention_q8"}


@pytest.mark.parametrize("seqs", CHUNKS[1:], ids=[str(i) for i in range(1, len(CHUNKS))])
def test_chunks_without_scratch(without_scratch, seqs):
    c = Case(*without_scratch, seqs, seed=60, tail=3)
    c.check(c.run())


@pytest.mark.parametrize("mask", MASKS, ids=[str(m) for m in MASKS])
def test_chunks_with_masks_without_scratch(without_scratch, mask):
    c = Case(*without_scratch, [(700, 150), (0, 1), (0, 260), (100, 5), (1500, 40)], seed=61)
    c.check(c.run(**mask), **mask)


@pytest.mark.parametrize("mask", [dict(), dict(window=100, keep_first=4, sinks=True)], ids=["all", "window"])
def test_missing_pages_without_scratch(without_scratch, mask):
    c = Case(*without_scratch, [(300, 200), (0, 70), (30, 100)], seed=62)
    table = c.table.clone()
    table[0, 2], table[1, 0], table[2, :] = -1, 10 ** 6, -1
    out = c.run(table=table, **mask)
    c.check(out, gone=[(0, 2), (1, 0)] + [(2, p) for p in range(table.shape[1])], **mask)
    assert not out[270:].any()


@pytest.mark.parametrize("which", [0, 1], ids=["keys", "values"])
@pytest.mark.parametrize("softcap", [0.0, 4.0])
def test_a_row_that_is_not_finite_without_scratch(without_scratch, which, softcap):
    H, KV, hd = without_scratch
    c = Case(H, KV, hd, [(130, 100), (130, 100)], seed=63)
    clean = c.run(window=50, softcap=softcap).view(-1, H, hd)
    c.check(clean.view(c.n, -1), window=50, softcap=softcap)
    c.codes[which][1, c.table[0, 2], KV - 1, 12] = 0                # key 140 of sequence 0
    c.scales[which][1, c.table[0, 2], KV - 1, 12] = 255
    out = c.run(window=50, softcap=softcap).view(-1, H, hd)
    p = torch.arange(130, 230, device="cuda")
    hit = torch.zeros(out.shape[0], H, dtype=torch.bool, device="cuda")
    hit[:100, H - H // KV:] = ((140 <= p) & (p - 140 < 50))[:, None]
    assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("softcap,size", [(0.5, 40.0), (30.0, 60.0), (50.0, 0.01)])
def test_capped_scores_without_scratch(without_scratch, softcap, size):
    c = Case(*without_scratch, [(70, 90), (0, 129)], seed=64, q_size=size)
    c.check(c.run(softcap=softcap), softcap=softcap)


def test_long_chunks_in_two_shares_without_scratch(without_scratch):
    c = Case(*without_scratch, [(6000, 300), (6100, 90)], seed=65, tail=1)
    c.check(c.run())


SHORT = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (48, 8, 64), (10, 2, 128)]


@pytest.mark.parametrize("H,KV,hd", SHORT)
@pytest.mark.parametrize("new", range(2, 11))
def test_short_turns_behind_hundreds_of_keys(H, KV, hd, new):
    """2 to 10 new tokens with groups of 5 to 7: every form by number of rows, and ragged beside single tokens."""
    c = Case(H, KV, hd, [(700, new), (333, 1), (64 * 5 - new, new), (0, new), (450, max(1, new - 3))], seed=66, tail=2)
    c.check(c.run())
    c.check(c.run(window=130, keep_first=3, sinks=True, softcap=20.0), window=130, keep_first=3, sinks=True, softcap=20.0)


@pytest.mark.parametrize("H,hd", [(28, 128), (12, 128), (20, 64), (28, 48)])
@pytest.mark.parametrize("seqs", [[(500, 1), (20, 1), (3000, 1)], [(700, 2), (90, 2)], [(300, 200), (0, 33), (64, 1)]], ids=["single", "two", "chunk"])
def test_shared_rows_for_many_heads(H, hd, seqs):
    """One row of keys that are the values too, for up to 28 heads: more than a block of single tokens takes."""
    c = Case(H, 1, hd, seqs, seed=67, shared=True, tail=1)
    c.check(c.run())
    c.check(c.run(window=100, keep_first=2, sinks=True), window=100, keep_first=2, sinks=True)


@pytest.mark.parametrize("group", range(1, 17))
@pytest.mark.parametrize("hd", [64, 128])
def test_every_group_of_single_tokens_joined_in_clusters(hd, group):
    """Rows that fill a warp's columns and rows that do not, in a cluster of blocks that join among themselves."""
    plan = kernels().attention_q8_plan(1, 2, 2001, group, 1, hd, torch.cuda.get_device_properties(0).multi_processor_count)
    assert plan[1] > 1 and plan[3]
    c = Case(group, 1, hd, [(2000, 1), (77, 1)], seed=68, tail=1)
    c.check(c.run())
    c.check(c.run(sinks=True, softcap=8.0), sinks=True, softcap=8.0)


@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (12, 2, 128), (28, 1, 128)])
@pytest.mark.parametrize("seqs", [[(2000, 1)], [(8000, 1), (17, 1)], [(20000, 1)] * 2, [(3000, 1)] * 90, [(700, 6)] * 3, [(900, 150)], [(30, 90), (500, 40)]], ids=str)
def test_every_form_gives_the_same_bits_again(H, KV, hd, seqs):
    c = Case(H, KV, hd, seqs, seed=69)
    first = c.run()
    for _ in range(3):
        assert torch.equal(first, c.run())


@pytest.mark.parametrize("width", [0, 1, 3, 9])
@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (12, 2, 128), (6, 2, 48)])
@pytest.mark.parametrize("seqs", [[(700, 1), (64, 1), (20, 1)], [(700, 150), (0, 260), (100, 5), (560, 40)]], ids=["single", "chunk"])
@pytest.mark.parametrize("mask", [dict(), dict(window=100), dict(window=64, keep_first=130, sinks=True), dict(chunk=100, softcap=5.0)], ids=str)
def test_page_lists_that_end_before_the_sequences(H, KV, hd, seqs, mask, width):
    """Keys behind what a list holds are not seen, and a list may hold nothing."""
    c = Case(H, KV, hd, seqs, seed=70, tail=1)
    table = c.table[:, :width].contiguous()
    c.check(c.run(table=table, **mask), gone=[(b, p) for b in range(len(seqs)) for p in range(width, c.table.shape[1])], **mask)


@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (6, 2, 48)])
@pytest.mark.parametrize("seqs", [[(700, 1), (64, 1)], [(700, 90), (0, 130)]], ids=["single", "chunk"])
@pytest.mark.parametrize("mask,same", [(dict(window=(1 << 32) + 5), dict()), (dict(chunk=1 << 40), dict()), (dict(window=3, keep_first=(1 << 31) - 1), dict()),
                                       (dict(window=(1 << 31) - 1, keep_first=4), dict())], ids=str)
def test_masks_longer_than_any_sequence(H, KV, hd, seqs, mask, same):
    c = Case(H, KV, hd, seqs, seed=71, tail=1)
    out = c.run(**mask)
    c.check(out, **same)
