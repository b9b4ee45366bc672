"""The engine with an 8-bit cache: what it caches, what it computes from it, windows, slots and refusals."""
import pytest
import torch

import helpers
import plain_impl
import plain_quantised as plain

pytestmark = pytest.mark.gpu

import mini_llama_cpp_release_b200 as ml
from mini_llama_cpp_release_b200.engine import MiniBatch
from mini_llama_cpp_release_b200.sampling import DeviceSampler, SamplingParams


def folder(name):
    """"A" ... "D": a tiny Qwen2; "design/config": that design's."""
    if "/" not in name:
        return helpers.model_folder(name)
    design, config = name.split("/")
    return __import__(design + "_helpers").folder_of(config)


def feed(llm, prompts, fed):
    """Prompts of unequal lengths in two steps, then for every sequence the tokens `fed`: three through `forward_batch`, the rest
    through captured decode steps.  Returns the slots and the logits of the last prompt tokens and of every fed one."""
    ctx = llm.context
    slots = [ctx.acquire() for _ in prompts]
    cut = [max(1, len(p) // 3) for p in prompts]
    out = []
    ctx.forward_batch(MiniBatch.prefill(slots, [p[:c] for p, c in zip(prompts, cut)]))
    rest = [i for i, (p, c) in enumerate(zip(prompts, cut)) if len(p) > c]
    if rest:
        ctx.forward_batch(MiniBatch.prefill([slots[i] for i in rest], [prompts[i][cut[i]:] for i in rest]))
    sampler = DeviceSampler(SamplingParams(), llm.model.runtime.device)
    for k in range(len(fed[0])):
        tokens = [f[k] for f in fed]
        if k < 3:
            out.append(ctx.forward_batch(MiniBatch.prefill(slots, [[t] for t in tokens])).float().cpu())
        else:
            out.append(ctx.decode_and_sample(slots, tokens, sampler, list(range(len(slots))))[1].float().cpu().clone())
    return slots, out


FIRST_LAYER_ATTENDS = ["A", "B", "C", "D", "W", "kebesun/attention", "kebesun/latent", "lonulix/latent", "nobonex/gated", "nobonex/conv", "bizenex/attention",
                       "bizenex/latent", "betepel/attention", "betepel/parallel"]


@pytest.mark.parametrize("name", FIRST_LAYER_ATTENDS)
def test_the_first_layer_caches_the_16_bit_rows_quantised(name):
    """The first layer's keys and values do not depend on the cache: an 8-bit cache holds what a 16-bit one holds, quantised as the format
    says, whichever kernels wrote it (short and long prompts, single tokens, captured steps)."""
    f = folder(name)
    vocab = ml.ModelConfig.from_folder(f).vocab_size
    prompts = [helpers.random_tokens(n, vocab, 10 + n) for n in (150, 1, 64, 20)]
    fed = [helpers.random_tokens(9, vocab, 20 + i) for i in range(4)]
    rows = {}
    for cache_dtype in (None, "float8_e4m3"):
        llm = ml.load(f, max_tokens=2048, cache_dtype=cache_dtype)
        slots, _ = feed(llm, prompts, fed)
        cache = llm.context.cache
        entry = next(e for e, w in enumerate(cache.where) if w is not None)
        rows[cache_dtype] = [cache.read(entry, s) for s in slots]
        cache.check()
        for s in slots:
            llm.context.release(s)
    for i, ((k16, v16), (k8, v8)) in enumerate(zip(rows[None], rows["float8_e4m3"])):
        for a, b in ((k16, k8), (v16, v8)):
            assert (a is None) == (b is None)
            if a is not None:
                assert a.shape == b.shape and a.shape[0] == len(prompts[i]) + 9
                assert torch.equal(b.double().cpu(), plain.values(*plain.quantise(a.cpu()))), f"sequence {i}"
                assert b.abs().max() > 0


@pytest.mark.parametrize("name", ["A", "C", "D", "W"])
def test_logits_against_the_plain_model_with_quantised_rows(name, monkeypatch):
    """The plain model with its keys and values rounded to 16 bits and quantised.  The engine's rows carry 16-bit roundings of the layers below, so that
    some of its numbers go to the neighbouring code: a whole step where quantisation itself is off by half a step at most.  So beside the 16-bit
    engine's tolerance the logits may be off by twice what the plain model's logits move when its rows are quantised."""
    f = folder(name)
    attention = plain_impl.attention

    def quantised(q, k, v, window=None):
        return attention(q, *(plain.values(*plain.quantise(x.to(torch.bfloat16))).to(x.dtype) for x in (k, v)), window)

    model = helpers.plain_model(f)
    vocab = ml.ModelConfig.from_folder(f).vocab_size
    prompts = [helpers.random_tokens(n, vocab, 30 + n) for n in (90, 3, 33)]
    fed = [helpers.random_tokens(8, vocab, 40 + i) for i in range(3)]
    llm = ml.load(f, max_tokens=1024, cache_dtype="fp8")
    _, got = feed(llm, prompts, fed)
    for i, (p, more) in enumerate(zip(prompts, fed)):
        monkeypatch.setattr(plain_impl, "attention", attention)
        exact = model.logits(p + more)[len(p):]
        monkeypatch.setattr(plain_impl, "attention", quantised)
        want = model.logits(p + more)[len(p):]
        moved = (exact - want).abs().max()
        for k in range(len(more)):
            off = (got[k][i] - want[k]).abs().max()
            assert off <= helpers.TOL["bfloat16"] * want[k].abs().max() + 2 * moved, (i, k, float(off), float(moved))


@pytest.mark.parametrize("name", ["C", "D", "kebesun/mixed", "betepel/mixed", "bizenex/mixed", "nobonex/mixed", "lonulix/mixed", "mepolix/mixed"])
def test_every_design_generates(name):
    f = folder(name)
    vocab = ml.ModelConfig.from_folder(f).vocab_size
    prompts = [helpers.random_tokens(n, vocab, 50 + n) for n in (70, 2, 130)]
    llm = ml.load(f, max_tokens=1024, cache_dtype="float8_e4m3")
    seen = []
    out = llm.generate(prompts, n_predict=70, stop_token_ids=[], on_step=lambda live, chosen, logits: seen.append(bool(torch.isfinite(logits).all())))
    assert all(len(t) == 70 and all(0 <= x < vocab for x in t) for t in out) and all(seen)
    assert not llm.context.cache.length
    llm.context.cache.check()
    again = llm.generate(prompts[:1], n_predict=4, stop_token_ids=[], temperature=0.8, top_k=5, seed=3)
    assert len(again[0]) == 4


def test_decode_steps_without_the_host_between_them():
    """`decode_on_device` moves the tokens' places on by itself: its cache is that of steps which the host describes."""
    f = folder("C")
    prompts = [helpers.random_tokens(n, 777, 60 + n) for n in (60, 5)]
    kept = []
    for alone in (True, False):
        llm = ml.load(f, max_tokens=1024, cache_dtype="float8_e4m3")
        ctx = llm.context
        slots = [ctx.acquire() for _ in prompts]
        ctx.forward_batch(MiniBatch.prefill(slots, prompts))
        sampler = DeviceSampler(SamplingParams(), llm.model.runtime.device)
        tokens = [1, 2]
        if alone:
            chosen = ctx.decode_on_device(slots, tokens, sampler, [0, 1], 12).tolist()
        else:
            chosen = []
            for _ in range(12):
                tokens, _ = ctx.decode_and_sample(slots, tokens, sampler, [0, 1])
                chosen.append(tokens)
        kept.append((chosen, [ctx.cache.read(0, s) for s in slots]))
    (a, rows_a), (b, rows_b) = kept
    same = next((i for i, (x, y) in enumerate(zip(a, b)) if x != y), 12)
    assert same >= 4                     # 16-bit adding products add in any order: a near-tie may go either way later on
    for (ka, va), (kb, vb), p in zip(rows_a, rows_b, prompts):
        n = len(p) + same
        assert torch.equal(ka[:n], kb[:n]) and torch.equal(va[:n], vb[:n])       # the first layer's rows follow from the tokens


def test_pages_that_a_window_gave_back_read_as_zeros():
    f = folder("kebesun/attention")                     # a window of 33 and two kept first keys
    llm = ml.load(f, max_tokens=1024, cache_dtype="float8_e4m3")
    ctx = llm.context
    slot = ctx.acquire()
    ctx.forward_batch(MiniBatch.prefill([slot], [helpers.random_tokens(300, 200, 1)]))
    k, v = ctx.cache.read(0, slot)
    assert k.shape[0] == 300
    kept = torch.zeros(300, dtype=torch.bool)
    kept[:64] = True                                    # the page of the first keys
    kept[(300 - 33 + 1) // 64 * 64:] = True
    for x in (k, v):
        assert torch.equal(x.abs().amax(dim=(1, 2)).cpu() > 0, kept)


def test_what_it_holds():
    f = folder("D")
    half, full = (ml.load(f, max_tokens=4096, cache_dtype=d).context.cache for d in ("float8_e4m3", None))
    assert full.bytes_per_token() == 2 * 2 * 2 * 128 * 2 and half.bytes_per_token() == 2 * 2 * 2 * (128 + 1)
    assert half.bytes() * 256 == full.bytes() * 129


def test_a_16_bit_cache_reads_what_was_written():
    f = folder("D")
    llm = ml.load(f, max_tokens=1024)
    ctx = llm.context
    slot = ctx.acquire()
    ctx.forward_batch(MiniBatch.prefill([slot], [helpers.random_tokens(70, 1000, 1)]))
    k, v = ctx.cache.read(1, slot)
    pages = ctx.cache.page_lists[slot][0]
    assert torch.equal(k[65], ctx.cache.k_pools[0][1, pages[1], :, 1]) and torch.equal(v[3], ctx.cache.v_pools[0][1, pages[0], :, 3])


def test_refusals():
    with pytest.raises(ValueError, match="bfloat16 engine"):
        ml.load(folder("A"), dtype="float32", cache_dtype="float8_e4m3")
    with pytest.raises(ValueError, match="cache_dtype"):
        ml.load(folder("A"), cache_dtype="int3")
    with pytest.raises(ValueError, match="8-bit cache"):
        ml.load(folder("kebesun/big_latent"), cache_dtype="float8_e4m3")          # rows of 304 numbers
    from mini_llama_cpp_release_b200.engine.context import Context
    llm = ml.load(folder("A"))
    llm.model.parts.blocks[0].mixer.takes_quantised_cache = False
    with pytest.raises(ValueError, match="16-bit keys and values only"):
        Context(llm.model, 1024, cache_dtype="float8_e4m3")
    with pytest.raises(ValueError, match="pages of 64"):
        Context(ml.load(folder("A")).model, 1024, page_size=32, cache_dtype="float8_e4m3")


@pytest.mark.parametrize("n", [5, 3, 7])
def test_no_row_of_the_cache_is_written_twice_in_a_step(n, monkeypatch):
    """A captured step is made for a few batch sizes and fills its spare rows with copies of the last sequence.  A copy's sums may differ in
    their last bits, and its codes beside the other's scale would be another row."""
    import mini_llama_cpp_release_b200.kernels as kernels
    calls = []
    quantise = kernels.quantise_kv

    def spy(k, v, positions, tok_seq, kv):
        calls.append((positions, tok_seq, kv.page_table))
        quantise(k, v, positions, tok_seq, kv)

    monkeypatch.setattr(kernels, "quantise_kv", spy)
    ctx = ml.load(folder("C"), max_tokens=2048, cache_dtype="float8_e4m3").context
    slots = [ctx.acquire() for _ in range(n)]
    ctx.forward_batch(MiniBatch.prefill(slots, [helpers.random_tokens(10 + i, 777, 80 + i) for i in range(n)]))
    sampler = DeviceSampler(SamplingParams(), ctx.model.runtime.device)
    ctx.decode_and_sample(slots, list(range(n)), sampler, list(range(n)))
    for live in (n, n - 1):                         # the second in the same captured step, where there is one
        ctx.decode_and_sample(slots[:live], list(range(live)), sampler, list(range(live)))
        torch.cuda.synchronize()
        for positions, tok_seq, table in calls:
            places = [(int(table[s, p // 64]), int(p) % 64) for p, s in zip(positions.tolist(), tok_seq.tolist()) if s >= 0]
            assert len(set(places)) == len(places)
    assert any(t.shape[0] > n - 1 for _, t, _ in calls[2:])


@pytest.mark.parametrize("name", ["C", "D", "kebesun/attention", "lonulix/latent"])
def test_prompt_steps_replayed_from_their_graph(name):
    """A step whose shape comes again is captured and replayed: other tokens in other slots, and a second chunk of each, give what the same steps give issued one by one,
    and the first layer's cached rows follow from the tokens."""
    f = folder(name)
    vocab = ml.ModelConfig.from_folder(f).vocab_size
    steps = [[helpers.random_tokens(n, vocab, 100 * k + n) for n in (90, 71, 90)] for k in range(4)]
    more = [[helpers.random_tokens(n, vocab, 50 + 100 * k + n) for n in (70, 70, 66)] for k in range(4)]
    kept = []
    for graphs in (True, False):
        ctx = ml.load(f, max_tokens=4096, cache_dtype="float8_e4m3").context
        ctx.use_graphs = graphs
        out = []
        for first, second in zip(steps, more):
            slots = [ctx.acquire() for _ in first]
            logits = [ctx.forward_batch(MiniBatch.prefill(slots, x)).float().cpu().clone() for x in (first, second)]
            entry = next(e for e, w in enumerate(ctx.cache.where) if w is not None)
            out.append((logits, [ctx.cache.read(entry, s) for s in slots]))
        assert len(getattr(ctx, "_step_graphs", {})) == (2 if graphs else 0)
        kept.append(out)
    for (logits, rows), (other, other_rows) in zip(*kept):
        for a, b in zip(logits, other):
            assert (a - b).abs().max() <= helpers.TOL["bfloat16"] * b.abs().max()
        for pair, other_pair in zip(rows, other_rows):
            for x, y in zip(pair, other_pair):
                assert (x is None) == (y is None) and (x is None or torch.equal(x, y))


def test_a_step_with_spare_rows_writes_none_of_them(monkeypatch):
    """Batches that a captured step has more rows for than sequences: the step's rows past the sequences are marked, at every step and after the batch has changed."""
    import mini_llama_cpp_release_b200.kernels as kernels
    calls = []
    quantise = kernels.quantise_kv

    def spy(k, v, positions, tok_seq, kv):
        calls.append(tok_seq)
        quantise(k, v, positions, tok_seq, kv)

    monkeypatch.setattr(kernels, "quantise_kv", spy)
    ctx = ml.load(folder("C"), max_tokens=4096, cache_dtype="float8_e4m3").context
    slots = [ctx.acquire() for _ in range(16)]
    ctx.forward_batch(MiniBatch.prefill(slots, [helpers.random_tokens(10 + i, 777, 90 + i) for i in range(16)]))
    sampler = DeviceSampler(SamplingParams(), ctx.model.runtime.device)
    spare = 0
    for live in (16, 13, 15, 11, 9, 5, 7, 3, 6):
        before = len(calls)
        for _ in range(2):
            ctx.decode_and_sample(slots[:live], list(range(live)), sampler, list(range(live)))
        torch.cuda.synchronize()
        runner = next(reversed(ctx._runners.values()))
        assert len(calls) > before or runner.n_live == live                # captured now, or a captured step that was loaded again
        seq = runner.view("store_seq")
        assert any(t.data_ptr() == seq.data_ptr() for t in calls)
        assert seq.tolist() == list(range(live)) + [-1] * (runner.B - live)
        spare += runner.B > live
    assert spare >= 4
