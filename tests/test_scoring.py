"""Forked sequences, several continuations and scored texts on a machine without a GPU: the cache's bookkeeping over CPU tensors, the engine
over the plain kernel functions, and what the entry points refuse."""
import random

import numpy as np
import pytest
import torch

import kernel_refs
import plain_gemma2 as plain
import scoring_refs
from rust_deeplearning_b200.cache.cache import Cache, CacheError, KVRequirement, PagePool, RunNeeds, StateRequirement
from rust_deeplearning_b200.engine.api import Generator
from rust_deeplearning_b200.engine.generate import generate, plan_batches, score
from rust_deeplearning_b200.engine.step import StepError
from rust_deeplearning_b200.kernels import ops
from rust_deeplearning_b200.kernels.library import KernelError
from rust_deeplearning_b200.sampling.sampler import SamplingParams
from test_engine_host import build, close, prompt

PAGE = 4


# ---- pages with several holders ----

def test_a_page_is_free_when_its_last_holder_gives_it_back():
    p = PagePool(3)
    a, b = p.take(2)
    p.share([a], 2)
    assert p.holders(a) == 3 and p.holders(b) == 1 and p.n_shared == 1
    p.share([b], 0); p.share([])
    p.give_back([a, b])
    assert p.n_shared == 1
    p.give_back([a])
    assert p.n_free == 2 and p.holders(a) == 1 and p.n_shared == 0
    p.give_back([a])
    assert p.n_free == 3
    with pytest.raises(CacheError):
        p.give_back([a])
    with pytest.raises(CacheError):
        p.share([b])
    with pytest.raises(CacheError):
        p.share([7])
    c, = p.take(1)
    with pytest.raises(CacheError):
        p.share([c, 7])
    assert p.holders(c) == 1 and p.n_shared == 0


class Model:
    """What every live slot should read: for each slot the number written at each position, and its state."""

    def __init__(self, window):
        self.window, self.text, self.state = window, {}, {}


def write(cache, group, slot, first, values):
    g = cache.kv_groups[group]
    for pos, v in enumerate(values, first):
        page = g.pages[slot][(pos // PAGE) % g.ring_pages]
        g.k[:, page, 0, pos % PAGE] = float(v)
        g.v[:, page, 0, pos % PAGE] = float(-v)


def read(cache, group, slot, pos):
    g = cache.kv_groups[group]
    page = g.pages[slot][(pos // PAGE) % g.ring_pages]
    k, v = g.k[:, page, 0, pos % PAGE], g.v[:, page, 0, pos % PAGE]
    assert (k == k.flatten()[0]).all() and (v == -k.flatten()[0]).all()
    return int(k.flatten()[0])


@pytest.mark.parametrize("seed", range(12))
def test_forked_slots_read_what_they_would_read_alone(monkeypatch, seed):
    """Slots are made, forked, stepped (several in one step, one or many positions) and freed at random; before a step's own positions are
    written every one of its queries must find the earlier positions it sees, and after it every live slot too."""
    scoring_refs.install(monkeypatch)
    rnd = random.Random(seed)
    windows = [None, 5, 8, 13]
    needs = [RunNeeds(KVRequirement(1, 1, w)) for w in windows for _ in range(2)] + [RunNeeds(None, StateRequirement((3,)))]
    cache = Cache(needs, max_tokens=600, max_seqs=7, max_context=90, page_size=PAGE, dtype=torch.float32, device="cpu")
    text, counter, copies = {}, [0], [0]
    plain_copy = scoring_refs.copy_rows

    def counted(moves):
        copies[0] += 1
        plain_copy(moves)
    monkeypatch.setattr(ops, "copy_rows", counted)

    def sees(slot, query, upto):
        for gi, g in enumerate(cache.kv_groups):
            w = g.requirement.window
            for pos in range(0 if w is None else max(0, query - w + 1), upto):
                assert read(cache, gi, slot, pos) == text[slot][pos], (seed, slot, pos, w)

    for _ in range(150):
        live = cache.live_slots()
        do = rnd.random()
        if (do < 0.15 or not live) and cache.n_free_slots:
            s = cache.alloc_slot()
            text[s] = []
            cache.state_groups[0].data[:, s] = float(s + 1)
        elif do < 0.4 and live:
            s, n = rnd.choice(live), rnd.randint(1, 3)
            if n > cache.n_free_slots:
                before = cache.live_slots()
                with pytest.raises(CacheError):
                    cache.fork(s, n)
                assert before == cache.live_slots()
                continue
            for c in cache.fork(s, n):
                text[c] = list(text[s])
                assert (cache.state_groups[0].data[:, c] == cache.state_groups[0].data[:, s]).all() and cache.length(c) == cache.length(s)
        elif do < 0.55 and live:
            s = rnd.choice(live)
            cache.free_slot(s)
            del text[s]
        elif live:
            some = rnd.sample(live, rnd.randint(1, len(live)))
            new = [rnd.choice([1, 1, 1, 2, 5, 11]) for _ in some]
            some, new = zip(*[(s, n) for s, n in zip(some, new) if len(text[s]) + n <= 90] or [(None, 0)])
            if some[0] is None:
                continue
            try:
                cache.reserve(some, new)
            except CacheError:
                for s in cache.live_slots():
                    sees(s, len(text[s]), len(text[s]))          # nothing has changed
                continue
            for s in some:
                sees(s, len(text[s]), len(text[s]))              # what the step's first query reads, before anything is written
            for s, n in zip(some, new):
                values = [counter[0] + i + 1 for i in range(n)]
                counter[0] += n
                for gi in range(len(cache.kv_groups)):
                    write(cache, gi, s, len(text[s]), values)
                text[s] += values
            cache.advance(some, new)
        for s in cache.live_slots():
            sees(s, len(text[s]), len(text[s]))
    assert copies[0] > 5
    for g in cache.kv_groups:
        assert g.pool.n_shared == sum(g.pool.holders(p) > 1 for p in range(g.pool.n_pages))
    for s in cache.live_slots():
        cache.free_slot(s)
    assert all(g.pool.n_free == g.pool.n_pages and g.pool.n_shared == 0 for g in cache.kv_groups)


def test_only_what_a_slot_still_sees_is_copied(monkeypatch):
    scoring_refs.install(monkeypatch)
    calls = []
    monkeypatch.setattr(ops, "copy_rows", lambda moves: calls.append([(list(s), list(d)) for _, s, d in moves]))
    cache = Cache([RunNeeds(KVRequirement(1, 1))], max_tokens=200, max_seqs=4, page_size=PAGE, dtype=torch.float32, device="cpu")
    s = cache.alloc_slot()
    cache.reserve([s], [8]); cache.advance([s], [8])          # two whole pages
    free = cache.kv_groups[0].pool.n_free
    a, b = cache.fork(s, 2)
    assert cache.kv_groups[0].pool.n_free == free and not calls               # nothing is taken or copied (and there is no state)
    cache.reserve([s, a, b], [1, 1, 1]); cache.advance([s, a, b], [1, 1, 1])
    assert not calls and cache.kv_groups[0].pool.n_free == free - 3           # new pages, the prompt's two stay shared
    c, = cache.fork(a)
    cache.reserve([a, c], [1, 1])
    page = cache.kv_groups[0].pages[c][2]
    assert [len(m) for m in calls] == [2] and calls[0][0] == calls[0][1]      # keys and values of one page
    assert calls[0][0] == ([page], [cache.kv_groups[0].pages[a][2]]) and cache.kv_groups[0].pool.n_free == free - 4
    cache.free_slot(s); cache.free_slot(b); cache.free_slot(a)
    assert cache.kv_groups[0].pool.n_free == cache.kv_groups[0].pool.n_pages - 3


def test_a_failed_copy_leaves_the_cache_as_it_was(monkeypatch):
    def fail(moves):
        raise KernelError("no")
    monkeypatch.setattr(ops, "copy_rows", fail)
    cache = Cache([RunNeeds(KVRequirement(1, 1), StateRequirement((2,)))], max_tokens=64, max_seqs=4, page_size=PAGE, dtype=torch.float32, device="cpu")
    s = cache.alloc_slot()
    cache.reserve([s], [2]); cache.advance([s], [2])
    with pytest.raises(KernelError):
        cache.fork(s)
    assert cache.live_slots() == [s] and cache.n_free_slots == 3 and cache.kv_groups[0].pool.holders(cache.kv_groups[0].pages[s][0]) == 1
    cache.state_groups[0].data = None
    t, = cache.fork(s)
    before = {k: list(v) for k, v in cache.kv_groups[0].pages.items()}
    free = cache.kv_groups[0].pool.n_free
    with pytest.raises(KernelError):
        cache.reserve([s, t], [1, 1])
    assert before == cache.kv_groups[0].pages and free == cache.kv_groups[0].pool.n_free


def test_what_a_fork_refuses(monkeypatch):
    scoring_refs.install(monkeypatch)
    cache = Cache([RunNeeds(KVRequirement(1, 1))], max_tokens=8, max_seqs=4, page_size=PAGE, dtype=torch.float32, device="cpu")
    with pytest.raises(CacheError):
        cache.fork(0)
    s = cache.alloc_slot()
    cache.reserve([s], [7]); cache.advance([s], [7])
    with pytest.raises(CacheError):
        cache.fork(s, 4)
    with pytest.raises(CacheError):
        cache.fork(s, -1)
    assert cache.fork(s, 0) == []
    t, = cache.fork(s)
    with pytest.raises(CacheError, match="cache is full"):     # the shared page would have to become two, both pages are held
        cache.reserve([s, t], [1, 1])
    cache.free_slot(t)
    cache.reserve([s], [1])


# ---- the engine over the plain kernels ----

@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_forked_sequences_equal_plain(tmp_path, monkeypatch, name):
    engine, cfg, w = build(tmp_path, name, monkeypatch)
    scoring_refs.install(monkeypatch)
    rng = np.random.default_rng(11)
    V = cfg["vocab_size"]
    head = prompt(rng, 22, V)                          # past both windows, in the middle of a page
    tails = [prompt(rng, n, V) for n in (9, 17, 6)]
    want = [plain.forward(cfg, w, head + t) for t in tails]
    first = engine.new_sequence()
    engine.step([first], [head], "last")
    slots = [first] + engine.fork(first, 2)
    close(engine.step(slots, [t[:1] for t in tails], "last"), np.stack([x[22] for x in want]))
    engine.step(slots[:2], [tails[0][1:4], tails[1][1:8]], "last")                    # several tokens at once, while the third waits
    again, = engine.fork(slots[1])
    close(engine.step([slots[0], slots[1], slots[2]], [tails[0][4:], tails[1][8:], tails[2][1:]], "last"), np.stack([x[-1] for x in want]))
    close(engine.step([again], [tails[1][8:]], "all"), want[1][22 + 8:])              # and the fork of a fork
    for s in slots + [again]:
        engine.release(s)
    assert all(g.pool.n_free == g.pool.n_pages for g in engine.cache.kv_groups)


def log_p(cfg, w, ids):
    z = plain.forward(cfg, w, ids)
    z = z - z.max(axis=1, keepdims=True)
    return z - np.log(np.exp(z).sum(axis=1, keepdims=True))


def test_scored_texts_equal_plain(tmp_path, monkeypatch):
    engine, cfg, w = build(tmp_path, "A", monkeypatch, max_tokens=64, max_seqs=2)      # small: several batches
    scoring_refs.install(monkeypatch)
    rng = np.random.default_rng(12)
    texts = [prompt(rng, n, cfg["vocab_size"]) for n in (30, 1, 9, 2, 40, 17)]
    for r, ids in zip(score(engine, texts, top=3), texts):
        p = log_p(cfg, w, ids)
        assert len(r.logprobs) == len(r.entropy) == len(r.top) == len(ids) - 1
        for i, t in enumerate(ids[1:]):
            assert abs(r.logprobs[i] - p[i, t]) < 1e-4 and abs(r.entropy[i] + (np.exp(p[i]) * p[i]).sum()) < 1e-4
            assert [k for k, _ in r.top[i]] == np.argsort(-p[i], kind="stable")[:3].tolist()
            assert all(abs(v - p[i, k]) < 1e-4 for k, v in r.top[i])
        assert abs(r.perplexity - np.exp(-np.mean([p[i, t] for i, t in enumerate(ids[1:])] or [0]))) < 1e-3
    assert engine.cache.n_free_slots == 2
    # in portions: the first token of the second portion is what follows the first
    ids = texts[0]
    slot = engine.new_sequence()
    a = engine.score([slot], [ids[:10]], following=[ids[10]])
    b = engine.score([slot], [np.array(ids[10:])])
    got = torch.cat([a.logprobs, b.logprobs]).numpy()
    assert np.abs(got - [log_p(cfg, w, ids)[i, t] for i, t in enumerate(ids[1:])]).max() < 1e-4
    engine.release(slot)


def test_scoring_refusals(tmp_path, monkeypatch):
    engine, cfg, w = build(tmp_path, "A", monkeypatch)
    scoring_refs.install(monkeypatch)
    s = engine.new_sequence()
    for kw in (dict(tokens=[[1, 2]], following=[1, 2]), dict(tokens=[[1, 2]], following=[cfg["vocab_size"]]), dict(tokens=[[1, -2]]),
               dict(tokens=[[1, 2]], top=33), dict(tokens=[[1, 2]], top=-1), dict(tokens=[[1, 2]], top=True), dict(tokens=[[1, 2.5]]),
               dict(tokens=[[]]), dict(tokens=[[1], [2]]), dict(tokens=[[1, 2]], following=[2.5]), dict(tokens=[[1, 2]], following=[[2, 3]])):
        with pytest.raises(StepError):
            engine.score([s], **kw)
    assert engine.length(s) == 0
    with pytest.raises(ValueError):
        score(engine, [[]])
    assert score(engine, []) == []


def test_ids_of_different_whole_types(tmp_path, monkeypatch):
    engine, cfg, w = build(tmp_path, "A", monkeypatch)
    scoring_refs.install(monkeypatch)
    a, b = engine.new_sequence(), engine.new_sequence()
    got = engine.score([a, b], [np.array([5, 6, 7], dtype=np.uint64), np.array([8, 9], dtype=np.int8)], following=[3, np.uint64(4)])
    c, d = engine.new_sequence(), engine.new_sequence()
    want = engine.score([c, d], [[5, 6, 7], [8, 9]], following=[3, 4])
    assert got.logprobs.shape == (5,) and torch.equal(got.logprobs, want.logprobs)


@pytest.mark.parametrize("name", ["A", "B"])
def test_several_continuations_equal_as_many_requests(tmp_path, monkeypatch, name):
    engine, cfg, w = build(tmp_path, name, monkeypatch, max_tokens=512, max_seqs=6)
    scoring_refs.install(monkeypatch)
    rng = np.random.default_rng(13)
    prompts = [prompt(rng, n, cfg["vocab_size"]) for n in (5, 18, 7)]
    for options in (dict(temperature=0.9, seed=3), dict(temperature=1.1, top_k=20, repetition_penalty=1.3, seed=4), dict(temperature=0.0)):
        sampling = SamplingParams(**options)
        got = generate(engine, prompts, max_new_tokens=9, sampling=sampling, stop_token_ids=[3, 77], samples=3, logprobs=2)
        alone = generate(engine, [p for p in prompts for _ in range(3)], max_new_tokens=9, sampling=sampling, stop_token_ids=[3, 77])
        assert [r.tokens for r in got] == [r.tokens for r in alone] and [r.finish_reason for r in got] == [r.finish_reason for r in alone]
        for i, r in enumerate(got):
            ids = prompts[i // 3] + r.tokens
            p, n = log_p(cfg, w, ids), len(prompts[i // 3])
            assert len(r.logprobs) == len(r.tokens) == len(r.entropy) == len(r.top)
            for k, t in enumerate(r.tokens):
                assert abs(r.logprobs[k] - p[n + k - 1, t]) < 1e-4 and r.top[k][0][0] == int(p[n + k - 1].argmax())
        assert alone[0].logprobs is None and alone[0].top is None
        assert engine.cache.n_free_slots == 6 and all(g.pool.n_free == g.pool.n_pages for g in engine.cache.kv_groups)


def test_a_stop_token_that_is_kept_has_its_log_probability(tmp_path, monkeypatch):
    engine, cfg, w = build(tmp_path, "A", monkeypatch)
    scoring_refs.install(monkeypatch)
    ids = prompt(np.random.default_rng(14), 6, cfg["vocab_size"])
    free = generate(engine, [ids], max_new_tokens=5, sampling=SamplingParams(0.0), stop_token_ids=[])[0].tokens
    for keep in (True, False):
        r = generate(engine, [ids], max_new_tokens=5, sampling=SamplingParams(0.0), stop_token_ids=[free[-1]], include_stop=keep, logprobs=0)[0]
        assert len(r.logprobs) == len(r.tokens) and r.top == [[]] * len(r.tokens)


def test_options_of_the_entry_point(tmp_path, monkeypatch):
    engine, cfg, w = build(tmp_path, "A", monkeypatch)
    scoring_refs.install(monkeypatch)
    gen = Generator(engine.model, max_batch=4, max_context=64, use_graphs=False).with_temperature(0.0).with_logprobs(2).with_bos_token(2)
    r = gen.generate_batch_results([[5, 6]], 4, samples=2)
    assert len(r) == 2 and r[0] == r[1] and len(r[0].logprobs) == len(r[0].tokens)
    assert gen.generate_several([5, 6], 3, 4) == [[2, 5, 6] + r[0].tokens] * 3
    text = gen.score([[5, 6] + r[0].tokens], 2)[0]
    assert np.allclose(text.logprobs[2:], r[0].logprobs, atol=1e-4) and len(text.logprobs) == 2 + len(r[0].tokens)
    assert gen.generate_batch_results([[5]], 0, samples=2)[1].logprobs == []
    assert gen.with_logprobs(None).generate_batch_results([[5]], 1)[0].logprobs is None
    for bad in (dict(samples=0), dict(samples=5), dict(samples=True)):
        with pytest.raises(ValueError):
            gen.generate_batch_results([[5]], 1, **bad)
    with pytest.raises(ValueError):
        gen.with_logprobs(33).generate_batch_results([[5]], 1)


def test_batches_of_requests_with_several_continuations():
    kw = dict(max_seqs=6, max_tokens=640, page_size=64, max_context=256)
    assert plan_batches([5, 5, 5], 8, samples=3, **kw) == [[0, 1], [2]]
    assert plan_batches([130, 130], 62, samples=5, prompt_shared=True, **kw) == [[0], [1]]              # 128 + 5 * 64
    assert plan_batches([130, 130], 62, samples=3, prompt_shared=True, **kw) == [[0, 1]]                # 2 * (128 + 3 * 64)
    with pytest.raises(ValueError):
        plan_batches([130], 62, samples=4, **kw)                                                        # 4 * 192, not shared
    with pytest.raises(ValueError):
        plan_batches([5], 8, samples=7, **kw)


def test_batches_of_continuations_where_some_layers_keep_a_window():
    kw = dict(max_seqs=8, max_tokens=640, page_size=64, max_context=512, samples=4, prompt_shared=True)
    assert plan_batches([400, 400], 40, rings=[(128, 1024)], **kw) == [[0], [1]]                        # 384 + 4 * 64 fill the pages that are shared
    assert plan_batches([130, 130], 20, rings=[(128, 1024)], **kw) == [[0], [1]]                        # 2 * (128 + 4 * 64) do not fit
    assert plan_batches([30, 30], 20, rings=[(128, 1024)], **kw) == [[0, 1]]
    assert plan_batches([30, 30], 20, rings=[(128, 1024), (64, 448)], **kw) == [[0], [1]]               # 2 * 4 * 64 of 448
    with pytest.raises(ValueError):
        plan_batches([400], 40, rings=[(128, 511)], **kw)


@pytest.mark.parametrize("name,n,samples", [("A", 40, 5), ("B", 40, 5)])
def test_continuations_that_fit_only_as_they_share_a_prompt(tmp_path, monkeypatch, name, n, samples):
    """A cache with room for the prompt once and a page or two of each continuation, and for every continuation's window."""
    engine, cfg, w = build(tmp_path, name, monkeypatch, page_size=8, max_tokens=(n // 8 * 8) + samples * 16, max_seqs=samples)
    scoring_refs.install(monkeypatch)
    assert any(g.is_ring for g in engine.cache.kv_groups)
    ids = prompt(np.random.default_rng(15), n, cfg["vocab_size"])
    sampling = SamplingParams(temperature=0.9, seed=5)
    got = generate(engine, [ids], max_new_tokens=14, sampling=sampling, stop_token_ids=[], samples=samples)
    roomy, _, _ = build(tmp_path, name, monkeypatch, page_size=8, max_tokens=1024, max_seqs=samples)
    scoring_refs.install(monkeypatch)
    want = generate(roomy, [ids] * samples, max_new_tokens=14, sampling=sampling, stop_token_ids=[])
    assert [r.tokens for r in got] == [r.tokens for r in want]
    assert all(g.pool.n_free == g.pool.n_pages for g in engine.cache.kv_groups)


def test_a_dropped_engine_waits_for_its_uploads(tmp_path, monkeypatch):
    engine, cfg, w = build(tmp_path, "A", monkeypatch)
    waited = []

    class Event:
        def __init__(self, fails=False):
            self.fails = fails

        def synchronize(self):
            waited.append(self)
            if self.fails:
                raise RuntimeError("the context is gone")
    engine._pinned_event = [Event(True), Event()]
    del engine
    assert len(waited) == 2


def test_status_words_nobody_can_vouch_for_are_kept(monkeypatch):
    from rust_deeplearning_b200.engine import step

    class Event:
        def __init__(self, answer):
            self.answer = answer

        def query(self):
            if self.answer is None:
                raise RuntimeError("the event was captured")
            return self.answer
    kept = {1: ("a", Event(False)), 3: ("b", None), 4: ("c", Event(None))}
    monkeypatch.setattr(step, "_retired", {**kept, 2: ("d", Event(True))})
    step._release_retired()
    assert step._retired == kept


def test_an_engine_dropped_while_status_words_are_gone_through(monkeypatch):
    from rust_deeplearning_b200.engine import step

    class Event:
        def query(self):
            step._retired[9] = ("another engine's", None)      # as the collector may do at any time
            return True
    monkeypatch.setattr(step, "_retired", {1: ("a", Event()), 2: ("b", Event())})
    step._release_retired()
    assert step._retired == {9: ("another engine's", None)}


def test_perplexity():
    from rust_deeplearning_b200 import ScoredText
    inf = float("inf")
    assert ScoredText([], [], []).perplexity == 1.0 and abs(ScoredText([-1.0, -3.0], [], []).perplexity - np.exp(2)) < 1e-9
    assert ScoredText([-inf, -1.0], [], []).perplexity == inf and ScoredText([-1e4], [], []).perplexity == inf


# ---- refusals that need no device ----

def test_refused_copies():
    t = torch.zeros((2, 6, 4, 5))
    for moves in ([(t, [0, 1], [2])], [(t, [0, 1], [2, 2])], [(t, [0, 1], [1, 2])], [(t, [0], [6])], [(t, [6], [0])], [(t, [0], [-1])], [(t, [-1], [0])],
                  [(t[0, 0, 0], [0], [1])], [(t.transpose(2, 3), [0], [1])], [(t[..., ::2], [0], [1])],
                  [(t[:, :1].expand(2, 6, 4, 5), [0], [1])], [(t[:1].expand(3, 6, 4, 5), [0], [1])],
                  [(t, [0], [1]), (t, [2], [3])], [(t[:, :4], [0], [1]), (t[:, 3:], [0], [1])],
                  [(torch.zeros((1, 3, 4)).as_strided((1, 3, 4), (12, 2, 1)), [0], [1])],
                  [(torch.zeros((1, 2, 3)), [0], [1])] * 65):
        with pytest.raises(KernelError):
            ops.copy_rows(moves)
    with pytest.raises(TypeError):
        ops.copy_rows([(t, [0.0], [1.0])])
    with pytest.raises(KernelError, match="CUDA"):
        ops.copy_rows([(t, [0], [1])])
    assert not t.any()


def test_rows_that_no_launch_has_blocks_for_are_refused_before_anything_is_copied():
    import ctypes
    from rust_deeplearning_b200.kernels import library
    pack = ops._copy_tensor
    fine, large = pack(256, 64, 64, 64, 1, 0, 1, 0), pack(4096, 1 << 20, 1 << 20, 65536, 2 ** 31 - 1, 0, 1, 0)
    pairs = (ctypes.c_int * 2)(0, 1)
    for tensors in ([large], [fine, large]):
        with pytest.raises(KernelError, match="no blocks"):
            library.check(library.load().rdl_copy_rows(b"".join(tensors), len(tensors), ctypes.addressof(pairs), None))


def test_refused_scoring_calls():
    z = torch.zeros((3, 10))
    ids = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: ops.token_logprobs(z[0]), lambda: ops.token_logprobs(z.t()), lambda: ops.token_logprobs(z.double()),
                 lambda: ops.token_logprobs(z, ids.long()), lambda: ops.token_logprobs(z, ids[:2]), lambda: ops.token_logprobs(z, ids.repeat(2)[::2]),
                 lambda: ops.token_logprobs(z, None, 11), lambda: ops.token_logprobs(z, None, -1), lambda: ops.token_logprobs(z, None, True),
                 lambda: ops.token_logprobs(z, None, 1.0), lambda: ops.token_logprobs(torch.zeros((3, 50)), None, 33), lambda: ops.token_logprobs(z[:, :0]),
                 lambda: ops.linear_logprobs(z, torch.zeros((5, 9))), lambda: ops.linear_logprobs(z, torch.zeros((5, 10), dtype=torch.bfloat16)),
                 lambda: ops.linear_logprobs(z, torch.zeros((5, 10)), ids, 6), lambda: ops.linear_logprobs(z, torch.zeros((5, 10)), softcap=0.0),
                 lambda: ops.linear_logprobs(z, torch.zeros((10, 5)).t()), lambda: ops.linear_logprobs(z.t(), torch.zeros((5, 3))),
                 lambda: ops.linear_logprobs(z[0], torch.zeros((5, 10))), lambda: ops.linear_logprobs(z[:, :0], torch.zeros((5, 0))),
                 lambda: ops.linear_logprobs(z.half(), torch.zeros((5, 10)).half())):
        with pytest.raises(KernelError):
            call()
    for call in (lambda: ops.token_logprobs(z, ids, 2), lambda: ops.linear_logprobs(z, torch.zeros((5, 10)), ids, 2)):
        with pytest.raises(KernelError, match="CUDA"):
            call()


@pytest.mark.parametrize("kw", [dict(softcap=float("inf")), dict(softcap=float("nan")), dict(softcap=1e39), dict(softcap=1e-40), dict(softcap=-30.0),
                                dict(scale=float("inf")), dict(scale=float("nan")), dict(scale=1e39)])
def test_numbers_that_float32_does_not_hold_are_refused(kw):
    with pytest.raises(KernelError, match="float32"):
        ops.linear_logprobs(torch.zeros((3, 10)), torch.zeros((5, 10)), None, 2, **kw)


def test_command_line_refusals():
    from rust_deeplearning_b200.cli import main
    for more in (["--stream", "--logprobs", "1"], ["--stream", "--score"], ["--score", "--samples", "2"]):
        with pytest.raises(SystemExit):
            main(["nowhere", "--prompt-ids", "1", *more])
