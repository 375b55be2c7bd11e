"""Forked sequences, several continuations and scored texts with every architecture on the GPU."""
import numpy as np
import pytest
import torch

import model_helpers as mh
import plain_gemma2 as plain
import tiny_configs, tiny_dokulorn, tiny_gasetar, tiny_kitonex, tiny_ligirax, tiny_paditar, tiny_revepel
from rust_deeplearning_b200 import Engine, Generator, random_model
from test_cli_gpu import run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MODELS = [(tiny_configs, "A"), (tiny_configs, "D"), (tiny_ligirax, "LA"), (tiny_ligirax, "LC"), (tiny_dokulorn, "DA"), (tiny_dokulorn, "DC"),
          (tiny_revepel, "RA"), (tiny_revepel, "RC"), (tiny_gasetar, "GA"), (tiny_gasetar, "GB"), (tiny_kitonex, "KA"), (tiny_kitonex, "KB"),
          (tiny_paditar, "PA"), (tiny_paditar, "PC")]


def ids_of(seed, n, vocab):
    return [int(t) for t in np.random.default_rng(seed).integers(0, vocab, size=n)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("module,name", MODELS, ids=[n for _, n in MODELS])
def test_forked_sequences_equal_separate_ones(module, name, dtype):
    """A prompt forked three ways against three sequences that ran the prompt alone: the same steps behind it, the same logits bit for bit (what
    pages a sequence's keys lie in, and whose they were before, changes nothing)."""
    cfg, seed = module.config(name)
    model = random_model(cfg, seed, dtype)
    V = model.vocab_size
    head, tails = ids_of(1, 77, V), [ids_of(2 + i, 40, V) for i in range(4)]
    got = []
    for forked in (True, False):
        eng = Engine(model, max_tokens=4096, max_seqs=6, max_context=256, page_size=16)
        out = []
        if forked:
            first = eng.new_sequence()
            eng.step([first], [head], "last")
            a, b = eng.fork(first, 2)
            slots = [first, a, b]
        else:
            slots = []
            for _ in range(3):
                slots.append(eng.new_sequence())
                eng.step([slots[-1]], [head], "last")
        for t in range(5):                                               # single tokens (the later ones in a graph)
            out.append(eng.step(slots, [[x[t]] for x in tails[:3]], "last").clone())
        out.append(eng.step(slots[:1], [tails[0][5:25]], "last").clone())          # one goes on by many tokens
        if forked:
            slots += eng.fork(slots[0])
        else:
            fourth = eng.new_sequence()
            eng.step([fourth], [head], "last")
            for t in range(5):
                eng.step([fourth], [[tails[0][t]]], "last")
            slots.append(fourth)
            eng.step([fourth], [tails[0][5:25]], "last")
        for t in range(25, 40):                                          # the fourth one's logits are compared where its past came in the same steps
            out.append(eng.step(slots, [[x[t]] for x in tails], "last")[:3].clone())
        torch.cuda.synchronize()
        eng.check_status()
        for s in slots:
            eng.release(s)
        assert all(g.pool.n_free == g.pool.n_pages for g in eng.cache.kv_groups)
        got.append(out)
    for i, (x, y) in enumerate(zip(*got)):
        assert torch.isfinite(x).all() and torch.equal(x, y), f"step {i}"


def test_an_engine_dropped_with_steps_in_flight():
    """The next engine's pinned buffers are the last one's: its first description must not reach a kernel of the last one's steps."""
    cfg, seed = tiny_configs.config("A")
    model = random_model(cfg, seed, "float32")
    ids = ids_of(60, 40, model.vocab_size)

    def steps(n):
        eng = Engine(model, max_tokens=512, max_seqs=2, max_context=128)
        a, b = eng.new_sequence(), eng.new_sequence()
        eng.step([a, b], [ids[:9], ids[9:13]], "last")
        out = [eng.step([a, b], [[ids[t]], [ids[-t]]], "last").clone() for t in range(1, n)]
        return out                                           # the engine is gone, its steps may not be

    want = steps(30)
    torch.cuda.synchronize()
    want = [w.clone() for w in want]
    for _ in range(5):
        torch.cuda._sleep(20_000_000)                        # ten milliseconds: the host is ahead by all of the steps
        runs = [steps(30), steps(7)]
        torch.cuda.synchronize()
        for got in runs:
            assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_the_status_word_of_a_dropped_engine_is_nobody_elses():
    """Kernels that are still to run may report to it: it stays out of the allocator's hands until the engine's last step is over."""
    from rust_deeplearning_b200.engine import step
    cfg, seed = tiny_configs.config("A")
    model = random_model(cfg, seed, "float32")
    ids = ids_of(61, 9, model.vocab_size)
    Engine(model, max_tokens=64)                             # whatever earlier engines left is released
    for side in (False, True):
        stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            eng = Engine(model, max_tokens=64)
            eng.step([eng.new_sequence()], [ids], "last")
            word = eng.status.data_ptr()
            torch.cuda._sleep(200_000_000)                   # stands for what is left of the step: a tenth of a second
        del eng
        held = [torch.zeros(1, dtype=torch.int32).pin_memory() for _ in range(20)]
        assert all(t.data_ptr() != word for t in held) and word in step._retired
        torch.cuda.synchronize()
        del held
        other = Engine(model, max_tokens=64)
        assert word not in step._retired
        other.check_status()


def log_p(z):
    z = z.double().cpu().numpy()
    z = z - z.max(axis=1, keepdims=True)
    return z - np.log(np.exp(z).sum(axis=1, keepdims=True))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("module,name", MODELS, ids=[n for _, n in MODELS])
def test_scores_are_those_of_the_logits(module, name, dtype):
    """`Engine.score` against the log softmax of `Engine.step`'s logits over the same texts.  Both heads multiply the same rows: sums of up to 192
    products in float, so the logits agree to 192 * 2^-23 of their magnitudes' sum; 2^-10 of the largest logit holds that many times over."""
    cfg, seed = module.config(name)
    model = random_model(cfg, seed, dtype)
    V = model.vocab_size
    texts = [ids_of(20 + i, n, V) for i, n in enumerate((90, 3, 1, 40, 33))]
    eng = Engine(model, max_tokens=2048, max_seqs=8, page_size=16)
    slots = [eng.new_sequence() for _ in texts]
    z = eng.step(slots, texts, [list(range(len(t) - 1)) for t in texts])
    want = log_p(z)
    for s in slots:
        eng.release(s)
    slots = [eng.new_sequence() for _ in texts]
    r = eng.score(slots, texts, top=4)
    eng.check_status()
    tol = 2.0 ** -10 * (float(z.abs().max()) + 1)
    targets = [t for x in texts for t in x[1:]]
    assert np.abs(r.logprobs.cpu().numpy() - want[np.arange(len(targets)), targets]).max() <= tol
    assert np.abs(r.entropy.cpu().numpy() + (np.exp(want) * want).sum(1)).max() <= 2 * tol
    assert np.abs(r.top_logprobs.cpu().numpy() - -np.sort(-want, axis=1)[:, :4]).max() <= tol
    # one token behind each text, single tokens
    nxt = [[5 % V] for _ in texts]
    one = eng.score(slots, nxt, following=[t[0] for t in texts], top=1)
    assert one.logprobs.shape == (5,) and torch.isfinite(one.logprobs).all()
    assert eng.score(slots, nxt).entropy.shape == (0,)
    for s in slots:
        eng.release(s)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_continuations_with_log_probabilities(dtype):
    name = "A"
    cfg, w = mh.plain_model(name)
    model = mh.loaded_model(name, dtype)
    V = model.vocab_size
    prompts = [mh.prompt(900, 21, V), mh.prompt(901, 6, V)]
    gen = Generator(model, max_batch=8, max_context=128).with_temperature(1.0).with_seed(5).with_stop_tokens([]).with_logprobs(3)
    got = gen.generate_batch_results(prompts, 12, samples=4)
    assert len(got) == 8 and len({tuple(r.tokens) for r in got[:4]}) > 1
    for i, r in enumerate(got):
        ids = prompts[i // 4] + r.tokens
        z = plain.forward(cfg, w, ids)
        z = z - z.max(axis=1, keepdims=True)
        p = z - np.log(np.exp(z).sum(axis=1, keepdims=True))
        n = len(prompts[i // 4])
        lp = np.array([p[n + k - 1, t] for k, t in enumerate(r.tokens)])
        assert np.abs(np.array(r.logprobs) - lp).max() <= 2 * mh.tolerance(dtype, z)
        assert all(len(t) == 3 for t in r.top)
    if dtype == "float32":
        alone = gen.generate_batch_results([prompts[0]] * 4 + [prompts[1]] * 4, 12)
        assert [r.tokens for r in alone] == [r.tokens for r in got]
    scored = gen.score([prompts[i // 4] + r.tokens for i, r in enumerate(got)])
    for s, r in zip(scored, got):
        assert np.abs(np.array(s.logprobs[-12:]) - np.array(r.logprobs)).max() <= 4 * mh.tolerance(dtype, z)


@pytest.mark.parametrize("weights", ["mx4", "mx4+head"])
def test_scores_with_4_bit_weights(weights):
    cfg, seed = tiny_configs.config("D")
    model = random_model(cfg, seed, "bfloat16", weight_format=weights)
    eng = Engine(model, max_tokens=1024, max_seqs=4)
    texts = [ids_of(40 + i, n, model.vocab_size) for i, n in enumerate((50, 9))]
    a = [eng.new_sequence() for _ in texts]
    want = log_p(eng.step(a, texts, [list(range(len(t) - 1)) for t in texts]))
    b = [eng.new_sequence() for _ in texts]
    r = eng.score(b, texts, top=2)
    targets = [t for x in texts for t in x[1:]]
    assert np.abs(r.logprobs.cpu().numpy() - want[np.arange(len(targets)), targets]).max() <= 1e-3


def test_the_command_line(tmp_path):
    folder = mh.model_folder("A")
    ids = mh.prompt(902, 9, mh.loaded_model("A", "float32").vocab_size)
    base = [folder, "--prompt-ids", ",".join(map(str, ids)), "--dtype", "float32", "--max-context", "128"]
    out, err = run(base + ["--score", "--logprobs", "2"])
    lines = [line.split("\t") for line in out.strip().split("\n")]
    want = Generator(mh.loaded_model("A", "float32"), max_batch=1, max_context=128).score([ids], 2)[0]
    assert [int(line[0]) for line in lines] == ids[1:] and "perplexity" in err
    assert np.allclose([float(line[1]) for line in lines], want.logprobs, atol=2e-6) and all(len(line) == 5 for line in lines)
    out, err = run(base + ["--samples", "3", "--max-tokens", "4", "--temperature", "0", "--logprobs", "1"])
    lines = out.strip().split("\n")
    assert len(lines) == 3 * 5 and lines[:5] == lines[5:10] == lines[10:] and [line.split("\t")[0] for line in lines[1:5]] == lines[0].split()
    assert "continuation 2" in err
