"""Log probabilities of tokens and copies of a cache's rows on the GPU, against float64 (tests/scoring_refs.py, where the tolerances are derived)."""
import numpy as np
import pytest
import torch

import scoring_refs as ref
from rust_deeplearning_b200.kernels import library, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def logits_of(rows, vocab, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn((rows, vocab), generator=g) * spread
    z *= torch.exp2(torch.arange(rows).float() % 4 - 1)[:, None]        # flat rows and nearly certain ones
    return z.to(dtype).to(DEV)


def targets_of(rows, vocab, seed):
    return torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).to(DEV)


def f64(t):
    return t.detach().double().cpu().numpy()


# ---- rows of logits ----

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 2), (3, 3, 0), (2, 7, 7), (5, 31, 31), (4, 32, 32), (6, 33, 20), (9, 1003, 3),
                                            (333, 777, 5), (2, 4096, 32), (16, 8191, 1), (3, 50001, 20), (2, 256000, 20), (150, 12345, 4), (2000, 130, 8)])
def test_rows_of_logits(rows, vocab, top, dtype):
    z = logits_of(rows, vocab, dtype, rows + vocab)
    t = targets_of(rows, vocab, 1)
    ref.check(ops.token_logprobs(z, t, top), f64(z), t.cpu().numpy(), top, f"{rows} x {vocab}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [1, 2, 3, 5, 8])
def test_rows_that_start_anywhere_and_lie_apart(dtype, offset):
    wide = logits_of(5, 2500, dtype, 3)
    z = wide[:, offset:offset + 2111]
    t = targets_of(5, 2111, 2)
    ref.check(ops.token_logprobs(z, t, 7), f64(z), t.cpu().numpy(), 7, f"columns from {offset}")
    same = wide[:1, offset:].expand(4, -1)                               # one row four times
    r = ops.token_logprobs(same, None, 3)
    ref.check(r, f64(same), None, 3, "one row four times")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_ties_infinities_and_nan(dtype):
    vocab = 3001
    z = logits_of(13, vocab, dtype, 9)
    lowest = torch.finfo(dtype).min
    z[0, ::2] = -float("inf")                        # half of the tokens forbidden
    z[1] = -float("inf"); z[1, 1234] = -5.0          # all but one
    z[2] = -float("inf")                             # all: no distribution
    z[3] = lowest                                    # masked with the lowest value: uniform
    z[4] = lowest; z[4, 17] = 2.0
    z[5] = 1.25                                      # all equal: the lowest ids first
    z[6] = 0.0; z[6, 1::2] = -0.0                    # one value
    z[7, 2000] = float("nan")
    z[8, 100] = float("inf")
    z[9] = float("nan")
    z[10] = torch.arange(vocab, device=DEV).to(dtype)               # rising: every logit enters the list for a while (equal ones in bfloat16)
    z[11] = -torch.arange(vocab, device=DEV).to(dtype)
    z[12] = float("nan"); z[12, 5] = 1.0; z[12, 3] = -float("inf")
    t = torch.tensor([1, 1234, 0, 5, 17, 3000, 3, 4, 100, 0, 3000, 2999, 5], dtype=torch.int32, device=DEV)
    for top in (0, 1, 20, 32):
        ref.check(ops.token_logprobs(z, t, top), f64(z), t.cpu().numpy(), top, f"masks, {top} alternatives")
    forbidden = torch.full((13,), 0, dtype=torch.int32, device=DEV)
    assert ops.token_logprobs(z, forbidden, 0).logprobs[1].item() == -float("inf")


def test_tokens_that_are_none_or_outside_the_vocabulary():
    z = logits_of(4, 100, torch.float32, 4)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    t = torch.tensor([-1, 99, -100, 0], dtype=torch.int32, device=DEV)
    ref.check(ops.token_logprobs(z, t, 2, status=status), f64(z), t.cpu().numpy(), 2, "no token asked for")
    assert status.item() == 0
    t = torch.tensor([5, 100, 2 ** 31 - 1, 0], dtype=torch.int32, device=DEV)
    r = ops.token_logprobs(z, t, 2, status=status)
    assert torch.isnan(r.logprobs).tolist() == [False, True, True, False] and torch.isfinite(r.entropy).all()
    assert "token_logprobs" in library.FAULTS[status.item()]
    x, w = torch.ones((4, 64), device=DEV), torch.ones((100, 64), device=DEV)
    status.zero_()
    r = ops.linear_logprobs(x, w, t, status=status)
    assert torch.isnan(r.logprobs).tolist() == [False, True, True, False] and status.item() == 11


def test_no_rows():
    r = ops.token_logprobs(torch.empty((0, 50), device=DEV), torch.empty(0, dtype=torch.int32, device=DEV), 3)
    assert r.logprobs.shape == (0,) and r.entropy.shape == (0,) and r.top_ids.shape == (0, 3) and r.top_logprobs.shape == (0, 3)
    r = ops.linear_logprobs(torch.empty((0, 64), device=DEV), torch.ones((50, 64), device=DEV), None, 3)
    assert r.logprobs is None and r.top_ids.shape == (0, 3)


def test_offsets_beyond_32_bits():
    rows, vocab = 8600, 256000                           # 2.2e9 logits
    z = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=DEV)
    z[-1] = logits_of(1, vocab, torch.bfloat16, 6)[0]
    z[-2, 77] = 3.0
    t = torch.full((rows,), 77, dtype=torch.int32, device=DEV)
    r = ops.token_logprobs(z, t, 3)
    last = ops.TokenLogprobs(*(v[-2:] for v in r))
    ref.check(last, f64(z[-2:]), [77, 77], 3, "the last rows")
    assert (r.top_ids[:-2] == torch.arange(3, device=DEV)).all() and torch.allclose(r.entropy[:-2], torch.tensor(float(np.log(vocab)), device=DEV))


def test_a_row_does_not_depend_on_the_others_and_calls_repeat():
    z = logits_of(40, 9001, torch.float32, 8)
    t = targets_of(40, 9001, 8)
    a, b = ops.token_logprobs(z, t, 9), ops.token_logprobs(z, t, 9)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    z2 = z.clone()
    z2[1:] = float("nan")
    c = ops.token_logprobs(z2, t, 9)
    assert all(torch.equal(x[0], y[0]) for x, y in zip(a, c))


@pytest.mark.parametrize("form", ["logits", "head"])
def test_captured_replayed_and_on_other_streams(form):
    x = [torch.randn((24, 256), generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(DEV) for i in range(3)]
    w = (torch.randn((1500, 256), generator=torch.Generator().manual_seed(9)) * 0.1).to(torch.bfloat16).to(DEV)
    z = [v.float() @ w.float().t() for v in x]
    t = targets_of(24, 1500, 3)
    call = (lambda i: ops.token_logprobs(z[i], t, 4)) if form == "logits" else (lambda i: ops.linear_logprobs(x[i], w, t, 4, softcap=20.0))
    want = [call(i) for i in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append([call(i) for _ in range(5)][-1])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    # two graphs of the same call, replayed in turn on two streams, with other inputs in place
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = call(i)
        graphs.append((g, r))
    (x if form == "head" else z)[0].copy_((x if form == "head" else z)[2])
    for _ in range(3):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, r), b in zip(graphs, (want[2], want[1])):
        assert all(torch.equal(u, v) for u, v in zip(r, b))


def test_calls_of_several_threads_at_once():
    import threading
    g = torch.Generator().manual_seed(30)
    x = torch.randn((200, 256), generator=g).to(torch.bfloat16).to(DEV)
    w = (torch.randn((5000, 256), generator=g) * 0.1).to(torch.bfloat16).to(DEV)
    z, t = logits_of(50, 30000, torch.float32, 31), targets_of(50, 30000, 32)
    k = torch.randn((3, 20, 1000), device=DEV)
    want_head, want_rows = ops.linear_logprobs(x, w, None, 7, softcap=20.0), ops.token_logprobs(z, t, 7)
    moved_k = moved(k, [0, 1], [5, 6])
    torch.cuda.synchronize()
    wrong = []

    def work(form):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                own = k.clone()
                for _ in range(30):
                    if form == 0:
                        ok = all(torch.equal(a, b) for a, b in zip(ops.linear_logprobs(x, w, None, 7, softcap=20.0)[1:], want_head[1:]))
                    elif form == 1:
                        ok = all(torch.equal(a, b) for a, b in zip(ops.token_logprobs(z, t, 7), want_rows))
                    else:
                        ops.copy_rows([(own, [0, 1], [5, 6])])
                        ok = torch.equal(own, moved_k)
                    if not ok:
                        wrong.append(form)
        except Exception as e:
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(i % 3,)) for i in range(6)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


# ---- behind an output head ----

def head_case(rows, width, vocab, dtype, seed, scale=0.1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, width), generator=g).to(dtype)
    w = (torch.randn((vocab, width), generator=g) * scale).to(dtype)
    return x.to(DEV), w.to(DEV)


def head_logits(x, w, softcap, scale):
    """float64 logits, and what 32 bits may make of them: K products and sums of up to sum |x w|, 2^-24 each (2^-23 where tensor cores round
    towards zero), the soft-cap's argument, tanh and product (2^-21 of the cap up to 64, of the result above), the scale."""
    x, w = f64(x), f64(w)
    z = x @ w.T
    off = (np.abs(x) @ np.abs(w).T).max() * (x.shape[1] + 2) * 2.0 ** -23
    if softcap:
        z = softcap * np.tanh(z / softcap)
        off += (softcap if softcap <= 64 else np.abs(z).max()) * 2.0 ** -20
    return z * scale, (off + np.abs(z).max() * 2.0 ** -22) * abs(scale)


HEADS = [(1, 64, 100, "bfloat16"), (1, 2304, 5000, "bfloat16"), (16, 256, 777, "bfloat16"), (17, 256, 777, "bfloat16"), (64, 512, 3001, "bfloat16"),
         (127, 96, 256, "bfloat16"), (128, 64, 257, "bfloat16"), (129, 72, 1000, "bfloat16"), (300, 1000, 1111, "bfloat16"), (700, 128, 20000, "bfloat16"),
         (33, 8, 5, "bfloat16"), (20, 130, 90, "bfloat16"), (40, 1003, 50, "bfloat16"),
         (1, 64, 100, "float32"), (33, 1003, 777, "float32"), (130, 96, 2000, "float32")]


@pytest.mark.parametrize("rows,width,vocab,kind", HEADS)
@pytest.mark.parametrize("softcap,scale", [(None, 1.0), (8.0, 1.0), (None, 0.25), (5.0, -1.5), (64.0, 1.0), (1e4, 1.0), (1e30, 2.0), (1e-3, 1.0)])
def test_behind_an_output_head(rows, width, vocab, kind, softcap, scale):
    x, w = head_case(rows, width, vocab, getattr(torch, kind), rows + width)
    t = targets_of(rows, vocab, 5)
    z, off = head_logits(x, w, softcap, scale)
    top = min(5, vocab)
    r = ops.linear_logprobs(x, w, t, top, softcap=softcap, scale=scale)
    ref.check(r, z, t.cpu().numpy(), top, "head", more=off)
    # the ids named are those of logits within the error of the largest ones
    ids = r.top_ids.cpu().numpy()
    named = np.take_along_axis(z, ids, 1)
    best = -np.sort(-z, axis=1)[:, :top]
    assert (np.abs(named - best) <= 2 * off).all() and all(len(set(row)) == top for row in ids)


@pytest.mark.parametrize("rows,width,vocab", [(1, 320, 3000), (8, 64, 700), (40, 320, 3000), (150, 320, 3000), (257, 128, 513), (600, 64, 9000)])
@pytest.mark.parametrize("top", [0, 1, 20, 32])
def test_equal_logits_name_the_lowest_ids(rows, width, vocab, top):
    """Values on a coarse grid: sums are exact, many logits are equal, the ids are settled."""
    g = torch.Generator().manual_seed(rows)
    x = torch.randint(-3, 4, (rows, width), generator=g).to(torch.bfloat16).to(DEV)
    w = (torch.randint(-2, 3, (vocab, width), generator=g) / 16).to(torch.bfloat16).to(DEV)
    x[0] = 0                                             # all equal
    t = targets_of(rows, vocab, 6)
    ref.check(ops.linear_logprobs(x, w, t, top), f64(x) @ f64(w).T, t.cpu().numpy(), top, "exact sums")
    ref.check(ops.linear_logprobs(x, w, None, top), f64(x) @ f64(w).T, None, top, "without tokens")


@pytest.mark.parametrize("rows", [3, 40, 200])
def test_infinities_and_nan_behind_a_head(rows):
    x, w = head_case(rows, 64, 900, torch.bfloat16, 12)
    w[5] = 0
    w[5, 0] = -float("inf")                              # a token forbidden by its weight
    x[:, 0] = x[:, 0].abs() + 0.5
    x[1] = float("nan")
    x[2, 3] = float("inf")                               # logits of both infinities
    t = targets_of(rows, 900, 7)
    r = ops.linear_logprobs(x, w, t, 4)
    good = [i for i in range(rows) if i not in (1, 2)]
    z = f64(x[good]) @ f64(w[:5]).T
    z = np.concatenate([z, np.full((len(good), 1), -np.inf), f64(x[good]) @ f64(w[6:]).T], axis=1)
    part = ops.TokenLogprobs(*(v[good] for v in r))
    off = (np.abs(f64(x[good])) @ np.abs(f64(w[6:])).T).max() * 66 * 2.0 ** -23
    ref.check(part, z, t.cpu().numpy()[good], 4, "beside rows without a distribution", more=off)
    assert torch.isnan(r.logprobs[1:3]).all() and torch.isnan(r.entropy[1:3]).all()


@pytest.mark.parametrize("rows,vocab", [(20, 20001), (300, 20001), (17, 300), (140, 5000)])
@pytest.mark.parametrize("top", [1, 5, 20, 32])
@pytest.mark.parametrize("falling", [False, True])
def test_logits_that_rise_or_fall_along_the_vocabulary(rows, vocab, top, falling):
    """Rising logits all exceed what came before: more than a thread can put aside.  id = 256 a + b with exact numbers a, b; some equal ones."""
    ids = torch.arange(vocab - 1, -1, -1) if falling else torch.arange(vocab)
    ids = ids // 3 * 3
    w = torch.zeros((vocab, 64))
    w[:, 0], w[:, 1] = (ids // 256).float(), (ids % 256).float() / 256
    x = torch.zeros((rows, 64))
    x[:, :2] = 0.25
    x[1, :2] = 2.0                                       # steep
    x[2, :2] = -0.25
    x, w = x.to(torch.bfloat16).to(DEV), w.to(torch.bfloat16).to(DEV)
    t = targets_of(rows, vocab, 11)
    ref.check(ops.linear_logprobs(x, w, t, top), f64(x) @ f64(w).T, t.cpu().numpy(), top, "rising logits")


def test_rows_without_a_distribution_name_the_lowest_ids():
    x, w = head_case(40, 64, 5000, torch.bfloat16, 14)
    x[3] = float("nan")                                  # every logit
    w[:, 0] = 0
    w[7:5000:9, 0] = float("nan")                        # some logits of every row
    x[:, 0] = 1.0
    r = ops.linear_logprobs(x, w, None, 32)
    assert torch.isnan(r.entropy).all() and r.top_ids[3].tolist() == list(range(32))
    z = f64(x) @ f64(w).T
    for i in (0, 39):
        assert not np.isnan(z[i, r.top_ids[i].cpu().numpy()]).any()
    w[:, 1:] = 0
    w[:, 0] = -float("inf")
    r = ops.linear_logprobs(x[:2].repeat(20, 1), w, None, 5)
    assert torch.isnan(r.entropy).all() and (r.top_ids == torch.arange(5, device=DEV)).all()
    w[4000:, 0] = 1.0                                    # behind many tokens of no probability
    r = ops.linear_logprobs(x[:2].repeat(20, 1), w, None, 5)
    assert (r.top_ids == torch.arange(4000, 4005, device=DEV)).all() and torch.allclose(r.entropy, torch.tensor(float(np.log(1000)), device=DEV))


@pytest.mark.parametrize("rows,vocab", [(19000, 300), (20000, 70)])
def test_more_rows_than_one_launch_has_blocks_for(rows, vocab):
    g = torch.Generator().manual_seed(15)
    x = torch.randint(-3, 4, (rows, 64), generator=g).to(torch.bfloat16).to(DEV)
    w = (torch.randint(-2, 3, (vocab, 64), generator=g) / 16).to(torch.bfloat16).to(DEV)
    t = targets_of(rows, vocab, 12)
    r = ops.linear_logprobs(x, w, t, 3)
    some = list(range(0, rows, 997)) + [rows - 1]
    part = ops.TokenLogprobs(*(v[some] for v in r))
    ref.check(part, f64(x[some]) @ f64(w).T, t.cpu().numpy()[some], 3, "many rows")
    want = ops.token_logprobs(ops.linear(x, w, torch.float32), t, 3)
    assert torch.equal(r.top_ids, want.top_ids) and torch.allclose(r.logprobs, want.logprobs, atol=1e-5) and torch.allclose(r.entropy, want.entropy, atol=1e-5)


@pytest.mark.parametrize("rows", [40, 300, 200])
def test_a_token_outside_the_vocabulary_behind_a_head(rows):
    x, w = head_case(rows, 64, 300, torch.bfloat16, 16)
    t = torch.full((rows,), 5, dtype=torch.int32, device=DEV)
    t[1], t[2], t[3], t[rows - 1] = 300, -1, 2 ** 31 - 1, 299
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    r = ops.linear_logprobs(x, w, t, 2, status=status)
    assert status.item() == 11 and torch.isnan(r.logprobs).nonzero().flatten().tolist() == [1, 3] and r.logprobs[2].item() == 0.0
    want = ops.token_logprobs(ops.linear(x, w, torch.float32), t, 2)
    assert torch.allclose(r.logprobs, want.logprobs, atol=1e-4, equal_nan=True)


SHORT_WAIT = 200_000       # clock cycles, about a tenth of a millisecond


@pytest.mark.parametrize("rows", [40, 200, 300])
@pytest.mark.parametrize("top", [0, 5])
def test_a_wait_that_runs_out(rows, top):
    lib = library.load()
    x, w = head_case(rows, 256, 3000, torch.bfloat16, 17)
    t = targets_of(rows, 3000, 13)
    want = ops.linear_logprobs(x, w, t, top)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    try:
        lib.rdl_set_wait_test(12, SHORT_WAIT, 64)
        ops.linear_logprobs(x, w, t, top, status=status)
        torch.cuda.synchronize()                         # the kernels returned by themselves
    finally:
        lib.rdl_set_wait_test(0, 0, 0)
    assert "linear_logprobs" in library.FAULTS[status.item()]
    status.zero_()
    got = ops.linear_logprobs(x, w, t, top, status=status)
    assert status.item() == 0 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_long_kernel_ahead_is_no_wait_in_vain():
    lib, status = library.load(), torch.zeros(1, dtype=torch.int32, device=DEV)
    x, w = head_case(200, 256, 3000, torch.bfloat16, 18)
    want = ops.linear_logprobs(x, w, None, 3)
    a = torch.ones((4096, 4096), device=DEV)
    try:
        lib.rdl_set_wait_test(12, SHORT_WAIT, 0)
        for _ in range(3):
            ops.linear(a, a)                             # 2 ms
            got = ops.linear_logprobs(x, w, None, 3, status=status)
        torch.cuda.synchronize()
    finally:
        lib.rdl_set_wait_test(0, 0, 0)
    assert status.item() == 0 and all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))


def test_a_4_bit_head_in_pieces(monkeypatch):
    """The last rows of many are taken as the others are."""
    x, w = head_case(150, 320, 1000, torch.bfloat16, 21)
    packed = ops.pack_mx4(w)
    want = ops.token_logprobs(ops.linear(x, packed, torch.float32), None, 6)
    monkeypatch.setattr(ops, "LOGPROBS_PIECE", 1000 * 70)
    got = ops.linear_logprobs(x, packed, None, 6)
    # 8-bit rows are multiplied by another kernel where they are fewer than 129: the order of 320 products' sums
    assert torch.allclose(got.entropy, want.entropy, atol=1e-3) and torch.allclose(got.top_logprobs, want.top_logprobs, atol=1e-3)


@pytest.mark.parametrize("rows", [1, 16, 17, 130])
@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_a_4_bit_head(rows, kind):
    x, w = head_case(rows, 320, 1000, getattr(torch, kind), 20)
    packed = ops.pack_mx4(w)
    t = targets_of(rows, 1000, 8)
    want = ops.token_logprobs(ops.scale_(ops.linear(x, packed, torch.float32, 9.0), 0.5), t, 6)
    got = ops.linear_logprobs(x, packed, t, 6, softcap=9.0, scale=0.5)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- copies ----

def moved(t, src, dst):
    out = t.clone()
    for a, b in zip(src, dst):
        out[:, b] = t[:, a]
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8, torch.int32, torch.float64])
@pytest.mark.parametrize("sets,rows,shape", [(1, 2, (1,)), (3, 5, (7,)), (2, 6, (3, 7, 33)), (13, 4, (4, 64, 64)), (2, 3, ()), (1, 2, (100003,)), (5, 9, (2, 16, 32))])
def test_copied_rows(dtype, sets, rows, shape):
    t = torch.randint(0, 200, (sets, rows, *shape), generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    order = np.random.default_rng(rows).permutation(rows).tolist()
    src, dst = order[:rows // 2], order[rows // 2:2 * (rows // 2)]
    want = moved(t, src, dst)
    ops.copy_rows([(t, src, dst)])
    assert torch.equal(t, want)


def test_one_row_into_many_several_tensors_and_no_rows():
    k, v, s = (torch.randn((4, 40, n), device=DEV) for n in (512, 96, 33))
    empty = torch.empty((4, 40, 0), device=DEV)
    want = [moved(k, [3, 3, 3], [0, 39, 7]), moved(v, [3, 3, 3], [0, 39, 7]), moved(s, [5], [6])]
    ops.copy_rows([(k, [3, 3, 3], [0, 39, 7]), (v, [3, 3, 3], [0, 39, 7]), (empty, [1], [2]), (s, (5,), np.array([6]))])
    assert all(torch.equal(a, b) for a, b in zip((k, v, s), want))
    ops.copy_rows([(k, [], [])])
    ops.copy_rows([])
    assert torch.equal(k, want[0])


def test_rows_and_sets_that_lie_apart():
    base = torch.randn((3, 10, 6, 50), device=DEV)
    before = base.clone()
    part = base[:, 2:8, 1:4]                             # rows with gaps
    want = moved(part, [0, 1], [5, 3])
    ops.copy_rows([(part, [0, 1], [5, 3])])
    before[:, 2:8, 1:4] = want
    assert torch.equal(base, before)
    turned = torch.randn((8, 3, 20), device=DEV).transpose(0, 1)     # sets nearer than rows
    want = moved(turned, [7], [1])
    ops.copy_rows([(turned, [7], [1])])
    assert torch.equal(turned, want)
    odd = torch.randn(1 + 2 * 4 * 37, device=DEV).to(torch.bfloat16)[1:].view(2, 4, 37)
    want = moved(odd, [3, 0], [1, 2])
    ops.copy_rows([(odd, [3, 0], [1, 2])])
    assert torch.equal(odd, want)


@pytest.mark.parametrize("n", [64, 65, 2048, 2049, 5000])
def test_long_lists(n):
    k, v = torch.randn((2, 2 * n, 24), device=DEV), torch.randn((2, 2 * n, 5), device=DEV)
    order = np.random.default_rng(n).permutation(2 * n).tolist()
    src, dst = order[:n], order[n:]
    want = []
    for t in (k, v):
        o = t.clone()
        o[:, dst] = t[:, src]
        want.append(o)
    ops.copy_rows([(k, src, dst), (v, src, dst)])
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_copies_beyond_32_bits_and_in_a_graph():
    t = torch.zeros((2, 3, 1 << 30), dtype=torch.uint8, device=DEV)          # 6 GB
    t[0, 2, -1000:], t[1, 2, :1000] = 7, 9
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.copy_rows([(t, [2], [0])])
    assert int(t[:, 0].max()) == 0
    g.replay()
    assert torch.equal(t[:, 0], t[:, 2]) and int(t[0, 0, -1]) == 7 and int(t[:, 1].max()) == 0


def test_more_rows_than_a_launch_has_blocks_for():
    """2^31 and more blocks of a byte each: the list is divided where the blocks end, and the tensor behind it, which shares the list, goes on."""
    sets, pairs = 1 << 20, 2100
    t = torch.zeros((sets, 2 * pairs), dtype=torch.uint8, device=DEV)        # 4.4 GB
    t[:, :pairs] = (torch.arange(pairs, device=DEV) % 251 + 1).to(torch.uint8)
    t[:, :pairs] += (torch.arange(sets, device=DEV) % 5).to(torch.uint8)[:, None]
    small = torch.randn((2, 2 * pairs, 5), device=DEV)
    src, dst = list(range(pairs)), list(range(pairs, 2 * pairs))
    want = moved(small, src, dst)
    ops.copy_rows([(t, src, dst), (small, src, dst)])
    assert torch.equal(t[:, pairs:], t[:, :pairs]) and torch.equal(small, want)


@pytest.mark.parametrize("rows,width,vocab,shift", [(300, 63, 900, 0), (257, 1003, 50, 0), (300, 64, 900, 1), (600, 7, 2000, 0)])
def test_many_rows_of_odd_widths_take_the_kernel(monkeypatch, rows, width, vocab, shift):
    """Widths that are no multiple of 8, and operands that start anywhere: sums that are exact, and no library product."""
    g = torch.Generator().manual_seed(rows + width)
    x, w = torch.empty(rows * width + shift, dtype=torch.bfloat16, device=DEV)[shift:], torch.empty(vocab * width + shift, dtype=torch.bfloat16, device=DEV)[shift:]
    x, w = x.view(rows, width), w.view(vocab, width)
    x.copy_(torch.randint(-3, 4, (rows, width), generator=g))
    w.copy_(torch.randint(-2, 3, (vocab, width), generator=g) / 16)

    def refuse(*args, **kw):
        raise AssertionError("a library product")
    monkeypatch.setattr(torch, "mm", refuse)
    t = targets_of(rows, vocab, 6)
    ref.check(ops.linear_logprobs(x, w, t, 7), f64(x) @ f64(w).T, t.cpu().numpy(), 7, "an odd width")


def test_pieces_of_logits_are_held_one_at_a_time(monkeypatch):
    x, w = head_case(1200, 320, 5000, torch.bfloat16, 22)
    packed = ops.pack_mx4(w)
    monkeypatch.setattr(ops, "LOGPROBS_PIECE", 400 * 5000)
    want = ops.linear_logprobs(x, packed, None, 3)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = ops.linear_logprobs(x, packed, None, 3)
    # a piece of logits is 8 MB; its rows in 8 bits and the results are less than one
    assert torch.cuda.max_memory_allocated() - held < 10e6
    assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))
