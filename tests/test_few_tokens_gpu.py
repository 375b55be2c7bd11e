"""Rows of which few tokens are allowed, or whose logits are equal: alternatives against float64, and no slower than other rows."""
import numpy as np
import pytest
import torch

import scoring_refs as ref
from rust_deeplearning_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def f64(t):
    return t.detach().double().cpu().numpy()


def only(z, allowed, seed):
    """z with all but `allowed` of each row's tokens forbidden."""
    keep = torch.stack([torch.randperm(z.shape[1], generator=torch.Generator().manual_seed(seed + r))[:allowed] for r in range(len(z))]).to(DEV)
    return torch.full_like(z, -float("inf")).scatter_(1, keep, z.gather(1, keep))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,offset", [(8, 256000, 0), (3, 50001, 3), (300, 5003, 1), (700, 1500, 0)])
@pytest.mark.parametrize("allowed", [1, 4, 19, 33, 300])
def test_few_allowed_tokens(rows, vocab, offset, allowed, dtype):
    g = torch.Generator().manual_seed(rows + allowed)
    wide = torch.randn((rows, vocab + offset), generator=g).to(dtype).to(DEV)
    z = wide[:, offset:]
    z.copy_(only(z.contiguous(), allowed, 1))
    some = list(range(0, rows, max(1, rows // 8)))
    for top in (1, 5, 20, 32):
        r = ops.token_logprobs(z, None, top)
        ref.check(ops.TokenLogprobs(None, *(v[some] for v in r[1:])), f64(z[some]), None, top, f"{allowed} of {vocab} allowed")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,offset", [(8, 256000, 0), (3, 50001, 1), (300, 5003, 7)])
def test_few_distinct_values(rows, vocab, offset, dtype):
    """One value, or three of them in runs, in turn and at the ends, infinities, NaN and both zeros among them."""
    base = torch.zeros((rows, vocab + offset), dtype=dtype, device=DEV)
    z = base[:, offset:]
    z[0] = 1.25
    z[1] = -0.0; z[1, ::3] = 0.0
    z[2] = -2.0; z[2, 7::1000] = 3.0; z[2, -5:] = 3.0
    if rows > 3:
        z[3] = torch.finfo(dtype).min; z[3, 5000:] = -float("inf"); z[3, 100::640] = 1.0
        z[4] = -float("inf"); z[4, -1] = 0.5; z[4, 0] = 0.5
        z[5] = float("nan"); z[5, 11::900] = -float("inf")
        z[6] = float("inf")
        z[7] = -float("inf")
    some = list(range(min(rows, 9)))
    for top in (1, 5, 32):
        r = ops.token_logprobs(z, None, top)
        ref.check(ops.TokenLogprobs(None, *(v[some] for v in r[1:])), f64(z[some]), None, top, "few values")


def device_time(call, n=5):
    """Seconds a call on the device, the least of several graphs' replays."""
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(n):
            call()
    times = []
    for _ in range(6):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        g.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e-3 / n)
    return min(times)


@pytest.mark.parametrize("rows,vocab,dtype", [(8, 256000, torch.float32), (2048, 32000, torch.float32), (1024, 64000, torch.bfloat16)])
@pytest.mark.parametrize("kind", [4, 30, "equal"])
def test_rows_of_few_tokens_take_no_longer(rows, vocab, dtype, kind):
    """Putting every forbidden token aside took 5 to 15 times as long.  Twice covers what a row's first logits cost and the clock."""
    z = torch.randn((rows, vocab), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dtype)
    other = torch.full_like(z, 1.25) if kind == "equal" else torch.full_like(z, -float("inf"))
    if kind != "equal":
        other[:, 1000:1000 + 700 * kind:700] = z[:, :kind]
    usual, few = device_time(lambda: ops.token_logprobs(z, None, 20)), device_time(lambda: ops.token_logprobs(other, None, 20))
    assert few < 2 * usual, f"{few * 1e6:.1f} us instead of {usual * 1e6:.1f}"


# ---- behind an output head ----

@pytest.mark.parametrize("rows,width,vocab", [(40, 64, 9000), (200, 64, 9000), (300, 64, 20001)])
@pytest.mark.parametrize("top", [1, 5, 32])
def test_equal_logits_behind_a_head(rows, width, vocab, top):
    """Rows of zeros, rows of two values, and rows that rise in steps of many equal logits."""
    w = torch.zeros((vocab, width))
    w[:, 0] = (torch.arange(vocab) // 1000).float()
    w[:, 1] = (torch.arange(vocab) % 777 == 5).float()
    w[:, 2] = torch.where(torch.arange(vocab) % 3 == 0, 0.0, -1.0)
    x = torch.zeros((rows, width))
    x[1, 0], x[2, 0], x[3, 1], x[4, 2], x[5, :2], x[6, 1] = 0.25, -0.25, 1.0, 4.0, 0.5, -2.0
    x, w = x.to(torch.bfloat16).to(DEV), w.to(torch.bfloat16).to(DEV)
    some = list(range(8)) + [rows - 1]
    r = ops.linear_logprobs(x, w, None, top)
    ref.check(ops.TokenLogprobs(None, *(v[some] for v in r[1:])), f64(x[some]) @ f64(w).T, None, top, "equal logits")


@pytest.mark.parametrize("top", [5, 20])
def test_equal_logits_behind_a_head_take_no_longer(top):
    """Sorting every logit in took 6.4 and 8.2 times as long (now 1.5 and 2.2 times)."""
    g = torch.Generator(device=DEV).manual_seed(1)
    x, w = torch.randn((512, 256), generator=g, device=DEV).to(torch.bfloat16), torch.randn((32000, 256), generator=g, device=DEV).to(torch.bfloat16)
    zero = torch.zeros_like(x)
    usual, equal = device_time(lambda: ops.linear_logprobs(x, w, None, top)), device_time(lambda: ops.linear_logprobs(zero, w, None, top))
    assert equal < 4 * usual, f"{equal * 1e6:.1f} us instead of {usual * 1e6:.1f}"
