"""Soft-capped logits behind an output head: what the soft-cap itself may cost, told apart from the products in front of it by sums that are exact.

A capped logit is off by at most 4.5 * 2^-22 of itself: from half of the cap on, cap (1 - 2 r), r = 1 / (e + 1), e = e^(2 y).  y and the power's argument
carry 3 roundings and a constant's (3.5 u, u = 2^-24, times 2 |y|), the power 2^-22, the sum u, the reciprocal 2^-23, each times what r or its own
share of e + 1 is: worst at y = -1/2, where r = 0.73, e / (e + 1) = 0.27 and the logit 0.46 caps: ((3.5 + 4) 0.27 + 1 + 2) u 2 * 0.73 / 0.46
+ u = 17 u = 4.2 * 2^-22.  Below half of the cap the odd polynomial (2^-26) and its roundings: less than 2^-22.  `linear`'s form (few rows,
float32): a division, tanhf (2 units in the last place at most) and a product: 6 u.  A scale rounds once more."""
import numpy as np
import pytest
import torch

import scoring_refs as ref
from rust_deeplearning_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
OFF = 4.75 * 2.0 ** -22


def f64(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("rows,width,vocab,kind", [(5, 64, 700, "bfloat16"), (17, 64, 700, "bfloat16"), (64, 128, 3001, "bfloat16"), (200, 64, 1000, "bfloat16"),
                                                   (300, 64, 2500, "bfloat16"), (40, 63, 700, "bfloat16"), (33, 64, 700, "float32")])
@pytest.mark.parametrize("softcap,scale", [(1e-3, 1.0), (0.5, 40.0), (5.0, -1.5), (30.0, 1.0), (30.0, 100.0), (64.0, 1.0), (1e4, 1.0), (1e30, 2.0), (3e38, 1.0)])
def test_a_soft_cap_of_exact_sums(rows, width, vocab, kind, softcap, scale):
    g = torch.Generator().manual_seed(rows + vocab)
    dtype = getattr(torch, kind)
    x = torch.randint(-3, 4, (rows, width), generator=g).to(dtype).to(DEV)
    w = (torch.randint(-2, 3, (vocab, width), generator=g) / 64).to(dtype).to(DEV)
    t = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32).to(DEV)
    cap = float(np.float32(softcap))
    z = cap * np.tanh(f64(x) @ f64(w).T / cap) * scale
    r = ops.linear_logprobs(x, w, t, 20, softcap=softcap, scale=scale)
    ref.check(r, z, t.cpu().numpy(), 20, "a soft-cap", more=OFF * np.abs(z).max())
    # the k-th named logit is within the error of the k-th largest
    named = np.take_along_axis(z, r.top_ids.cpu().numpy().astype(np.int64), 1)
    best = -np.sort(-z, axis=1)[:, :20]
    assert (np.abs(named - best) <= 2.1 * OFF * np.abs(best)).all() and all(len(set(row)) == 20 for row in r.top_ids.tolist())


@pytest.mark.parametrize("rows", [3, 17, 64, 200, 300])
@pytest.mark.parametrize("softcap,scale", [(None, 1.0), (1.0, 1.0), (8.0, 1.0), (30.0, 1.0), (30.0, 64.0), (64.0, 1.0), (1000.0, 1.0)])
def test_small_distinct_logits_keep_their_order(rows, softcap, scale):
    """65,536 logits between 0 and 2^-4, 2^-20 apart, in no order: 2^-20 is ten times what two of them may be off by together."""
    values = torch.randperm(65536, generator=torch.Generator().manual_seed(1))
    w = torch.zeros((65536, 64))
    w[:, 0], w[:, 1] = (values // 256).float() * 2.0 ** -12, (values % 256).float() * 2.0 ** -20
    x = torch.zeros((rows, 64))
    x[:, :2] = 1.0
    x[1] /= 8
    x[2] /= -2
    w, x = w.to(torch.bfloat16).to(DEV), x.to(torch.bfloat16).to(DEV)
    some = [0, 1, 2, rows - 1]
    z = f64(x[some]) @ f64(w).T
    z = (softcap * np.tanh(z / softcap) if softcap else z) * scale
    assert all(len(np.unique(row)) == 65536 for row in z)
    want = np.argsort(-z, axis=1, kind="stable")[:, :32]
    r = ops.linear_logprobs(x, w, None, 32, softcap=softcap, scale=scale)
    assert (r.top_ids[some].cpu().numpy() == want).all()
    ref.check(ops.TokenLogprobs(None, *(v[some] for v in r[1:])), z, None, 32, "small logits", more=OFF * np.abs(z).max())
