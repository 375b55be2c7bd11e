"""Plain forms, in 64 bits, of what scores tokens and copies rows of a cache."""
import numpy as np
import torch

from rust_deeplearning_b200.kernels import ops

U = 2.0 ** -24          # half a step of float32


def rows64(z, targets, top):
    """float64 numpy rows of logits -> (log probabilities, entropies, ids, their log probabilities, tolerance of each log probability as
    a function of its own d = z - m, tolerance of the entropies).

    Tolerances.  With d = z - m and p = exp(d) / s: d is rounded (u |d|, u = 2^-24), its product with log2 e too, and that constant (u |d| each), 2^x
    is off by 2 ulp (4 u): an exponential is off by (3 |d| + 4) u of itself.  A thread adds up vocab / 16384 batches of up to 32 logits (the
    fewest threads a row gets are 512, 32 a batch; shorter rows fewer), and what the batches, lanes, warps and blocks hold joins in fewer than
    100 further steps, each of which rounds and multiplies by a factor near 1 that is off by as much: (200 + vocab / 4096) u generously.  So ln s
    is off by (3 E|d| + 204 + vocab / 4096) u, and by the logarithm's own 2 ulp (4 u |ln s|); a log probability adds u |d| and
    a rounding of the result.  The entropy's second term is sum p |d|, whose terms are off by (3 |d| + 6) u."""
    z = np.asarray(z, dtype=np.float64)
    rows, vocab = z.shape
    lp, ent, ids, tops, tol, tol_e = np.full(rows, np.nan), np.full(rows, np.nan), np.zeros((rows, top), np.int32), np.full((rows, top), np.nan), [], []
    for r in range(rows):
        key = np.where(np.isnan(z[r]), -np.inf, z[r])
        order = np.lexsort((np.arange(vocab), -key, np.isnan(z[r])))[:top]
        ids[r] = order
        good = not np.isnan(z[r]).any() and np.isfinite(z[r].max())
        if good:
            d = z[r] - z[r].max()
            e = np.exp(d)
            s = e.sum()
            a = np.where(e > 0, -d, 0.0)
            ln_s = np.log(s)
            ent[r] = ln_s + (e * a).sum() / s
            if targets is not None and 0 <= targets[r] < vocab:
                lp[r] = d[targets[r]] - ln_s
            tops[r] = d[order] - ln_s
            mean, square, many = (e * a).sum() / s, (e * a * a).sum() / s, 204 + vocab / 4096
            base = 3 * mean + many + 4 * ln_s
            tol.append(base)
            tol_e.append(U * (base + 3 * square + mean * (2 * many + 6) + 2 * ent[r] + 2))
        else:
            tol.append(0.0)
            tol_e.append(0.0)
        if targets is not None and targets[r] < 0:
            lp[r] = 0.0
    base = np.asarray(tol)
    # 2^-24 (|d| + what ln s is off by) and a rounding of the result: |d| <= |lp|
    of = lambda v: U * (base.reshape((-1,) + (1,) * (v.ndim - 1)) + 2 * np.abs(np.where(np.isfinite(v), v, 0.0)) + 1)
    return lp, ent, ids, tops, of(lp), np.asarray(tol_e), of(tops)


def same(got, want, tol, what):
    got = got.detach().double().cpu().numpy() if isinstance(got, torch.Tensor) else np.asarray(got)
    assert got.shape == want.shape, f"{what}: {got.shape} instead of {want.shape}"
    assert (np.isnan(got) == np.isnan(want)).all(), f"{what}: NaN in other places"
    exact = ~np.isfinite(want)
    assert (got[exact & ~np.isnan(want)] == want[exact & ~np.isnan(want)]).all(), f"{what}: infinities differ"
    err = np.abs(np.where(exact, 0, got) - np.where(exact, 0, want)) - np.where(exact, 0, tol)
    assert err.size == 0 or (err <= 0).all(), f"{what}: {float(err.max()):.3e} beyond the tolerance"


def check(result, z, targets, top, what, more=0.0):
    """A TokenLogprobs against float64 logits; more: what the logits themselves may be off by."""
    lp, ent, ids, tops, tol, tol_e, tol_t = rows64(z, targets, top)
    if targets is None:
        assert result.logprobs is None
    else:
        same(result.logprobs, lp, tol + 2 * more, what + ": log probabilities")
    # dH = -sum p_i (ln p_i + H) dz_i
    spread = np.where(np.isfinite(ent), 2 * np.abs(ent) + 2, 0.0)
    same(result.entropy, ent, tol_e + more * spread, what + ": entropy")
    assert tuple(result.top_ids.shape) == (len(ids), top)
    if more == 0.0:
        assert (result.top_ids.cpu().numpy() == ids).all(), what + ": ids"
    same(result.top_logprobs, tops, tol_t + 2 * more, what + ": alternatives")


def copy_rows(moves):
    for t, src, dst in moves:
        t[:, list(dst)] = t[:, list(src)].clone()


def token_logprobs(logits, targets=None, top=0, status=None):
    z = logits.double()
    p = torch.log_softmax(z, dim=1)
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
    lp = None if targets is None else torch.gather(p, 1, targets.long().clamp(min=0).unsqueeze(1)).squeeze(1).float()
    return ops.TokenLogprobs(lp, -(p.exp() * p).nansum(dim=1).float(), order.to(torch.int32), torch.gather(p, 1, order).float())


def linear_logprobs(x, weight, targets=None, top=0, softcap=None, scale=1.0, status=None):
    z = x.double() @ weight.double().t()
    return token_logprobs((softcap * torch.tanh(z / softcap) if softcap else z) * scale, targets, top)


def install(monkeypatch):
    for f in (copy_rows, token_logprobs, linear_logprobs):
        monkeypatch.setattr(ops, f.__name__, f)
