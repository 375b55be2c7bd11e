"""What the speed of scoring tokens and of forking sequences is measured on.

Three operators, by the case's "op":

    logits    log probabilities of given tokens, entropy and top alternatives of rows of logits    (beside sampling, in decode steps)
    head      the same from the rows that enter the output head: the logits are never kept         (scoring texts)
    copy      pages of keys and values, and states, copied in every layer run of a cache            (several continuations of a prompt)

For a row z of logits with largest value m and s = sum exp(z - m), a token's log probability is z_i - m - ln s and the row's
entropy ln s - sum (z - m) exp(z - m) / s; alternatives are the tokens of the largest logits, equal ones in the order of their ids.
The head's logits are x W^T, behind a soft-cap cap * tanh(. / cap) where there is one.

Sizes are those of the Gemma 2 2B shape, of shapes with a vocabulary of 32,000, and odd ones.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
BYTES = {"bfloat16": 2, "float32": 4}
PIECE = 1 << 26                     # logits the plain form and the exact one hold at a time
LARGEST_LOGITS = 2048 * 256000
LARGEST_HEAD = 8192 * 2304 * 256000
LARGEST_COPY = 128 * 26 * 4 * 64 * 256 * 2      # elements of bfloat16 in the pages of the largest copy, keys and values


def listed():
    return [
        # one sequence's decode step, vocabulary of 32,000: latency
        {"name": "logits_one", "op": "logits", "rows": 1, "vocab": 32000, "x": "float32", "top": 5, "masked": False},
        # a decode step of eight sequences, 2B shape, as many alternatives as are usually offered
        {"name": "logits_batch", "op": "logits", "rows": 8, "vocab": 256000, "x": "float32", "top": 20, "masked": False},
        # rows of bfloat16 (many equal values) with tokens that a grammar forbids, sizes that nothing divides
        {"name": "logits_odd", "op": "logits", "rows": 333, "vocab": 1003, "x": "bfloat16", "top": 3, "masked": True},
        # the logits of a whole prompt of 2,048 tokens
        {"name": "logits_prompt", "op": "logits", "rows": 2048, "vocab": 256000, "x": "float32", "top": 5, "masked": False},
        # the last row of one sequence through the 2B shape's output head
        {"name": "head_one", "op": "head", "rows": 1, "in": 2304, "vocab": 256000, "x": "bfloat16", "cap": 30.0, "top": 5},
        # short texts scored together, or the rows of a batch of 64
        {"name": "head_some", "op": "head", "rows": 64, "in": 2304, "vocab": 256000, "x": "bfloat16", "cap": 30.0, "top": 20},
        # the 32-bit path, sizes that nothing divides
        {"name": "head_odd", "op": "head", "rows": 333, "in": 1003, "vocab": 777, "x": "float32", "cap": 0.0, "top": 1},
        # perplexity of a text of 2,048 tokens
        {"name": "head_prompt", "op": "head", "rows": 2048, "in": 2304, "vocab": 256000, "x": "bfloat16", "cap": 30.0, "top": 0},
        # a long text with its alternatives
        {"name": "head_long", "op": "head", "rows": 8192, "in": 2304, "vocab": 256000, "x": "bfloat16", "cap": 30.0, "top": 5},
        # one page of the 2B shape's window layers, as a sequence that shares it is about to write to it
        {"name": "copy_one", "op": "copy", "sets": 13, "heads": 4, "page": 64, "dim": 256, "x": "bfloat16", "rows": 1, "state_heads": 0, "state_dim": 0},
        # eight continuations of one sequence with a state a layer (4 heads of 256 x 256) and pages of a size that nothing divides
        {"name": "copy_states", "op": "copy", "sets": 3, "heads": 3, "page": 7, "dim": 33, "x": "bfloat16", "rows": 8, "state_heads": 4, "state_dim": 256},
        # all pages of a sequence of 8,192 tokens, 2B shape, in all layers
        {"name": "copy_long", "op": "copy", "sets": 26, "heads": 4, "page": 64, "dim": 256, "x": "bfloat16", "rows": 128, "state_heads": 0, "state_dim": 0},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logits", "logits", "head", "head", "head", "copy"])
    if op == "logits":
        vocab = _spread(rng, 100, 256000)
        rows = min(_spread(rng, 1, 8192), LARGEST_LOGITS // vocab)
        return {"op": op, "rows": rows, "vocab": vocab, "x": rng.choice(["float32", "float32", "bfloat16"]), "top": rng.randint(0, 20),
                "masked": rng.random() < 0.3}
    if op == "head":
        kind = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        width, vocab = _spread(rng, 64, 4608), _spread(rng, 100, 256000)
        if kind == "bfloat16" or rng.random() < 0.5:
            width = width // 8 * 8
        largest = LARGEST_HEAD if kind == "bfloat16" else LARGEST_HEAD // 64
        rows = max(1, min(_spread(rng, 1, 8192), largest // (width * vocab)))
        return {"op": op, "rows": rows, "in": width, "vocab": vocab, "x": kind, "cap": rng.choice([0.0, 30.0]), "top": rng.randint(0, 20)}
    kind = rng.choice(["bfloat16", "bfloat16", "float32"])
    sets, heads, page, dim = rng.randint(1, 26), rng.randint(1, 8), rng.choice([16, 64, 64, 64, 7]), rng.choice([32, 64, 128, 256, 33])
    with_state = rng.random() < 0.4
    most = LARGEST_COPY // (sets * heads * page * dim * BYTES[kind]) // (2 if with_state else 1)
    return {"op": op, "sets": sets, "heads": heads, "page": page, "dim": dim, "x": kind, "rows": max(1, min(_spread(rng, 1, 128), most)),
            "state_heads": rng.randint(1, 4) if with_state else 0, "state_dim": rng.choice([64, 128, 127]) if with_state else 0}


# ---- inputs ----

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32)


def _grid(gen, rows, width, std, step, kind):
    """Normal values on a grid.  Sums of products of such values are exact in 32 bits, so that the order of the logits (and which
    are equal) does not hang on the order of additions."""
    out = torch.empty(rows, width, dtype=kind, device=DEVICE)
    for part in out.split(max(1, PIECE // width)):
        part.copy_(torch.round(_normal(gen, *part.shape) * (std / step)) * step)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    state = {"case": case}
    kind = getattr(torch, case["x"])
    if case["op"] == "copy":
        n, copies = 2 * case["rows"] + 3, case["rows"]
        shape = (case["sets"], n, case["heads"], case["page"], case["dim"])
        state["k"], state["v"] = _normal(gen, *shape).to(kind), _normal(gen, *shape).to(kind)
        # lists of page ids, as a cache's bookkeeping holds them on the host
        order = torch.randperm(n, generator=gen, device=DEVICE).tolist()
        state["src"], state["dst"] = order[:copies], order[copies:2 * copies]
        if case["state_heads"]:
            state["state"] = _normal(gen, case["sets"], copies + 1, case["state_heads"], case["state_dim"], case["state_dim"])
            state["state_src"], state["state_dst"] = [copies] * copies, list(range(copies))     # one sequence forked into all others
        return state
    rows, vocab = case["rows"], case["vocab"]
    state["targets"] = torch.randint(0, vocab, (rows,), generator=gen, device=DEVICE, dtype=torch.int32)
    if case["op"] == "logits":
        # rows of different spread: some nearly certain, some nearly flat
        spread = torch.exp(0.5 * _normal(gen, rows, 1)) * 3.0
        z = torch.empty(rows, vocab, dtype=kind, device=DEVICE)
        for part, s in zip(z.split(max(1, PIECE // vocab)), spread.split(max(1, PIECE // vocab))):
            part.copy_(_normal(gen, *part.shape) * s)
        if case["masked"]:
            forbidden = torch.rand(rows, vocab, generator=gen, device=DEVICE) < 0.3
            forbidden.scatter_(1, state["targets"].long().unsqueeze(1), False)
            z.masked_fill_(forbidden, float("-inf"))
        state["logits"] = z
        return state
    state["x"] = _grid(gen, rows, case["in"], 1.0, 1 / 4, kind)
    state["weight"] = _grid(gen, vocab, case["in"], 0.08, 1 / 256, kind)
    return state


# ---- one pass ----

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _outputs(logprobs, entropy, ids, top):
    out = {"logprobs": logprobs, "entropy": entropy}
    if ids.shape[1]:
        out["top_ids"], out["top_logprobs"] = ids, top
    return out


def _buffers(state):
    return {name: state[name] for name in ("k", "v", "state") if name in state}


def _run_own(state):
    from rust_deeplearning_b200.kernels import ops
    case = state["case"]
    if case["op"] == "copy":
        moves = [(state["k"], state["src"], state["dst"]), (state["v"], state["src"], state["dst"])]
        if "state" in state:
            moves.append((state["state"], state["state_src"], state["state_dst"]))
        ops.copy_rows(moves)
        return _buffers(state)
    if case["op"] == "logits":
        r = ops.token_logprobs(state["logits"], state["targets"], top=case["top"])
    else:
        r = ops.linear_logprobs(state["x"], state["weight"], state["targets"], top=case["top"], softcap=case["cap"] or None)
    return _outputs(r.logprobs, r.entropy, r.top_ids, r.top_logprobs)


def _plain_rows(z, targets, top):
    """Of float32 rows of logits: log probabilities of the targets, entropies, top ids, their log probabilities."""
    m = z.max(dim=1, keepdim=True).values
    d = z - m
    e = torch.exp(d)
    s = e.sum(dim=1, keepdim=True)
    log_s = torch.log(s)
    entropy = log_s - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(dim=1, keepdim=True) / s
    logprobs = torch.gather(d, 1, targets.long().unsqueeze(1)) - log_s
    if top:
        # a logit's bits in an order that whole numbers have too, and below them its id, the lowest ahead
        bits = (z + 0.0).view(torch.int32).long()
        key = (torch.where(bits < 0, -0x80000000 - bits - 1, bits) << 32) + (0xFFFFFFFF - torch.arange(z.shape[1], device=z.device))
        ids = 0xFFFFFFFF - (torch.topk(key, top, dim=1).values & 0xFFFFFFFF)
    else:
        ids = torch.empty(z.shape[0], 0, dtype=torch.int64, device=z.device)
    return logprobs.squeeze(1), entropy.squeeze(1), ids.to(torch.int32), torch.gather(d, 1, ids) - log_s


def _run_plain(state):
    case = state["case"]
    if case["op"] == "copy":
        for name in ("k", "v"):
            src = torch.tensor(state["src"], device=DEVICE)
            dst = torch.tensor(state["dst"], device=DEVICE)
            state[name][:, dst] = state[name][:, src]
        if "state" in state:
            src = torch.tensor(state["state_src"], device=DEVICE)
            dst = torch.tensor(state["state_dst"], device=DEVICE)
            state["state"][:, dst] = state["state"][:, src]
        return _buffers(state)
    rows = max(1, PIECE // case["vocab"])
    if case["op"] == "head":
        weight = state["weight"].float().t()
    parts = []
    for r in range(0, case["rows"], rows):
        if case["op"] == "logits":
            z = state["logits"][r:r + rows].float()
        else:
            z = state["x"][r:r + rows].float() @ weight
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
        parts.append(_plain_rows(z, state["targets"][r:r + rows], case["top"]))
    return _outputs(*(torch.cat(p) for p in zip(*parts)))


# ---- the same in 64 bits, from the definition ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        # nothing is computed: every row of the result is a row of what was there
        out = {}
        for name, src, dst in (("k", "src", "dst"), ("v", "src", "dst"), ("state", "state_src", "state_dst")):
            if name in s:
                came_from = list(range(s[name].shape[1]))
                for a, b in zip(s[src], s[dst]):
                    came_from[b] = a
                out[name] = s[name].index_select(1, torch.tensor(came_from, device=DEVICE))
        return out
    lps, entropies, ids, tops = [], [], [], []
    for r in range(0, case["rows"], max(1, PIECE // case["vocab"])):
        some = slice(r, r + max(1, PIECE // case["vocab"]))
        if case["op"] == "logits":
            z = s["logits"][some].double()
        else:
            z = torch.cat([s["x"][some].double() @ w.double().t() for w in s["weight"].split(32768)], dim=1)
            if case["cap"]:
                # tanh(y) = 1 - 2 / (1 + exp(2 y))
                z = case["cap"] * (1.0 - 2.0 / (1.0 + torch.exp(z * (2.0 / case["cap"]))))
        order = torch.sort(z, dim=1, descending=True, stable=True)
        log_p = z - torch.logsumexp(z, dim=1, keepdim=True)
        p = torch.exp(log_p)
        entropies.append(-(p * log_p.masked_fill(p == 0, 0.0)).sum(dim=1))
        lps.append(log_p[torch.arange(z.shape[0], device=DEVICE), s["targets"][some].long()])
        ids.append(order.indices[:, :case["top"]].to(torch.int32))
        tops.append(torch.gather(log_p, 1, order.indices[:, :case["top"]]))
        del z, order, log_p, p
    return _outputs(torch.cat(lps), torch.cat(entropies), torch.cat(ids), torch.cat(tops))


def work(case):
    if case["op"] == "copy":
        moved = 2 * case["rows"] * case["sets"] * case["heads"] * case["page"] * case["dim"] * BYTES[case["x"]]
        read = moved
        if case["state_heads"]:
            one = case["sets"] * case["state_heads"] * case["state_dim"] ** 2 * 4
            moved, read = moved + case["rows"] * one, read + one
        return {"bytes": read + moved, "flops": 0}
    rows, vocab = case["rows"], case["vocab"]
    written = rows * (4 + 8 + 8 * case["top"])
    if case["op"] == "logits":
        return {"bytes": rows * vocab * BYTES[case["x"]] + written, "flops": 6 * rows * vocab}
    return {"bytes": (rows + vocab) * case["in"] * BYTES[case["x"]] + written, "flops": 2 * rows * case["in"] * vocab}
