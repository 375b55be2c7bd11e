"""What the speed of the 4-bit weight operators is measured on.

Weights are e2m1 codes with one power-of-two scale a group of 32 columns, rows of activations bfloat16, float32 or e4m3 with
such scales.  Four operators, by the case's "op":

    norm      h = residual + first(x); second(h) as e4m3 rows with scales      (what feeds a prompt's products)
    vector    few rows of bfloat16 or float32 times a 4-bit matrix            (decode steps, the output head)
    product   e4m3 rows times a 4-bit matrix                                  (prompts)
    pack      a bfloat16 matrix to 4 bits, and the values those stand for     (loading a model)

Cases' sizes are those of the Gemma 2 2B, 9B and 27B shapes, and odd ones.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
GROUP = 32
BLOCK = 128                       # columns are padded to whole blocks of four groups
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
CAP = 30.0
BYTES = {"bfloat16": 2, "float32": 4}


def listed():
    return [
        # the shortest step that is a prompt and not a decode step, in the 2B shape
        {"name": "norm_short", "op": "norm", "rows": 17, "width": 2304, "x": "bfloat16", "first": True},
        # a prompt of 2,048 tokens between attention and feed-forward, 2B shape
        {"name": "norm_prompt", "op": "norm", "rows": 2048, "width": 2304, "x": "bfloat16", "first": True},
        # the 27B shape's width and a long prompt; a float32 branch without a norm of its own
        {"name": "norm_long", "op": "norm", "rows": 8192, "width": 4608, "x": "float32", "first": False},
        # one token through the 2B shape's q/k/v matrix: latency
        {"name": "vector_one", "op": "vector", "rows": 1, "in": 2304, "out": 4096, "x": "bfloat16", "form": "plain"},
        # decode at batch 8, gate and up of the 2B shape
        {"name": "vector_gated", "op": "vector", "rows": 8, "in": 2304, "out": 9216, "x": "bfloat16", "form": "gated"},
        # the 32-bit type and sizes that nothing divides
        {"name": "vector_odd", "op": "vector", "rows": 5, "in": 1003, "out": 777, "x": "float32", "form": "plain"},
        # the output head of the 2B shape at batch 16: the largest matrix a decode step reads
        {"name": "vector_head", "op": "vector", "rows": 16, "in": 2304, "out": 256000, "x": "bfloat16", "form": "head"},
        # a ragged step of several short prompts, sizes that nothing divides
        {"name": "product_odd", "op": "product", "rows": 333, "in": 1003, "out": 777, "form": "plain"},
        # a prompt of 2,048 tokens, gate and up of the 2B shape, result in 8 bits for the matrix behind
        {"name": "product_gated", "op": "product", "rows": 2048, "in": 2304, "out": 9216, "form": "gated"},
        # a long prompt through the 27B shape's last feed-forward matrix
        {"name": "product_long", "op": "product", "rows": 8192, "in": 36864, "out": 4608, "form": "plain"},
        # loading: a small odd matrix, and the 27B shape's gate or up matrix
        {"name": "pack_odd", "op": "pack", "out": 777, "in": 1003},
        {"name": "pack_matrix", "op": "pack", "out": 36864, "in": 4608},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "vector", "vector", "product", "product", "pack"])
    if op == "norm":
        return {"op": op, "rows": _spread(rng, 1, 8192), "width": _spread(rng, 64, 4608), "x": rng.choice(["bfloat16", "float32"]),
                "first": rng.random() < 0.5}
    if op == "vector":
        form = rng.choice(["plain", "plain", "gated", "head"])
        width, out = _spread(rng, 100, 14336), _spread(rng, 100, 16384)
        if rng.random() < 0.5:
            width, out = max(64, width // 64 * 64), max(64, out // 64 * 64)
        return {"op": op, "rows": rng.randint(1, 16), "in": width, "out": out, "x": rng.choice(["bfloat16", "bfloat16", "float32"]), "form": form}
    if op == "product":
        width, out = _spread(rng, 100, 14336), _spread(rng, 100, 14336)
        if rng.random() < 0.5:
            width, out = max(64, width // 64 * 64), max(64, out // 64 * 64)
        return {"op": op, "rows": _spread(rng, 17, 4096), "in": width, "out": out, "form": rng.choice(["plain", "gated"])}
    return {"op": op, "out": _spread(rng, 64, 16384), "in": _spread(rng, 64, 4608)}


# ---- the formats, in elementary operations on 32-bit values ----

def _groups(v, multiple):
    """[rows, columns] -> [rows, groups, 32], zeros up to a whole multiple of columns."""
    rows, cols = v.shape
    pad = -cols % multiple
    if pad:
        v = torch.nn.functional.pad(v, (0, pad))
    return v.reshape(rows, -1, GROUP)


def _scale_codes(groups, top):
    """The smallest power of two that brings a group's largest value to at most `top`, as exponent + 127."""
    amax = groups.abs().amax(dim=-1)
    mantissa, exponent = torch.frexp(amax)                 # amax = mantissa 2^exponent, mantissa in [0.5, 1)
    top_m, top_e = math.frexp(top)
    e = exponent - top_e + (mantissa > top_m).to(torch.int32)
    return torch.where(amax > 0, e + 127, torch.zeros_like(e)).clamp(0, 254)


def _power(codes):
    return torch.ldexp(torch.ones((), dtype=torch.float32, device=codes.device), codes.to(torch.int32) - 127)


def _to_e2m1(v):
    """Codes 0 to 15 of scaled values, to nearest, ties to the even code."""
    a = v.abs()
    c = (a > 0.25).to(torch.uint8)
    for bound, even in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += (a >= bound) if even else (a > bound)
    return c + 8 * (v < 0).to(torch.uint8)


def _from_e2m1(codes):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
    return table[codes.long()]


def _pack(weight):
    """float32 [out, in] -> codes [out, groups, 32] (not yet two a byte) and scale codes [out, groups]."""
    groups = _groups(weight, GROUP)
    scales = _scale_codes(groups, 6.0)
    return _to_e2m1(groups * torch.ldexp(torch.ones((), device=weight.device), 127 - scales).unsqueeze(-1)), scales.to(torch.uint8)


def _values8(rows):
    """float32 rows -> e4m3 values [rows, width] and scale codes [rows, blocks, 4]."""
    groups = _groups(rows, BLOCK)
    scales = _scale_codes(groups, 448.0)
    scaled = groups * torch.ldexp(torch.ones((), device=rows.device), 127 - scales).unsqueeze(-1)
    values = scaled.to(torch.float8_e4m3fn).reshape(rows.shape[0], -1)[:, :rows.shape[1]]
    return values, scales.to(torch.uint8).reshape(rows.shape[0], -1, 4)


def _norm(v, weight, eps):
    return v / torch.sqrt((v * v).mean(dim=-1, keepdim=True) + eps) * (1.0 + weight.float())


def _weight32(state):
    """The packed matrix as float32 [out, in]."""
    out, cols = state["codes"].shape[0], state["columns"]
    codes = torch.stack((state["codes"] & 15, state["codes"] >> 4), dim=-1).reshape(out, -1, GROUP)
    return (_from_e2m1(codes) * _power(state["scales"]).unsqueeze(-1)).reshape(out, -1)[:, :cols]


def _finish(y, form):
    """What follows the sums of a product."""
    if form == "gated":
        g, u = y.chunk(2, dim=-1)
        return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g))) * u
    return CAP * torch.tanh(y / CAP) if form == "head" else y


# ---- inputs ----

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32)


def _activations(gen, rows, width):
    """Rows as a norm leaves them: unit size, a few columns far larger, the row's scale spread."""
    x = _normal(gen, rows, width)
    loud = torch.rand(width, generator=gen, device=DEVICE) < 0.01
    x *= torch.where(loud, 12.0, 1.0)
    return x * torch.exp(0.5 * _normal(gen, rows, 1))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    state = {"case": case}
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        state["x"] = _activations(gen, rows, width).to(getattr(torch, case["x"]))
        state["residual"] = 4.0 * _normal(gen, rows, width)
        state["first"] = (0.2 * _normal(gen, width)).to(torch.bfloat16) if case["first"] else None
        state["second"] = (0.2 * _normal(gen, width)).to(torch.bfloat16)
        state["sum"] = torch.empty_like(state["residual"])
        return state
    out = case["out"] * (2 if case.get("form") == "gated" else 1)
    weight = (0.02 * _normal(gen, out, case["in"])).to(torch.bfloat16)
    if case["op"] == "pack":
        state["weight"] = weight
        return state
    state["columns"] = case["in"]
    codes, scales = _pack(weight.float())
    codes = codes.reshape(out, -1)
    state["codes"] = (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous()
    state["scales"] = scales
    x = _activations(gen, case["rows"], case["in"])
    if case["op"] == "vector":
        state["x"] = x.to(getattr(torch, case["x"]))
    else:
        state["values"], state["row_scales"] = _values8(x)
    if own:
        from rust_deeplearning_b200.kernels import ops
        state["matrix"] = ops.mx4_weight(state["codes"], state["scales"], case["in"], gated=case["form"] == "gated")
        if case["op"] == "product":
            groups = -(-case["in"] // GROUP)
            state["packed"] = ops.mx8_rows(state["values"].contiguous(), state["row_scales"].reshape(case["rows"], -1)[:, :groups].contiguous())
    return state


# ---- one pass ----

def _rows8(rows):
    """e4m3 rows as what they stand for: values in 8 bits and powers of two."""
    values, scales = rows
    return {"values": values, "scales": scales.view(torch.float8_e8m0fnu)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from rust_deeplearning_b200.kernels import ops
    case = state["case"]
    form = case.get("form")
    if case["op"] == "norm":
        first = ops.NormParams(state["first"], 1e-6, 1.0) if state["first"] is not None else None
        rows = ops.norm_mx8(state["x"], first=first, residual=state["residual"], second=ops.NormParams(state["second"], 1e-6, 1.0),
                            residual_out=state["sum"])
        return dict(_rows8((rows.values, rows.scales)), sum=state["sum"])
    if case["op"] == "pack":
        return ops.expand_mx4(ops.pack_mx4(state["weight"]))
    if case["op"] == "vector":
        if form == "gated":
            return ops.linear_gated_mx4(state["x"], state["matrix"], "gelu_pytorch_tanh")
        if form == "head":
            return ops.linear_mx4(state["x"], state["matrix"], out_dtype=torch.float32, softcap=CAP)
        return ops.linear_mx4(state["x"], state["matrix"])
    if form == "gated":
        rows = ops.linear_gated_mx4(state["packed"], state["matrix"], "gelu_pytorch_tanh", out_mx8=True)
        return _rows8((rows.values, rows.scales))
    return ops.linear_mx4(state["packed"], state["matrix"])


def _run_plain(state):
    case = state["case"]
    form = case.get("form")
    if case["op"] == "norm":
        branch = state["x"].float()
        if state["first"] is not None:
            branch = _norm(branch, state["first"], 1e-6)
        h = state["residual"] + branch
        return dict(_rows8(_values8(_norm(h, state["second"], 1e-6))), sum=h)
    if case["op"] == "pack":
        codes, scales = _pack(state["weight"].float())
        return (_from_e2m1(codes) * _power(scales).unsqueeze(-1)).reshape(case["out"], -1)[:, :case["in"]].to(torch.bfloat16)
    if case["op"] == "vector":
        x = state["x"].float()
    else:
        groups = _groups(state["values"].float(), BLOCK)
        x = (groups * _power(state["row_scales"].reshape(case["rows"], -1)).unsqueeze(-1)).reshape(case["rows"], -1)[:, :case["in"]]
    y = _finish(x @ _weight32(state).t(), form)
    if case["op"] == "product" and form == "gated":
        return _rows8(_values8(y))
    return y if form == "head" or state.get("x") is not None and state["x"].dtype is torch.float32 else y.to(torch.bfloat16)


# ---- the same in 64 bits, from the definition ----

def _grid(bits, bias, top):
    """Every value of a small float format with `bits` of mantissa, from zero up to `top`, in order."""
    step = 2.0 ** -bits
    values = [m * step * 2.0 ** (1 - bias) for m in range(2 ** bits)]
    e = 1 - bias
    while values[-1] < top:
        values += [(1 + m * step) * 2.0 ** e for m in range(2 ** bits)]
        e += 1
    return [v for v in values if v <= top]


def _nearest(v, grid):
    """Values of v on the grid, to nearest, ties to the even index."""
    grid = torch.tensor(grid, dtype=torch.float64, device=v.device)
    a = v.abs().contiguous()
    hi = torch.searchsorted(grid, a).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    down, up = a - grid[lo], grid[hi] - a
    take_hi = (up < down) | ((up == down) & (hi % 2 == 0))
    return torch.where(take_hi, grid[hi], grid[lo]) * torch.sign(v)


def _quantised(v, top, grid, multiple):
    """float64 rows -> (values before their scale, scales): [rows, groups, 32] and [rows, groups]."""
    rows, cols = v.shape
    g = torch.zeros(rows, -(-cols // multiple) * multiple, dtype=torch.float64, device=v.device)
    g[:, :cols] = v
    g = g.reshape(rows, -1, GROUP)
    amax = g.abs().amax(dim=-1)
    e = torch.ceil(torch.log2(amax / top)).clamp(min=-127.0)
    e = torch.where(amax <= top * torch.exp2(e - 1), e - 1, e)          # a logarithm that was rounded up
    e = torch.where(amax > top * torch.exp2(e), e + 1, e).clamp(min=-127.0)
    scale = torch.exp2(e)
    return _nearest(g / scale.unsqueeze(-1), grid), scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["first"] is not None:
            h = h * torch.rsqrt(h.pow(2).sum(-1, keepdim=True) / case["width"] + 1e-6) * (s["first"].double() + 1.0)
        h = h + s["residual"].double()
        y = h * torch.rsqrt(h.pow(2).sum(-1, keepdim=True) / case["width"] + 1e-6) * (s["second"].double() + 1.0)
        q, scale = _quantised(y, 448.0, _grid(3, 7, 448.0), BLOCK)
        return {"values": q.reshape(case["rows"], -1)[:, :case["width"]], "scales": scale.reshape(case["rows"], -1, 4), "sum": h}
    if case["op"] == "pack":
        parts = []
        for w in s["weight"].split(4096):
            q, scale = _quantised(w.double(), 6.0, _grid(1, 1, 6.0), GROUP)
            parts.append((q * scale.unsqueeze(-1)).reshape(w.shape[0], -1)[:, :case["in"]])
        return torch.cat(parts)
    if case["op"] == "vector":
        x = s["x"].double()
    else:
        x = s["values"].double() * torch.exp2(s["row_scales"].double() - 127.0).reshape(case["rows"], -1).repeat_interleave(GROUP, dim=1)[:, :case["in"]]
    table = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    parts = []
    for codes, scales in zip(s["codes"].split(16384), s["scales"].split(16384)):
        nibbles = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.int64, device=x.device)
        nibbles[:, 0::2], nibbles[:, 1::2] = codes.long() % 16, codes.long() // 16
        w = table[nibbles % 8] * (1.0 - 2.0 * (nibbles // 8)) * torch.exp2(scales.double() - 127.0).repeat_interleave(GROUP, dim=1)
        parts.append(x @ w[:, :case["in"]].t())
    y = torch.cat(parts, dim=1)
    if case["form"] == "head":
        return CAP * torch.tanh(y / CAP)
    if case["form"] == "gated":
        n = case["out"]
        g, u = y[:, :n], y[:, n:]
        y = u * g / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))
        if case["op"] == "product":
            q, scale = _quantised(y, 448.0, _grid(3, 7, 448.0), BLOCK)
            return {"values": q.reshape(case["rows"], -1)[:, :n], "scales": scale.reshape(case["rows"], -1, 4)}
    return y


def work(case):
    if case["op"] == "norm":
        n, groups = case["rows"] * case["width"], case["rows"] * -(-case["width"] // GROUP)
        return {"bytes": n * (BYTES[case["x"]] + 4 + 4 + 1) + groups + 4 * case["width"], "flops": 10 * n}
    out, width = case["out"] * (2 if case.get("form") == "gated" else 1), case["in"]
    groups = -(-width // GROUP)
    packed = out * -(-width // 2) + out * groups
    if case["op"] == "pack":
        return {"bytes": out * width * 2 + 2 * packed + out * width * 2, "flops": 4 * out * width}
    rows = case["rows"]
    read = rows * width * BYTES[case["x"]] if case["op"] == "vector" else rows * (width + groups)
    if case["op"] == "product":
        written = rows * case["out"] * 2 if case["form"] == "plain" else rows * (case["out"] + -(-case["out"] // GROUP))
    else:
        written = rows * case["out"] * (4 if case["form"] == "head" or case["x"] == "float32" else 2)
    return {"bytes": packed + read + written, "flops": 2 * rows * out * width}
