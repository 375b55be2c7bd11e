"""4-bit weights, 8-bit rows and what is computed with them, against float64 (tests/plain_microscaling.py).

Tolerances, from the formats and the arithmetic:
  rounding to 4 or 8 bits of values that are given is exact: the same values, bit for bit;
  a norm's result in 8 bits is off by half a step (2^-4 of the value, or 2^-10 of the scale where the value is small) and by what
  float32 statistics move it (2^-18 of the value, generously);
  a sum of K products in float: each of G groups is summed by the tensor core (32 terms, 2^-23 each) and joins a float sum:
  (64 + G) 2^-23 of the sum of magnitudes; float32 rows enter with 22 bits: 2^-21 of the same more;
  a bfloat16 result: 2^-8 of the value (and of the largest value of the row where a gate's hardware tanh, 2^-11, came before)."""
import numpy as np
import pytest
import torch

import plain_microscaling as plain
from rust_deeplearning_b200.kernels import library, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def f64(t):
    return t.detach().double().cpu().numpy()


def rows_for(m, k, kind, seed):
    """Rows with quiet and loud ones, a row of zeros, a group of zeros."""
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(seed))
    x *= torch.exp2(torch.arange(m).float() % 5 * 3 - 6)[:, None]
    if m > 2:
        x[m // 2] = 0
    x[:, 32:64] = 0
    x = x.to(DEV)
    if kind == "mx8":
        r = ops.pack_mx8(x)
        return r, f64(r.dequantise())
    x = x.to(torch.bfloat16 if kind == "bfloat16" else torch.float32)
    return x, f64(x)


def sum_tolerance(x, w, kind):
    groups = -(-x.shape[1] // 32)
    return (np.abs(x) @ np.abs(w).T) * ((64 + groups) * 2.0 ** -23 + (2.0 ** -21 if kind == "float32" else 0.0))


def check(got, want, tol, what):
    err = np.abs(f64(got) - want) - tol
    assert np.isfinite(f64(got)).all(), f"{what}: non-finite output"
    assert (err <= 0).all(), f"{what}: {float(err.max()):.3e} beyond the tolerance"


# ---- the formats ----

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,columns,gated", [(1, 1, False), (3, 31, False), (17, 33, False), (16, 128, False), (50, 1003, False),
                                                (30, 260, True), (2, 32, True)])
def test_pack_mx4(rows, columns, gated, dtype):
    w = rnd((rows, columns), dtype, rows, 0.02)
    w *= torch.exp2(torch.randint(-30, 30, (rows, 1), generator=torch.Generator().manual_seed(1)).to(DEV)).to(dtype)
    w[rows // 2, :32] = 0
    want, codes = plain.quantise(f64(w), plain.E2M1)
    packed = ops.pack_mx4(w, gated)
    assert np.array_equal(f64(ops.expand_mx4(packed, torch.float32)), want)
    assert np.array_equal(f64(ops.expand_mx4(packed)), want)             # exact in bfloat16 too
    # the scales, and zeros in the padding
    by_row = packed.scales.transpose(2, 3).reshape(packed.tiles, -1, 128, 4).transpose(1, 2).reshape(packed.tiles * 128, -1).cpu().numpy()
    place = np.arange(rows)
    if gated:
        o = place % (rows // 2)
        place = o // 16 * 32 + place // (rows // 2) * 16 + o % 16
    assert np.array_equal(by_row[place, :codes.shape[1]], codes)
    by_row[place, :codes.shape[1]] = 0
    assert not by_row.any()
    assert int(packed.codes.count_nonzero()) <= rows * -(-columns // 2)


def test_pack_mx4_ties_and_edges():
    """Every tie between two codes, both signs, the largest value, a group that is not finite, the smallest scales."""
    w = torch.zeros((6, 64), device=DEV)
    w[0, :16] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6.0])
    w[1, 0], w[1, 32] = float("inf"), 1.0
    w[2, 5] = float("nan")
    w[3, 0], w[3, 1] = 2.0 ** -130, 2.0 ** -149
    w[4, 0], w[4, 1] = 3.0e38, 1.0
    w[5, 0], w[5, 32] = 6.0, 6.0000005
    want, codes = plain.quantise(f64(w), plain.E2M1)
    got = f64(ops.expand_mx4(ops.pack_mx4(w), torch.float32))
    with np.errstate(over="ignore"):
        want = want.astype(np.float32)                                   # 4 x 2^126 is not a float32: it comes back as an infinity
    assert np.array_equal(got[[0, 3, 4, 5]], want[[0, 3, 4, 5]])
    for r in (1, 2):
        assert np.isnan(got[r, :32]).all() and np.array_equal(got[r, 32:], want[r, 32:])
    assert codes[5, 0] == 127 and codes[5, 1] == 128


def test_mx4_weight_from_codes_is_the_packed_one():
    for rows, columns, gated in ((20, 75, False), (26, 128, True)):
        w = rnd((rows, columns), torch.float32, 3)
        packed = ops.pack_mx4(w, gated)
        q, codes = plain.quantise(f64(w), plain.E2M1)
        scale = 2.0 ** (codes - 127.0)
        wide = plain.groups_of(q) / scale[..., None]
        nib = (plain.nearest(wide, plain.E2M1) + 8 * (np.signbit(wide) & (wide != 0))).reshape(rows, -1)[:, :columns + columns % 2].astype(np.uint8)
        if columns % 2:
            nib[:, -1] = 13                                              # what lies behind the last column does not count
        given = ops.mx4_weight(torch.from_numpy(nib[:, 0::2] | nib[:, 1::2] << 4).to(DEV), torch.from_numpy(codes.astype(np.uint8)).to(DEV), columns, gated)
        assert torch.equal(given.scales, packed.scales)
        assert np.array_equal(f64(ops.expand_mx4(given, torch.float32)), q)


@pytest.mark.parametrize("rows,columns,gated", [(1, 1, False), (3, 33, False), (130, 257, False), (2, 31, True), (34, 300, True), (270, 1003, True)])
def test_layout_of_given_codes_and_rows(rows, columns, gated):
    """Any strides and starts: views of wider tensors, every second column, a start at an odd byte; whatever the padding held does not enter."""
    groups, used = -(-columns // 32), -(-columns // 2)
    g = torch.Generator().manual_seed(70)
    codes = torch.randint(0, 256, (rows, used), generator=g, dtype=torch.uint8)          # an odd row's last half byte holds something
    scales = torch.randint(100, 140, (rows, groups), generator=g, dtype=torch.uint8)
    nib = torch.stack([codes & 15, codes >> 4], dim=-1).view(rows, -1)[:, :columns].numpy()
    table = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6])
    want = table[nib] * np.repeat(2.0 ** (scales.numpy().astype(np.float64) - 127), 32, axis=1)[:, :columns]
    codes, scales = codes.to(DEV), scales.to(DEV)
    wide = torch.full((rows, used + 5), 255, dtype=torch.uint8, device=DEV)
    wide[:, 3:3 + used] = codes
    apart = torch.full((rows, 2 * used), 255, dtype=torch.uint8, device=DEV)
    apart[:, ::2] = codes
    padded = torch.full((rows, groups * 16), 255, dtype=torch.uint8, device=DEV)
    padded[:, :used] = codes
    wide_scales = torch.cat([scales, scales], dim=1)[:, :groups]
    first = None
    for c, s in ((codes, scales), (wide[:, 3:3 + used], wide_scales), (apart[:, ::2], scales), (padded, scales), (codes[:1].expand(rows, used) if rows == 1 else codes, scales)):
        w = ops.mx4_weight(c, s, columns, gated)
        assert np.array_equal(f64(ops.expand_mx4(w, torch.float32)), want)
        first = first or w
        assert torch.equal(w.codes, first.codes) and torch.equal(w.scales, first.scales)
    assert int((first.codes != 0).sum()) <= rows * used                  # nothing in the padding
    values = torch.randint(0, 120, (rows, columns), generator=g, dtype=torch.uint8).to(DEV)
    around = torch.full((rows, columns + 3), 120, dtype=torch.uint8, device=DEV)
    around[:, 1:1 + columns] = values
    for v in (values, around[:, 1:1 + columns]):
        r = ops.mx8_rows(v.view(torch.float8_e4m3fn), scales)
        assert torch.equal(r.values.view(torch.uint8), values) and torch.equal(r.scales.reshape(rows, -1)[:, :groups], scales)
        assert not r._data.view(torch.uint8)[:rows, columns:].any() and not r.scales.reshape(rows, -1)[:, groups:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,columns", [(1, 1), (5, 31), (3, 128), (7, 1003), (2, 8192), (2, 8197), (3, 20000)])
def test_pack_mx8(rows, columns, dtype):
    x = rnd((rows, columns), dtype, 5, 3.0)
    x[0, :1] = 448.0
    want, codes = plain.quantise(f64(x), plain.E4M3)
    got = ops.pack_mx8(x)
    assert np.array_equal(f64(got.dequantise()), want)
    padded = np.zeros((rows, -(-columns // 128) * 4))
    padded[:, :codes.shape[1]] = codes
    assert np.array_equal(got.scales.reshape(rows, -1).cpu().numpy(), padded)
    again = ops.mx8_rows(got.values.contiguous(), got.scales.reshape(rows, -1)[:, :codes.shape[1]].contiguous())
    assert torch.equal(again.values.view(torch.uint8), got.values.view(torch.uint8)) and torch.equal(again.scales, got.scales)


def test_pack_mx8_groups_that_are_not_finite():
    x = rnd((3, 96), torch.float32, 6)
    x[0, 40], x[1, 0], x[1, 95] = float("inf"), float("nan"), float("-inf")
    got = f64(ops.pack_mx8(x).dequantise())
    want = plain.quantise(f64(x), plain.E4M3)[0]
    bad = np.zeros((3, 3), bool)
    bad[0, 1] = bad[1, 0] = bad[1, 2] = True
    bad = np.repeat(bad, 32, axis=1)
    assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], want[~bad])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width", [(1, 64), (5, 80), (3, 131), (4, 2304), (2, 4608), (3, 8192), (2, 8196), (2, 10007)])
def test_norm_mx8(rows, width, dtype):
    x, res = rnd((rows, width), dtype, 1, 3.0), rnd((rows, width), torch.float32, 4, 2.0)
    w1 = ops.NormParams(rnd((width,), dtype, 2, 0.5), 1e-5, 1.0)
    w2 = ops.NormParams(rnd((width,), torch.float32, 3, 0.5), 1e-6, 0.0)
    for first, second, with_res in ((w1, w2, True), (None, w2, True), (w1, None, True), (None, w2, False), (w1, w2, False)):
        h = plain.rms_norm(f64(x), f64(w1.weight), 1e-5, 1.0) if first else f64(x)
        own = res.clone() if with_res else None
        h = h + f64(res) if with_res else h
        y = plain.rms_norm(h, f64(w2.weight), 1e-6, 0.0) if second else h
        got = ops.norm_mx8(x, first=first, residual=own, second=second)
        scale = 2.0 ** (got.scales.reshape(rows, -1).cpu().numpy().astype(np.float64) - 127)
        per_value = np.repeat(scale, 32, axis=1)[:, :width]
        check(got.dequantise(), y, np.abs(y) * (2.0 ** -4 + 2.0 ** -18) + per_value * 2.0 ** -10, "rows")
        amax = np.abs(plain.groups_of(y)).max(-1)
        used = scale[:, :amax.shape[1]]
        assert (amax <= 448 * used * (1 + 2.0 ** -18)).all() and (amax >= 224 * used * (1 - 2.0 ** -18)).all()
        if with_res:
            check(own, h, 2.0 ** -18 * np.abs(h) + 2.0 ** -18 * np.abs(f64(res)), "sum")
            out = torch.full_like(own, float("nan"))
            keep = res.clone()
            again = ops.norm_mx8(x, first=first, residual=keep, second=second, residual_out=out)
            assert torch.equal(out, own) and torch.equal(keep, res) and torch.equal(again.values.view(torch.uint8), got.values.view(torch.uint8))


def test_norm_mx8_is_the_same_row_by_row():
    x, res = rnd((9, 2304), torch.bfloat16, 1), rnd((9, 2304), torch.float32, 2)
    w = ops.NormParams(rnd((2304,), torch.bfloat16, 3), 1e-6, 1.0)
    whole = ops.norm_mx8(x, first=w, residual=res.clone(), second=w)
    for r in range(9):
        one = ops.norm_mx8(x[r:r + 1], first=w, residual=res[r:r + 1].clone(), second=w)
        assert torch.equal(one.values.view(torch.uint8), whole.values[r:r + 1].view(torch.uint8)) and torch.equal(one.scales[0], whole.scales[r])


def test_norm_mx8_beyond_32_bits():
    """2.4e9 values: the last rows lie behind what 32 bits can count."""
    rows, width = 600_000, 4096
    x = torch.zeros((rows, width), dtype=torch.bfloat16, device=DEV)
    x[-3:] = rnd((3, width), torch.bfloat16, 8)
    got = ops.pack_mx8(x)
    want = ops.pack_mx8(x[-3:].clone())
    assert torch.equal(got.values[-3:].view(torch.uint8), want.values.view(torch.uint8)) and torch.equal(got.scales[-3:], want.scales)


# ---- the products ----

SHAPES = [(1, 1, 1), (1, 3, 32), (2, 16, 33), (5, 777, 1003), (8, 100, 128), (9, 17, 2304), (16, 333, 640), (16, 40, 14336)]


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "mx8"])
@pytest.mark.parametrize("m,n,k", [(16, 19001, 4700), (9, 300, 36865)])
def test_few_rows_longer_than_shared_memory(m, n, k, kind):
    """The blocks of the rows pass through shared memory in turn, again for each tile; a row that is not finite keeps to itself."""
    w = ops.pack_mx4(rnd((n, k), torch.float32, 40, 0.05))
    x, x64 = rows_for(m, k, kind, 41)
    w64 = f64(ops.expand_mx4(w, torch.float32))
    want, tol = x64 @ w64.T, sum_tolerance(x64, w64, kind)
    whole = ops.linear_mx4(x, w, out_dtype=torch.float32)
    check(whole, want, tol, "float32")
    if kind != "mx8":
        x[2, k - 1] = float("nan")
        got = ops.linear_mx4(x, w, out_dtype=torch.float32)
        assert got[2].isnan().all() and torch.equal(torch.cat([got[:2], got[3:]]), torch.cat([whole[:2], whole[3:]]))


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "mx8"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_few_rows(m, n, k, kind):
    w = ops.pack_mx4(rnd((n, k), torch.float32, 7, 0.05))
    x, x64 = rows_for(m, k, kind, 8)
    w64 = f64(ops.expand_mx4(w, torch.float32))
    want = x64 @ w64.T
    tol = sum_tolerance(x64, w64, kind)
    check(ops.linear_mx4(x, w, out_dtype=torch.float32), want, tol, "float32")
    check(ops.linear_mx4(x, w, out_dtype=torch.bfloat16), want, tol + np.abs(want) * 2.0 ** -8, "bfloat16")


@pytest.mark.parametrize("m,n,k", [(17, 1, 1), (17, 40, 32), (33, 2304, 2304), (64, 4096, 1280), (100, 777, 1003), (128, 20000, 160), (127, 19001, 300), (130, 777, 1003), (128, 256, 128), (129, 257, 300), (300, 130, 2304), (40, 600, 14336)])
def test_many_rows(m, n, k):
    w = ops.pack_mx4(rnd((n, k), torch.float32, 7, 0.05))
    x, x64 = rows_for(m, k, "mx8", 8)
    w64 = f64(ops.expand_mx4(w, torch.float32))
    want = x64 @ w64.T
    tol = sum_tolerance(x64, w64, "mx8")
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    check(ops.linear_mx4(x, w, out_dtype=torch.float32, status=status), want, tol, "float32")
    check(ops.linear_mx4(x, w, status=status), want, tol + np.abs(want) * 2.0 ** -8, "bfloat16")
    assert status.item() == 0


@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_more_rows_of_a_tensor(kind):
    w = ops.pack_mx4(rnd((70, 200), torch.float32, 7, 0.05))
    x, x64 = rows_for(37, 200, kind, 8)
    w64 = f64(ops.expand_mx4(w, torch.float32))
    check(ops.linear_mx4(x, w, out_dtype=torch.float32), x64 @ w64.T, sum_tolerance(x64, w64, kind), "rows")


def norm64(v, p):
    w = f64(p.weight) + p.offset
    return v / np.sqrt((v ** 2).mean(-1, keepdims=True) + p.eps) * w


@pytest.mark.parametrize("m", [1, 4, 8])
@pytest.mark.parametrize("width,k_in,n_out", [(2304, 2048, 4096), (1000, 1101, 20003), (3584, 520, 600), (640, 4608, 131)])
def test_deferred_norms(m, width, k_in, n_out):
    """A branch's product and the product behind the two norms that follow it, without a kernel between, and each of the two with a
    bfloat16 weight on the other side.

    The tolerance follows the roundings to bfloat16, each 2^-8 of what is rounded: the branch times its column factors, both halves of the
    operand, the row that goes into parts; the row factors move by what the branch's rounding adds to the stream's norm."""
    x, x64 = rows_for(m, k_in, "bfloat16", 50)
    if m > 2:
        x[m // 2] = 1.0
        x64 = f64(x)
    w_p, w_c = ops.pack_mx4(rnd((width, k_in), torch.float32, 51, 0.2)), ops.pack_mx4(rnd((n_out, width), torch.float32, 52, 0.2))
    w_gu = ops.pack_mx4(rnd((2 * 72, width), torch.float32, 53, 0.1), gated=True)
    p64, c64, gu64 = (f64(ops.expand_mx4(w, torch.float32)) for w in (w_p, w_c, w_gu))
    h = rnd((m, width), torch.float32, 54, 2.0)
    post = ops.NormParams(rnd((width,), torch.bfloat16, 55, 0.5), 1e-5, 1.0)
    then = ops.NormParams(rnd((width,), torch.float32, 56, 0.5), 1e-6, 0.0)
    nxt = ops.NormParams(rnd((width,), torch.bfloat16, 57, 0.5), 1e-6, 1.0)
    h64, g1, g2, g3 = f64(h), f64(post.weight) + 1.0, f64(then.weight), f64(nxt.weight) + 1.0
    y = x64 @ p64.T
    added = norm64(y, post)
    new = h64 + added
    rows = norm64(new, then)
    z = rows @ c64.T
    s1 = 1 / np.sqrt((y ** 2).mean(-1, keepdims=True) + post.eps)
    s2 = 1 / np.sqrt((new ** 2).mean(-1, keepdims=True) + then.eps)
    float_y = s1 * np.abs(g1) * sum_tolerance(x64, p64, "bfloat16")
    h_tol = np.abs(added) * (2.0 ** -8 + 2.0 ** -18) + float_y + 2.0 ** -22 * (np.abs(h64) + np.abs(new))
    moved = np.linalg.norm(h_tol, axis=-1, keepdims=True) / np.linalg.norm(new, axis=-1, keepdims=True) + 2.0 ** -16
    x_tol = s2 * np.abs(g2) * (np.abs(h64) * 2.0 ** -8 + np.abs(added) * (2.0 ** -7 + 2.0 ** -15) + float_y) + np.abs(rows) * (2.0 ** -8 + moved) * (1 + 2.0 ** -7)
    z_tol = x_tol @ np.abs(c64).T + sum_tolerance(rows, c64, "bfloat16")
    bf16 = lambda want, tol: tol + (np.abs(want) + tol) * 2.0 ** -8

    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    bf_p, bf_c = ops.expand_mx4(w_p), ops.expand_mx4(w_c)                # the same values: 4 bits and a power of two are exact in bfloat16
    for wp, wc in ((w_p, w_c), (bf_p, w_c), (w_p, bf_c)):
        if type(wp) is torch.Tensor and k_in % 8:
            continue                                                     # the bfloat16 kernels' rule
        operand = ops.scaled_rows(h, then)
        branch = ops.linear_branch(x, wp, ops.BranchSink(h, post, then, operand), status=status)
        assert isinstance(branch, ops.Branch)
        h_out, next_operand = torch.empty_like(h), torch.empty_like(operand)
        d = ops.DeferredRows(branch, h_out, nxt, next_operand)
        check(ops.linear(d, wc, status=status), z, bf16(z, z_tol), "product")
        assert d.consumed
        check(h_out, new, h_tol, "stream")
        check(next_operand[:m], new * g3, np.abs(g3) * h_tol + np.abs(new * g3) * (2.0 ** -8 + 2.0 ** -15), "next operand")
        if wc is w_c:
            check(ops.linear(d, w_c, out_dtype=torch.float32, softcap=3.0, status=status), 3.0 * np.tanh(z / 3.0), z_tol + 2.0 ** -18, "soft-cap")
            v = rows @ gu64.T
            g, u = np.split(np.abs(v), 2, axis=-1)
            t = x_tol @ np.abs(gu64).T + sum_tolerance(rows, gu64, "bfloat16")
            check(ops.linear_gated(d, w_gu, "silu", status=status), plain.gated(v, "silu", 0.0),
                  2 * (g + u + 1 + t[:, :72] + t[:, 72:]) * (t[:, :72] + t[:, 72:]) + 2.0 ** -10 * np.maximum(g, 1) * (u + 1) + 2.0 ** -8 * g * u, "gated")
            chosen = torch.tensor([m - 1, 0], dtype=torch.int32, device=DEV)
            h_out2 = torch.empty_like(h)
            d2 = ops.DeferredRows(branch, h_out2, row_index=chosen)
            check(ops.linear(d2, w_c, status=status), z[[m - 1, 0]], bf16(z, z_tol)[[m - 1, 0]], "chosen rows")
            assert torch.equal(h_out2, h_out)
        d3 = ops.DeferredRows(branch, torch.empty_like(h), nxt, torch.empty_like(operand))
        check(d3.materialise(), rows, x_tol, "materialised")
    assert status.item() == 0


@pytest.mark.parametrize("m", [1, 4, 8])
def test_deferred_norms_in_front_of_many_tiles(m):
    """A block works on four tiles of weights or more, each of few products, while some of its warps still write the stream: no wait
    is in vain, and every call gives the same bits.

    The tolerance is that of test_deferred_norms."""
    width, n_out = 256, 80000
    x, _ = rows_for(m, 2048, "bfloat16", 70)
    x[x.abs().amax(1) == 0] = 1.0
    w_p, w_c = ops.pack_mx4(rnd((width, 2048), torch.float32, 71, 0.2)), ops.pack_mx4(rnd((n_out, width), torch.float32, 72, 0.2))
    h, norm = rnd((m, width), torch.float32, 73, 2.0), ops.NormParams(rnd((width,), torch.bfloat16, 74, 0.5), 1e-6, 1.0)
    x64, p64, c64 = f64(x), f64(ops.expand_mx4(w_p, torch.float32)), f64(ops.expand_mx4(w_c, torch.float32))
    h64, g = f64(h), f64(norm.weight) + 1.0
    y = x64 @ p64.T
    added = norm64(y, norm)
    new = h64 + added
    rows = norm64(new, norm)
    s1, s2 = (1 / np.sqrt((v ** 2).mean(-1, keepdims=True) + norm.eps) for v in (y, new))
    float_y = s1 * np.abs(g) * sum_tolerance(x64, p64, "bfloat16")
    h_tol = np.abs(added) * (2.0 ** -8 + 2.0 ** -18) + float_y + 2.0 ** -22 * (np.abs(h64) + np.abs(new))
    moved = np.linalg.norm(h_tol, axis=-1, keepdims=True) / np.linalg.norm(new, axis=-1, keepdims=True) + 2.0 ** -16
    x_tol = s2 * np.abs(g) * (np.abs(h64) * 2.0 ** -8 + np.abs(added) * (2.0 ** -7 + 2.0 ** -15) + float_y) + np.abs(rows) * (2.0 ** -8 + moved) * (1 + 2.0 ** -7)
    z_tol = x_tol @ np.abs(c64).T + sum_tolerance(rows, c64, "bfloat16")

    status, first = torch.zeros(1, dtype=torch.int32, device=DEV), None
    for _ in range(50):
        operand = ops.scaled_rows(h, norm)
        branch = ops.linear_branch(x, w_p, ops.BranchSink(h, norm, norm, operand), status=status)
        h_out, following = torch.empty_like(h), torch.empty_like(operand)
        z = ops.linear(ops.DeferredRows(branch, h_out, norm, following), w_c, out_dtype=torch.float32, status=status)
        got = (z, h_out, following[:m])
        assert first is None or all(torch.equal(a, b) for a, b in zip(got, first))
        first = first or got
    assert status.item() == 0
    check(first[0], rows @ c64.T, z_tol, "product")
    check(first[1], new, h_tol, "stream")


def test_deferred_norms_keep_rows_apart():
    """A row that is not finite reaches its own results only; the others have the same bits without it."""
    m, width = 5, 512
    x, h = rnd((m, 1024), torch.bfloat16, 60), rnd((m, width), torch.float32, 61)
    w_p, w_c = ops.pack_mx4(rnd((width, 1024), torch.float32, 62)), ops.pack_mx4(rnd((300, width), torch.float32, 63))
    norm = ops.NormParams(rnd((width,), torch.bfloat16, 64, 0.5), 1e-6, 1.0)

    def run():
        operand = ops.scaled_rows(h, norm)
        branch = ops.linear_branch(x, w_p, ops.BranchSink(h, norm, norm, operand))
        out = torch.empty_like(h)
        return ops.linear(ops.DeferredRows(branch, out, norm, torch.empty_like(operand)), w_c, out_dtype=torch.float32), out

    clean = run()
    x[3, 5] = float("inf")
    h[1, 7] = float("nan")
    for got, want in zip(run(), clean):
        assert torch.equal(got[[0, 2, 4]], want[[0, 2, 4]])
    z, out = run()
    assert z[1].isnan().all() and z[3].isnan().all() and out[1, 7].isnan()


def test_no_split_form_of_a_branch():
    """A matrix that no clusters share, and a gated one, say so; the plain result is delivered."""
    w = ops.pack_mx4(rnd((64, 64), torch.float32, 65))
    assert w.branch_units == 0 and ops.pack_mx4(rnd((512, 1024), torch.float32, 65), gated=True).branch_units == 0
    h, norm = rnd((2, 64), torch.float32, 66), ops.NormParams(rnd((64,), torch.bfloat16, 67), 1e-6, 1.0)
    x = rnd((2, 64), torch.bfloat16, 68)
    got = ops.linear_branch(x, w, ops.BranchSink(h, norm, norm, ops.scaled_rows(h, norm)))
    assert torch.equal(got, ops.linear_mx4(x, w))
    lib, d = library.load(), library.DeferredNormArgs()
    d.mode, d.sums, d.n_sums = library.NORM_DEFERRED, torch.zeros(64, device=DEV).data_ptr(), 2
    for rows, cap, n_out, text in ((0, 0.0, 1, "1 to 8"), (9, 0.0, 1, "1 to 8"), (2, -1.0, 2, "soft-cap"), (2, 0.0, 9, "9 output rows"), (2, 0.0, 3, "3 output rows")):
        d.n_out = n_out
        with pytest.raises(library.KernelError, match=text):
            library.check(lib.rdl_mx_few_rows_norm(h.data_ptr(), 0, x.data_ptr(), w.handle, rows, 0, 0.0, cap, d, None, None))
    d.mode = library.NORM_BRANCH
    d.residual = d.w1 = d.w2 = d.branch = d.scaled = h.data_ptr()
    with pytest.raises(library.KernelError, match="units of sums"):
        library.check(lib.rdl_mx_few_rows_norm(None, 0, x.data_ptr(), w.handle, 2, 0, 0.0, 0.0, d, None, None))


def test_a_product_behind_a_deferred_norm_has_all_rows_or_chosen_ones():
    """Without a list of rows the output has as many as the operand; any other number is refused, whether clusters share a tile or not."""
    lib, d = library.load(), library.DeferredNormArgs()
    h = rnd((16, 1024), torch.bfloat16, 69)
    for w in (ops.pack_mx4(rnd((64, 64), torch.float32, 65)), ops.pack_mx4(rnd((512, 1024), torch.float32, 65))):
        d.mode, d.sums, d.n_sums = library.NORM_DEFERRED, torch.zeros(64, device=DEV).data_ptr(), 2
        for rows, n_out in ((2, 1), (8, 7), (8, 1), (5, 4), (1, 2)):
            d.n_out = n_out
            out = torch.full((rows, w.rows), 7.0, device=DEV)
            with pytest.raises(library.KernelError, match=f"{n_out} output rows of {rows}"):
                library.check(lib.rdl_mx_few_rows_norm(out.data_ptr(), 0, h.data_ptr(), w.handle, rows, 0, 0.0, 0.0, d, None, None))
            torch.cuda.synchronize()
            assert (out == 7.0).all()


@pytest.mark.parametrize("act", ["gelu_pytorch_tanh", "silu", "swish_limit"])
@pytest.mark.parametrize("m,n,k,kind", [(1, 1, 32, "bfloat16"), (7, 37, 300, "bfloat16"), (16, 100, 5000, "float32"), (9, 64, 128, "mx8"), (17, 65, 128, "mx8"),
                                        (140, 190, 1003, "mx8"), (64, 33, 40, "mx8")])
def test_gated(m, n, k, kind, act):
    w = ops.pack_mx4(rnd((2 * n, k), torch.float32, 9, 0.1), gated=True)
    x, x64 = rows_for(m, k, kind, 10)
    w64 = f64(ops.expand_mx4(w, torch.float32))
    param = 7.0 if act == "swish_limit" else 0.0
    want = plain.gated(x64 @ w64.T, act, param)
    got = ops.linear_gated_mx4(x, w, act, param)
    # the activations' slopes are at most 1.2 (1.8 with the factor 1.702), so an error of a half moves the result by 2 (|g| + |u| + 1) times it
    t = sum_tolerance(x64, w64, kind)
    g, u = np.split(np.abs(x64 @ w64.T), 2, axis=-1)
    tol = 2 * (g + u + 1) * (t[:, :n] + t[:, n:])
    fast = 2.0 ** -10 * np.maximum(g, 1) * (u + 1)                       # the hardware's tanh and exponential
    exact_kind = kind == "float32"
    check(got, want, tol + (2.0 ** -21 * np.abs(want) if exact_kind else np.abs(want) * 2.0 ** -8 + fast), act)
    rows = ops.linear_gated_mx4(x, w, act, param, out_mx8=True)
    scale = np.repeat(2.0 ** (rows.scales.reshape(m, -1).cpu().numpy().astype(np.float64) - 127), 32, axis=1)[:, :n]
    check(rows.dequantise(), want, tol + fast + np.abs(want) * 2.0 ** -4 * (1 + 2.0 ** -6) + scale * 2.0 ** -10, act + " in 8 bits")
    # the padding of the 8-bit result is zeros: the product behind it reads it
    assert not rows._data.view(torch.uint8)[:m, n:].any() and not rows.scales.reshape(m, -1)[:, -(-n // 32):].any()


@pytest.mark.parametrize("m,kind", [(3, "bfloat16"), (16, "bfloat16"), (16, "mx8"), (40, "mx8"), (300, "mx8")])
def test_the_parts_of_a_row_are_the_row(m, kind):
    """A matrix with a single one in every row hands the rows through: nothing but how they enter shows.  bfloat16 values above 2^-13 of the
    largest of their group are exact, the others off by 2^-21 of it; 8-bit values are exact."""
    k = 200
    x = rnd((m, k), torch.float32, 100) * torch.exp2(torch.randint(-17, 1, (m, k), generator=torch.Generator().manual_seed(101)).float()).to(DEV)
    _enters(x, kind, 2.0 ** -21)


@pytest.mark.parametrize("m", [1, 8, 9, 16])
def test_the_parts_of_a_float32_row_are_the_row(m):
    """As above: float32 values above 2^-13 of the largest of their group are exact to the last bit, the others off by 2^-37 of it."""
    x = rnd((m, 200), torch.float32, 102) * torch.exp2(torch.randint(-30, 1, (m, 200), generator=torch.Generator().manual_seed(103)).float()).to(DEV)
    _enters(x, "float32", 2.0 ** -37)


def _enters(x, kind, below):
    m, k = x.shape
    rows = ops.pack_mx8(x) if kind == "mx8" else x.to(getattr(torch, kind))
    want = f64(rows.dequantise() if kind == "mx8" else rows)
    got = f64(ops.linear_mx4(rows, ops.pack_mx4(torch.eye(k, device=DEV)), out_dtype=torch.float32))
    top = np.repeat(np.abs(plain.groups_of(want)).max(-1), 32, axis=1)[:, :k]
    exact = np.abs(want) >= top * (0.0 if kind == "mx8" else 2.0 ** -13)
    assert np.array_equal(got[exact], want[exact])
    assert (np.abs(got - want) <= below * top).all()


@pytest.mark.parametrize("act,param", [("gelu_pytorch_tanh", 0.0), ("silu", 0.0), ("swish_limit", 3.0)])
@pytest.mark.parametrize("m,kind", [(5, "bfloat16"), (16, "bfloat16"), (16, "mx8"), (40, "mx8"), (300, "mx8")])
def test_the_gate_itself(m, kind, act, param):
    """Matrices with a single one in every row: the gate's and the other half's sums are known exactly, and what is left is the
    activation, in bfloat16 (2^-8) and in 8 bits, where a value takes the code of a value this near.

    With t = -log2(e) times what the sigmoid is taken of: off by 2^-20.5 + 2^-22 |t| of the result, zero where that is below 2^-126; up to
    16 rows whose result is in 8 bits take the library's functions in float32: 2^-22 |g u|."""
    gen = torch.Generator().manual_seed(110)
    g, u = (torch.rand((m, 64), generator=gen) - 0.5) * 19.0, (torch.rand((m, 64), generator=gen) + 0.25) * 2.0
    g = torch.where(g.abs() < 0.01, torch.full_like(g, 0.25), g)
    x = torch.cat([g, u], dim=1).to(DEV)
    x = ops.pack_mx8(x) if kind == "mx8" else x.to(torch.bfloat16)
    y = f64(x.dequantise() if kind == "mx8" else x)
    w = ops.pack_mx4(torch.eye(128, device=DEV), gated=True)
    g, u = np.split(y, 2, axis=-1)
    # 0.5 (1 + tanh z) as 1 / (1 + exp(-2 z)): far below zero the sum with one would lose the result in 64 bits too
    want = g * u / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3))) if act == "gelu_pytorch_tanh" else plain.gated(y, act, param)
    t = {"silu": g, "swish_limit": 1.702 * np.minimum(g, param)}.get(act, 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)) / np.log(2)
    near = np.abs(want) * (2.0 ** -20.5 + 2.0 ** -22 * np.abs(t)) + np.abs(g) * (u + 1) * 2.0 ** -126
    check(ops.linear_gated_mx4(x, w, act, param), want, near + (np.abs(want) + near) * 2.0 ** -8, act)
    if m <= 16:
        near = near + np.abs(g) * (u + 1) * 2.0 ** -22
    rows = ops.linear_gated_mx4(x, w, act, param, out_mx8=True)
    codes = plain.scale_codes(plain.groups_of(want), plain.E4M3[-1])
    assert np.array_equal(rows.scales.reshape(m, -1)[:, :2].cpu().numpy(), codes)
    scale = np.repeat(2.0 ** (codes - 127.0), 32, axis=1)                # a value this near must not move the group's scale
    low, high = (np.sign(v) * plain.E4M3[plain.nearest(np.abs(v) / scale, plain.E4M3)] * scale for v in (want - near, want + near))
    got = f64(rows.dequantise())
    assert (got >= low).all() and (got <= high).all(), act + " in 8 bits"


@pytest.mark.parametrize("m,kind", [(3, "bfloat16"), (12, "float32"), (16, "mx8"), (50, "mx8")])
def test_epilogues(m, kind):
    w = ops.pack_mx4(rnd((90, 256), torch.float32, 11, 0.2))
    x, x64 = rows_for(m, 256, kind, 12)
    w64 = f64(ops.expand_mx4(w, torch.float32))
    y, tol = x64 @ w64.T, sum_tolerance(x64, w64, kind)
    check(ops.linear_mx4(x, w, out_dtype=torch.float32, softcap=5.0), 5.0 * np.tanh(y / 5.0), tol + 2.0 ** -20 * 5, "soft-cap")
    check(ops.linear_mx4(x, w, out_dtype=torch.float32, activation="relu2"), np.maximum(y, 0) ** 2, 2 * np.abs(y) * tol + tol ** 2 + 2.0 ** -22 * y * y, "relu2")
    check(ops.linear_mx4(x, w, out_dtype=torch.float32, activation="silu_plain"), plain.act(y, "silu"), 2 * tol + 2.0 ** -20 * np.abs(y), "silu")


@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_rows_of_any_size(kind):
    """Values near the ends of the float range, and scales that undo them."""
    w = rnd((40, 128), torch.float32, 13)
    dtype = getattr(torch, kind)
    for factor in (2.0 ** 100, 2.0 ** -100, 2.0 ** -126):
        x = (rnd((6, 128), torch.float32, 14) * factor).to(dtype)
        packed = ops.pack_mx4(w / (factor if factor > 1 else max(factor, 2.0 ** -100)))
        w64 = f64(ops.expand_mx4(packed, torch.float32))
        check(ops.linear_mx4(x, packed, out_dtype=torch.float32), f64(x) @ w64.T, sum_tolerance(f64(x), w64, kind) + 2.0 ** -149 * 128, str(factor))


@pytest.mark.parametrize("spread", [2.0 ** 8, 2.0 ** 12, 2.0 ** 16, 2.0 ** 24])
@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_one_large_value_in_every_group(kind, spread):
    """The others of its group stay: exact down to 2^-13 of the largest, off by 2^-21 (float32: 2^-37) of it below that.  The weights of the large
    columns are zero, so that nothing hides what becomes of the small ones."""
    m, n, k = 7, 40, 320
    x = rnd((m, k), torch.float32, 80).to(getattr(torch, kind))
    large = torch.arange(k, device=DEV) % 32 == 5
    x[:, large] = spread * 1.1
    w = rnd((n, k), torch.float32, 81)
    w[:, large] = 0
    w = ops.pack_mx4(w)
    w64, x64 = f64(ops.expand_mx4(w, torch.float32)), f64(x)
    small = np.where(large.cpu().numpy(), 0.0, x64)
    top = spread * 1.1 * 1.01
    lost = np.where(np.abs(small) < top * 2.0 ** -13, top * 2.0 ** (-21 if kind == "bfloat16" else -37), 0.0)
    check(ops.linear_mx4(x, w, out_dtype=torch.float32), small @ w64.T, sum_tolerance(small, w64, kind) + lost @ np.abs(w64).T, kind)


@pytest.mark.parametrize("m,kind", [(4, "bfloat16"), (4, "float32"), (4, "mx8"), (40, "mx8")])
def test_infinities_and_nan(m, kind):
    """What is not finite reaches the outputs of its own row, and only those; a NaN scale of a weight reaches its own column."""
    w = torch.full((20, 96), 0.5, device=DEV)
    packed = ops.pack_mx4(w)
    x = rnd((m, 96), torch.float32, 15)
    x[1, 3] = float("nan")
    x[2, 50] = float("inf")
    x = ops.pack_mx8(x) if kind == "mx8" else x.to(getattr(torch, kind))
    got = f64(ops.linear_mx4(x, packed, out_dtype=torch.float32))
    assert np.isnan(got[1]).all()
    assert np.isnan(got[2]).all() if kind == "mx8" else np.isposinf(got[2]).all()
    assert np.isfinite(got[[0, 3] + list(range(4, m))]).all()
    w[7, 40] = float("nan")
    x = rnd((m, 96), torch.float32, 15)
    x = ops.pack_mx8(x) if kind == "mx8" else x.to(getattr(torch, kind))
    got = f64(ops.linear_mx4(x, ops.pack_mx4(w), out_dtype=torch.float32))
    assert np.isnan(got[:, 7]).all() and np.isfinite(np.delete(got, 7, axis=1)).all()


@pytest.mark.parametrize("m,kind", [(4, "bfloat16"), (4, "float32"), (13, "bfloat16"), (16, "mx8"), (40, "mx8"), (300, "mx8")])
def test_nan_passes_every_epilogue(m, kind):
    """A row with a NaN gives NaN whatever follows its sums; the other rows keep their bits."""
    x = rnd((m, 320), torch.float32, 90)
    x[1, 40] = float("nan")
    clean = x.clone()
    clean[1] = 1.0
    if kind == "mx8":
        x, clean = ops.pack_mx8(x), ops.pack_mx8(clean)
    else:
        x, clean = (t.to(getattr(torch, kind)) for t in (x, clean))
    w, gu = ops.pack_mx4(rnd((200, 320), torch.float32, 91)), ops.pack_mx4(rnd((2 * 100, 320), torch.float32, 92), gated=True)
    calls = {"silu_plain": lambda v: ops.linear_mx4(v, w, activation="silu_plain"), "relu2": lambda v: ops.linear_mx4(v, w, activation="relu2"),
             "soft-cap": lambda v: ops.linear_mx4(v, w, out_dtype=torch.float32, softcap=3.0)}
    for act, param in (("gelu_pytorch_tanh", 0.0), ("silu", 0.0), ("swish_limit", 2.0)):
        calls[act] = lambda v, act=act, param=param: ops.linear_gated_mx4(v, gu, act, param)
        calls[act + " in 8 bits"] = lambda v, act=act, param=param: ops.linear_gated_mx4(v, gu, act, param, out_mx8=True).dequantise()
    others = [i for i in range(m) if i != 1]
    for name, call in calls.items():
        got, want = call(x), call(clean)
        assert got[1].isnan().all(), name
        assert torch.isfinite(want).all() and torch.equal(got[others], want[others]), name


def test_a_row_does_not_depend_on_the_others():
    w = ops.pack_mx4(rnd((300, 1000), torch.float32, 16))
    x, _ = rows_for(16, 1000, "bfloat16", 17)
    whole = ops.linear_mx4(x[:8].contiguous(), w)
    other = x[:8].clone()
    other[1:] = float("nan")
    assert torch.equal(ops.linear_mx4(other, w)[0], whole[0])
    r, _ = rows_for(200, 1000, "mx8", 18)
    first = ops.linear_mx4(r, w)
    assert torch.equal(first, ops.linear_mx4(r, w))                      # the same bits every time
    r._data.view(torch.uint8)[40:200] = 0x7f                            # NaN
    assert torch.equal(ops.linear_mx4(r, w)[:40], first[:40])


def test_another_stream_and_a_graph():
    w = ops.pack_mx4(rnd((256, 512), torch.float32, 19))
    gw = ops.pack_mx4(rnd((512, 512), torch.float32, 20), gated=True)
    x = rnd((40, 512), torch.bfloat16, 21)

    def chain(x):
        rows = ops.norm_mx8(x, second=ops.NormParams(norm, 1e-6, 0.0))
        return ops.linear_mx4(ops.linear_gated_mx4(rows, gw2, "silu", out_mx8=True), w), ops.linear_mx4(x[:9].contiguous(), w)

    norm, gw2 = torch.ones(512, device=DEV), ops.pack_mx4(rnd((1024, 512), torch.float32, 22), gated=True)
    want = [t.clone() for t in chain(x)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = chain(x)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(x)
    x.copy_(rnd((40, 512), torch.bfloat16, 23))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, chain(x)))
    assert gw.gated


def test_clusters_of_several_streams():
    """Products whose tiles are shared by clusters, on streams of their own at the same time: blocks of different ones meet on a multiprocessor, every
    call ends and has the bits it has alone."""
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    calls = []
    for i, (m, n, k, gated) in enumerate([(40, 2304, 2304, False), (128, 700, 1100, False), (17, 2048, 600, True), (64, 300, 9000, False), (5, 1200, 2304, False), (16, 400, 700, False)]):
        w = ops.pack_mx4(rnd((n, k), torch.float32, 120 + i, 0.1), gated=gated)
        x = ops.pack_mx8(rnd((m, k), torch.bfloat16, 130 + i)) if m > 16 else rnd((m, k), torch.bfloat16, 130 + i)
        call = (lambda x=x, w=w: ops.linear_gated_mx4(x, w, "silu", status=status)) if gated else (lambda x=x, w=w: ops.linear_mx4(x, w, status=status))
        calls.append((torch.cuda.Stream(), call, call()))
    torch.cuda.synchronize()
    for _ in range(20):
        results = [[] for _ in calls]
        for _ in range(10):
            for (stream, call, _), out in zip(calls, results):
                with torch.cuda.stream(stream):
                    out.append(call())
        torch.cuda.synchronize()
        assert all(torch.equal(r, want) for (_, _, want), out in zip(calls, results) for r in out)
    assert status.item() == 0


def test_a_product_right_behind_the_packing():
    """The weights are read before the kernel ahead has ended: the packing keeps that safe by itself."""
    x = rnd((8, 2304), torch.bfloat16, 24)
    for seed in range(5):
        w = rnd((4096, 2304), torch.bfloat16, 30 + seed)
        first = ops.linear_mx4(x, ops.pack_mx4(w))
        packed = ops.pack_mx4(w)
        torch.cuda.synchronize()
        assert torch.equal(first, ops.linear_mx4(x, packed))


@pytest.mark.parametrize("m,k,code,name", [(8, 512, 8, "mx_few_rows"), (140, 512, 9, "mx_many_rows"), (40, 4096, 10, "mx_some_rows")])
def test_a_wait_that_runs_out(m, k, code, name):
    lib = library.load()
    w = ops.pack_mx4(rnd((300, k), torch.float32, 25))
    x, x64 = rows_for(m, k, "mx8", 26)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    try:
        lib.rdl_set_wait_test(code, 200_000, 64)
        ops.linear_mx4(x, w, status=status)
        torch.cuda.synchronize()
    finally:
        lib.rdl_set_wait_test(0, 0, 0)
    assert status.item() == code and name in library.FAULTS[code]
    status.zero_()
    w64 = f64(ops.expand_mx4(w, torch.float32))
    check(ops.linear_mx4(x, w, out_dtype=torch.float32, status=status), x64 @ w64.T, sum_tolerance(x64, w64, "mx8"), "the launch after")
    assert status.item() == 0


@pytest.mark.parametrize("m,n,k,code", [(8, 300, 9000, 8), (3, 19001, 1300, 8), (16, 19001, 4700, 8), (40, 300, 4096, 10), (100, 19001, 512, 10), (17, 19001, 300, 10)])
def test_a_long_kernel_ahead_is_no_wait_in_vain(m, n, k, code):
    """A product begins while the kernel ahead of it still runs; however long that takes, none of its waits counts it.  The kernel ahead: one tile of a
    million columns, over 2 ms, twenty times what the waits are given here."""
    lib, status = library.load(), torch.zeros(1, dtype=torch.int32, device=DEV)
    ahead, rows = ops.pack_mx4(torch.ones((256, 1 << 20), device=DEV)), ops.pack_mx8(torch.ones((200, 1 << 20), dtype=torch.bfloat16, device=DEV))
    w = ops.pack_mx4(rnd((n, k), torch.float32, 140, 0.1))
    x = rnd((m, k), torch.bfloat16, 141)
    x = ops.pack_mx8(x) if m > 16 else x
    want = ops.linear_mx4(x, w)
    for _ in range(3):
        try:
            lib.rdl_set_wait_test(code, 200_000, 0)
            first = ops.linear_mx4(rows, ahead, out_dtype=torch.float32)
            got = ops.linear_mx4(x, w, status=status)
            torch.cuda.synchronize()
        finally:
            lib.rdl_set_wait_test(0, 0, 0)
        assert status.item() == 0 and torch.equal(got, want) and (first == float(1 << 20)).all()


def test_tensors_that_start_anywhere():
    """Contiguous rows at an odd place of their memory: the same results as aligned ones."""
    w = rnd((70, 200), torch.float32, 33, 0.05)
    packed = ops.pack_mx4(w)
    norm = ops.NormParams(rnd((201,), torch.float32, 35)[1:], 1e-6, 1.0)
    for dtype in (torch.bfloat16, torch.float32):
        flat = rnd((1 + 6 * 200,), dtype, 34)
        odd = flat[1:].view(6, 200)
        even = odd.clone()
        assert odd.data_ptr() % 8 != 0 and even.data_ptr() % 16 == 0
        assert torch.equal(ops.linear_mx4(odd, packed), ops.linear_mx4(even, packed))
        a, b = ops.norm_mx8(odd, second=norm), ops.norm_mx8(even, second=ops.NormParams(norm.weight.clone(), 1e-6, 1.0))
        assert torch.equal(a.dequantise(), b.dequantise())
        flat = torch.cat([flat[:1], w.to(dtype).reshape(-1)])
        assert torch.equal(ops.expand_mx4(ops.pack_mx4(flat[1:].view(70, 200))), ops.expand_mx4(ops.pack_mx4(w.to(dtype))))


def test_a_weight_beyond_32_bits():
    """2.5e9 bytes of codes: the last rows' outputs come from behind what 32 bits can count."""
    rows, columns = 600_064, 8192
    w = torch.zeros((rows, columns), dtype=torch.bfloat16, device=DEV)
    tail = rnd((64, columns), torch.bfloat16, 36, 0.1)
    w[-64:] = tail
    packed, small = ops.pack_mx4(w), ops.pack_mx4(tail)
    del w
    x = rnd((3, columns), torch.bfloat16, 37)
    got = ops.linear_mx4(x, packed, out_dtype=torch.float32)
    want = f64(x) @ f64(ops.expand_mx4(small, torch.float32)).T
    check(got[:, -64:], want, sum_tolerance(f64(x), f64(ops.expand_mx4(small, torch.float32)), "bfloat16"), "last outputs")
    assert not got[:, :-64].any()
    rows8 = ops.pack_mx8(rnd((20, columns), torch.bfloat16, 38))
    got = ops.linear_mx4(rows8, packed)
    assert torch.equal(got[:, -64:], ops.linear_mx4(rows8, packed)[:, -64:]) and not got[:, :-64].any()
    w64, x64 = f64(ops.expand_mx4(small, torch.float32)), f64(rows8.dequantise())
    want = x64 @ w64.T
    check(got[:, -64:], want, sum_tolerance(x64, w64, "mx8") + np.abs(want) * 2.0 ** -8, "last outputs of 8-bit rows")


# ---- refusals ----

def test_refusals():
    w = ops.pack_mx4(rnd((32, 64), torch.float32, 27))
    g = ops.pack_mx4(rnd((32, 64), torch.float32, 27), gated=True)
    x = rnd((4, 64), torch.bfloat16, 28)
    for call in (lambda: ops.linear_mx4(x, rnd((32, 64), torch.bfloat16, 1)), lambda: ops.linear_mx4(x, g), lambda: ops.linear_gated_mx4(x, w, "silu"),
                 lambda: ops.linear_mx4(x[:, :32], w), lambda: ops.linear_mx4(rnd((4, 128), torch.bfloat16, 1)[:, ::2], w),
                 lambda: ops.linear_mx4(x.to(torch.float16), w), lambda: ops.linear_mx4(x, w, softcap=3.0),
                 lambda: ops.linear_mx4(x, w, activation="tanh"), lambda: ops.linear_gated_mx4(x, g, "relu2"),
                 lambda: ops.linear_mx4(x, w, out_dtype=torch.float32, softcap=-1.0),
                 lambda: ops.linear_mx4(x.cpu(), w), lambda: ops.linear_mx4(x[0], w),
                 lambda: ops.pack_mx4(x.to(torch.float16)), lambda: ops.pack_mx4(x[:3], gated=True), lambda: ops.pack_mx4(x[:, ::2]), lambda: ops.pack_mx4(x[0]),
                 lambda: ops.norm_mx8(x, residual=x), lambda: ops.norm_mx8(x, second=ops.NormParams(x[0, :32], 1e-6, 0.0)), lambda: ops.norm_mx8(x[:, ::2]),
                 lambda: ops.norm_mx8(x, residual_out=torch.empty(3, 64, device=DEV)), lambda: ops.norm_mx8(x.to(torch.float16)),
                 lambda: ops.mx8_rows(x, x), lambda: ops.mx4_weight(torch.zeros(4, 4, dtype=torch.uint8, device=DEV), torch.zeros(4, 2, dtype=torch.uint8, device=DEV), 8),
                 lambda: ops.expand_mx4(w, torch.float16)):
        with pytest.raises(library.KernelError):
            call()
    assert ops.linear_mx4(x[:0], w).shape == (0, 32) and ops.linear_mx4(ops.pack_mx8(x[:0]), w).shape == (0, 32)
    assert ops.linear_gated_mx4(x[:0], g, "silu", out_mx8=True).shape == (0, 16)


def test_rows_in_8_bits_go_with_a_4_bit_weight():
    x, w = ops.pack_mx8(rnd((20, 64), torch.bfloat16, 28)), rnd((32, 64), torch.bfloat16, 29)
    for call in (lambda: ops.linear(x, w), lambda: ops.linear_gated(x, w, "silu"), lambda: ops.linear_branch(x, w, None)):
        with pytest.raises(library.KernelError, match="4-bit weight"):
            call()
