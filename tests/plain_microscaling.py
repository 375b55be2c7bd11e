"""The microscaling formats and the operators on them in float64, from their definitions: groups of 32 columns, a power of two
as scale, e2m1 or e4m3 values found by comparing with every value the format has.  Shares no code with the kernels."""
import numpy as np

GROUP = 32
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])


def nearest(v, grid):
    """Index of the nearest value of the grid to every |v|, ties to the even index."""
    a = np.abs(v)
    hi = np.clip(np.searchsorted(grid, a), 0, len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    down, up = a - grid[lo], grid[hi] - a
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)


def groups_of(v):
    v = np.asarray(v, np.float64)
    out = np.zeros((v.shape[0], -(-v.shape[1] // GROUP) * GROUP))
    out[:, :v.shape[1]] = v
    return out.reshape(v.shape[0], -1, GROUP)


def scale_codes(groups, top):
    """The smallest c >= 0 with amax <= top 2^(c - 127); 255 where the group is not finite."""
    amax = np.abs(groups).max(-1)
    codes = np.zeros(amax.shape, np.int64)
    for i, a in np.ndenumerate(amax):
        if not np.isfinite(a):
            codes[i] = 255
            continue
        c = 0
        while a > top * 2.0 ** (c - 127):
            c += 1
        codes[i] = c
    return codes


def quantise(v, grid):
    """(values [rows, columns] the format keeps of v, scale codes [rows, groups])"""
    g = groups_of(v)
    codes = scale_codes(g, grid[-1])
    scale = np.where(codes == 255, np.nan, 2.0 ** (codes - 127.0))[..., None]
    with np.errstate(invalid="ignore"):
        q = grid[nearest(np.nan_to_num(g / scale), grid)] * np.sign(np.nan_to_num(g)) * scale
    return q.reshape(g.shape[0], -1)[:, :np.shape(v)[1]], codes


def rms_norm(v, weight, eps, offset):
    return v / np.sqrt((v * v).mean(-1, keepdims=True) + eps) * (weight + offset)


def act(g, kind, param=0.0):
    if kind == "silu":
        return g / (1 + np.exp(-g))
    return 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)))


def gated(y, kind, param=0.0):
    g, u = np.split(y, 2, axis=-1)
    if kind == "swish_limit":
        g, u = np.minimum(g, param), np.clip(u, -param, param)
        return g / (1 + np.exp(-1.702 * g)) * (u + 1)
    return act(g, kind) * u
