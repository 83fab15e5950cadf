"""A plain 64-bit statement of the block-scaled fp8 operators and the choice of experts, in numpy."""
import numpy as np

F32, F64 = np.float32, np.float64


def _e4m3():
    c = np.arange(128)
    ex, man = c >> 3, c & 7
    mag = np.where(ex == 0, man * 2.0 ** -9, (8 + man) * np.exp2(ex - 10.0))
    mag[127] = np.nan
    return np.concatenate([mag, -mag])


E4M3 = _e4m3()                       # by byte
MID = (E4M3[:126] + E4M3[1:127]) / 2  # between codes i and i + 1


def nearest(v):
    """v (numbers of magnitude at most 448) to e4m3 bytes, ties to the even code."""
    a = np.abs(v)
    lo = np.searchsorted(MID, a, side="left")    # midpoints below a
    tie = (lo < 126) & (a == MID[np.minimum(lo, 125)])
    code = np.where(tie & (lo % 2 == 1), lo + 1, lo)
    return (code | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def _blocks(x, weight):
    M, K = x.shape
    b = 128 if weight else 1
    x = np.pad(x, ((0, -M % b), (0, -K % 128)))
    return x.reshape(x.shape[0] // b, b, x.shape[1] // 128, 128)


def quantize(x, weight=False):
    """x [M, K] -> (bytes uint8 [M, K], scales f32): a block with an infinity or a NaN has a NaN scale, and its
    codes are 0x7f here (a NaN's sign is its own)."""
    x = np.asarray(x, F64)
    M, K = x.shape
    xb = _blocks(x, weight)
    bad = ~np.isfinite(xb).all((1, 3), keepdims=True)
    xb = np.where(bad, 0.0, xb)
    top = np.abs(xb).max((1, 3), keepdims=True) if xb.size else np.zeros((xb.shape[0], 1, xb.shape[2], 1))
    s = np.maximum((top / 448.0).astype(F32), F32(2.0 ** -126))
    inv = (1.0 / s.astype(F64)).astype(F32).astype(F64)
    code = np.where(bad, 0x7f, nearest((xb * inv).astype(F32).astype(F64))).astype(np.uint8)
    s = np.where(bad, F32(np.nan), s)
    return code.reshape(-1, xb.shape[2] * 128)[:M, :K], s[:, 0, :, 0]


def values(code, scale, weight=False):
    M, K = code.shape
    s = scale.astype(F64).repeat(128, 1)
    if weight:
        s = s.repeat(128, 0)
    return E4M3[code] * s[:M, :K]


def product(qa, sa, qw, sw, bias=None):
    """(y, sum of magnitudes) in 64 bits."""
    a, w = values(qa, sa), values(qw, sw, True)
    y, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    if bias is not None:
        y, mag = y + bias.astype(F64), mag + np.abs(bias.astype(F64))
    return y, mag


def bound(y, mag, K, half_step, exact):
    """How far a product may be off.  Products kept whole (binary32 outputs): an instruction adds 32 of them and the
    running sum, six levels of additions of at most one unit (2^-23) of the sum of magnitudes each, K / 32
    instructions; per block of 128 a unit for the scales' product and one for the FMA; one for the bias.  The fp8
    instruction besides drops, of eight products at a time, what lies below 2^-13 of the largest: at most 8 * 2^-13
    of the magnitudes.  And half a step of the output type."""
    units = 6 * (K / 32 + 1) + 2 * (K / 128 + 1) + 1
    return (units * 2.0 ** -23 + (0 if exact else 2.0 ** -10)) * mag + half_step * np.abs(y) + 1e-45


def route(g, k, scoring="softmax", bias=None, groups=1, keep=None, group_top=2, renormalize=True, scale=1.0):
    """(idx, w) of logits g [T, E] in 64 bits, one token after the other."""
    g = np.asarray(g, F64)
    T, E = g.shape
    keep = groups if keep is None else keep
    idx, w = np.zeros((T, k), np.int64), np.zeros((T, k))
    with np.errstate(all="ignore"):
        for t in range(T):
            if scoring == "sigmoid":
                p = 1.0 / (1.0 + np.exp(-g[t]))
            else:
                top = np.nan if np.isnan(g[t]).any() else g[t].max()
                p = np.zeros(E) if top == -np.inf else np.where(g[t] == -np.inf, 0.0 if np.isfinite(top) else np.nan, np.exp(g[t] - top))
                p = p / p.sum() if top != -np.inf else p
            c = p if bias is None else p + np.asarray(bias, F64)
            rank = np.where(np.isnan(c), -np.inf, c)      # (NaN: below -inf, told apart by the second key)
            nan = np.isnan(c)
            best = lambda r, n, at: at[np.lexsort((at, n[at], -r[at]))]  # noqa: E731
            alive = np.arange(E)
            if keep < groups:
                size = E // groups
                sums = np.zeros(groups)
                for q in range(groups):
                    top = best(rank, nan, np.arange(q * size, (q + 1) * size))[:group_top]
                    sums[q] = c[top].sum()
                order = best(np.where(np.isnan(sums), -np.inf, sums), np.isnan(sums), np.arange(groups))[:keep]
                alive = np.concatenate([np.arange(q * size, (q + 1) * size) for q in order])
            at = best(rank, nan, np.sort(alive))[:k]
            idx[t] = at
            total = p[at].sum()
            w[t] = (np.zeros(k) if total == 0 else p[at] / total) * scale if renormalize else p[at] * scale
    return idx, w
