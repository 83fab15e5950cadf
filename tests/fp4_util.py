"""A plain 64-bit statement of the MXFP4 operators and the logits penalties, in numpy."""
import numpy as np

F32, F64 = np.float32, np.float64
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], F64)


def quantize(x):
    """x [M, K] -> (codes uint8 [M, K], scales uint8 [M, K/32])."""
    x = np.asarray(x, F64)
    M, K = x.shape
    xb = x.reshape(M, K // 32, 32)
    bad = ~np.isfinite(xb)
    top = np.where(bad, 0.0, np.abs(xb)).max(-1)
    e = np.frexp(top)[1] - 1                                   # floor(log2 top)
    s = np.where(top > 0, np.clip(e - 2 + 127, 0, 254), 0)
    v = np.ldexp(np.where(bad, 0.0, xb), (127 - s)[..., None])
    a = np.abs(v)
    # halfway points between neighbours; a tie goes to the even code
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    code = np.zeros(a.shape, np.uint8)
    for i, m in enumerate(mid):
        code += (a >= m) if i % 2 else (a > m)
    code |= np.signbit(xb).astype(np.uint8) << 3
    anybad = bad.any(-1)
    code = np.where(anybad[..., None], np.where(bad, 7 | (np.signbit(xb).astype(np.uint8) << 3), 0), code)
    return code.reshape(M, K).astype(np.uint8), np.where(anybad, 255, s).astype(np.uint8)


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def values(codes, scales):
    v = E2M1[codes].reshape(*codes.shape[:-1], -1, 32)
    p = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v * p[..., None]).reshape(codes.shape)


def product(ca, sa, cw, sw, bias=None):
    """(y, sum of magnitudes) in 64 bits."""
    a, w = values(ca, sa), values(cw, sw)
    y, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    if bias is not None:
        y, mag = y + bias.astype(F64), mag + np.abs(bias.astype(F64))
    return y, mag


def bound(y, mag, K, half_step):
    """How far a product may be off: at most one unit of binary32 (2^-23) of the sum of magnitudes for
    each block added to the running sum and one for the bias, and half a step of the output type."""
    return (K // 32 + 1) * 2.0 ** -23 * mag + half_step * np.abs(y) + 1e-45


def counts(tokens, lens, V):
    B, L = tokens.shape
    n = np.zeros((B, V), np.int64)
    for b in range(B):
        for t in tokens[b, :min(max(int(lens[b]), 0), L)]:
            if 0 <= t < V:
                n[b, t] += 1
    return n


def penalize(l, prompt=None, prompt_lens=None, output=None, output_lens=None, repetition=None, frequency=None,
             presence=None, bias=None, mask=None):
    """The declared steps, each rounded to binary32 (numpy's elementwise binary32 operations)."""
    l = np.asarray(l, F32).copy()
    B, V = l.shape
    full = lambda t, ln: np.full(B, t.shape[1]) if ln is None else ln  # noqa: E731
    np_ = counts(prompt, full(prompt, prompt_lens), V) if prompt is not None else np.zeros((B, V), np.int64)
    no = counts(output, full(output, output_lens), V) if output is not None else np.zeros((B, V), np.int64)
    with np.errstate(all="ignore"):
        if bias is not None:
            l = l + bias.astype(F32)
        if repetition is not None:
            r = repetition.astype(F32)[:, None]
            l = np.where(np_ + no > 0, np.where(l > 0, l / r, l * r), l)
        if frequency is not None:
            l = np.where(no > 0, l - frequency.astype(F32)[:, None] * no.astype(F32), l)
        if presence is not None:
            l = np.where(no > 0, l - presence.astype(F32)[:, None], l)
    if mask is not None:
        v = np.arange(V)
        ok = (mask.view(np.uint32)[:, v // 32] >> (v % 32).astype(np.uint32)) & 1
        l = np.where(ok == 1, l, F32(-np.inf))
    assert l.dtype == F32
    return l
