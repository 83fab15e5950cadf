"""The MXFP4 quantiser and products (moe_mxfp4.quantize_mxfp4 / mm_mxfp4 / linear_mxfp4,
moe_ref.grouped_linear_mxfp4) against a plain 64-bit statement (fp4_util).

Codes and scales are compared bit for bit.  Products whose exact value and every partial sum are
binary32 numbers (scales of one row within two octaves: all terms are multiples of one power of two
and the sum of their magnitudes stays below 2^24 of it) are compared bit for bit; the others within
one binary32 unit of the sum of magnitudes a block, and half a step of the output type."""
import numpy as np
import pytest
import torch

import fp4_util as U
from gpu_util import bits, dev, say, to_dev

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import lockstep_amd._lib as L
    L.load()


def _values(g, M, K):
    x = g.standard_normal((M, K)) * np.exp2(g.integers(-20, 20, (M, K // 32))).repeat(32, 1)
    x[g.random((M, K)) < 0.02] = 0
    return x.astype(np.float32)


# ---------------------------------------------------------------- the quantiser
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", [(1, 32), (3, 96), (37, 2880), (257, 64), (2, 18944)])
def test_quantize(M, K, dtype):
    from lockstep_amd import moe_mxfp4 as X
    say("quantize", M, K, dtype)
    x = torch.from_numpy(_values(np.random.default_rng(M + K), M, K)).to(dtype)
    packed, scale = X.quantize_mxfp4(x.to(dev()))
    c, s = U.quantize(x.double().numpy())
    assert np.array_equal(bits(scale), s) and np.array_equal(bits(packed), U.pack(c))
    # (blocks whose float16 values overflowed to infinity hold no finite value to read back)
    back = X.dequant_mxfp4(packed, scale, torch.float32).double().cpu().numpy()
    finite = (s != 255).repeat(32, 1)
    assert np.array_equal(back[finite], U.values(c, s)[finite]) and not np.isfinite(back[~finite]).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_every_border(dtype):
    """Every halfway point and its neighbours in the input type, of both signs, under every largest
    value's exponent the type has; zeros of both signs, all-zero blocks, the smallest and largest
    numbers."""
    from lockstep_amd import moe_mxfp4 as X
    fi = torch.finfo(dtype)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 6.0, 7.0], dtype=torch.float64)
    lo, hi = int(np.log2(fi.tiny)) - 12, int(np.log2(fi.max))
    rows = []
    for e in range(lo, hi - 2):
        base = (mids * 2.0 ** e).to(dtype)
        up, down = torch.nextafter(base, torch.full_like(base, float("inf"))), torch.nextafter(base, torch.zeros_like(base))
        b = torch.cat([base, up, down, torch.tensor([0.0, -0.0], dtype=dtype)])
        assert b.numel() == 32
        rows += [b, -b]
    rows += [torch.zeros(32, dtype=dtype), -torch.zeros(32, dtype=dtype), torch.full((32,), fi.max, dtype=dtype)]
    smallest = torch.zeros(32, dtype=dtype)
    smallest[5] = torch.nextafter(torch.tensor(0.0, dtype=dtype), torch.tensor(1.0, dtype=dtype))
    rows.append(smallest)
    x = torch.stack(rows)
    packed, scale = X.quantize_mxfp4(x.to(dev()))
    c, s = U.quantize(x.double().numpy())
    assert np.array_equal(bits(scale), s) and np.array_equal(bits(packed), U.pack(c))


def test_quantize_infinities_and_nans():
    from lockstep_amd import moe_mxfp4 as X
    x = np.random.default_rng(5).standard_normal((4, 96)).astype(np.float32)
    x[0, 3], x[1, 40], x[2, 95], x[3, 64] = np.inf, -np.inf, np.nan, -np.nan
    packed, scale = X.quantize_mxfp4(to_dev(x))
    c, s = U.quantize(x)
    assert (s == 255).sum() == 4
    assert np.array_equal(bits(scale), s)
    assert np.array_equal(bits(packed) & 0x77, U.pack(c) & 0x77)        # (a NaN's sign is its own)


def test_quantize_strides_shapes_and_empty():
    from lockstep_amd import moe_mxfp4 as X
    g = np.random.default_rng(6)
    big = torch.from_numpy(_values(g, 40, 160)).to(dev())
    for view in (big[:, 32:128], big[:, 1:97], big[::3, :64], big[3:4, 5:37], big.t()[:96].t(), big[:32, :96].t()[:, :32]):
        c, s = U.quantize(view.double().cpu().numpy())
        packed, scale = X.quantize_mxfp4(view)
        assert np.array_equal(bits(packed), U.pack(c)) and np.array_equal(bits(scale), s)
    half = big.to(torch.bfloat16)[:, 3:99]
    c, s = U.quantize(half.double().cpu().numpy())
    assert np.array_equal(bits(X.quantize_mxfp4(half)[0]), U.pack(c))
    p, s = X.quantize_mxfp4(big.reshape(4, 10, 160))
    assert p.shape == (4, 10, 80) and s.shape == (4, 10, 5)
    assert [t.shape for t in X.quantize_mxfp4(big[:0])] == [(0, 80), (0, 5)]
    assert [t.shape for t in X.quantize_mxfp4(big[:, :0])] == [(40, 0), (40, 0)]
    p64, _ = X.quantize_mxfp4(big[:2].double())
    assert torch.equal(p64, X.quantize_mxfp4(big[:2])[0])
    for bad in (big[:, :33], big.to(torch.int32)):
        with pytest.raises((ValueError, TypeError)):
            X.quantize_mxfp4(bad)


# ---------------------------------------------------------------- the product
def _operand(g, rows, K, octaves):
    codes = g.integers(0, 16, (rows, K), dtype=np.uint8)
    scales = (127 + g.integers(-octaves, octaves + 1, (rows, K // 32))).astype(np.uint8)
    return codes, scales


def _mm(ca, sa, cw, sw, bias=None, out_dtype=torch.float32):
    from lockstep_amd import moe_mxfp4 as X
    return X.mm_mxfp4(to_dev(U.pack(ca)), to_dev(sa), to_dev(U.pack(cw)), to_dev(sw),
                      None if bias is None else to_dev(bias), out_dtype)


SIZES = [(1, 1, 32), (1, 17, 64), (2, 48, 96), (5, 33, 128), (16, 16, 160), (17, 100, 224), (31, 64, 512), (33, 257, 288),
         (64, 130, 1024), (65, 129, 352), (100, 300, 640), (129, 255, 256), (200, 520, 480), (257, 260, 544),
         (300, 1030, 128), (513, 512, 96), (600, 900, 32), (65, 5500, 64), (1100, 480, 96), (129, 3301, 160), (600, 901, 224),
         (600, 900, 288), (257, 1830, 352), (600, 907, 480), (1030, 515, 544), (2000, 280, 1056)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_exact(M, N, K):
    """Scales one octave up or down: every term is a multiple of 2^-4, and 36 * 2^2 * K < 2^24 * 2^-4
    for K <= 7281, so the sum is a binary32 number however it is ordered."""
    say("product exact", M, N, K)
    g = np.random.default_rng(M * N + K)
    ca, sa = _operand(g, M, K, 1)
    cw, sw = _operand(g, N, K, 1)
    y, _ = U.product(ca, sa, cw, sw)
    got = _mm(ca, sa, cw, sw)
    assert np.array_equal(got.double().cpu().numpy(), y)
    bias = g.standard_normal(N).astype(np.float32)
    want = torch.from_numpy(y.astype(np.float32) + bias)            # one binary32 addition
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        assert np.array_equal(bits(_mm(ca, sa, cw, sw, bias, dt)), bits(want.to(dt))), dt


@pytest.mark.parametrize("M,N,K", [(3, 8213, 96), (7, 25003, 64), (40, 4200, 160), (33, 13001, 96), (64, 6500, 1088),
                                   (700, 4500, 96), (2050, 3500, 160), (3700, 3400, 288), (3600, 3600, 64),
                                   (720, 8250, 96), (1760, 5800, 1472), (24, 20000, 96), (3000, 40, 1056), (9000, 16, 96)])
def test_product_exact_over_many_columns(M, N, K):
    """The same where there are enough blocks for the larger ones: of 32 and 64 columns for few rows, and
    tiles of every size."""
    say("product many columns", M, N, K)
    g = np.random.default_rng(M + N + K)
    ca, sa = _operand(g, M, K, 1)
    cw, sw = _operand(g, N, K, 1)
    y, _ = U.product(ca, sa, cw, sw)
    assert np.array_equal(_mm(ca, sa, cw, sw).double().cpu().numpy(), y)
    bias = g.standard_normal(N).astype(np.float32)
    want = torch.from_numpy(y.astype(np.float32) + bias)
    assert np.array_equal(bits(_mm(ca, sa, cw, sw, bias, torch.bfloat16)), bits(want.to(torch.bfloat16)))


@pytest.mark.parametrize("M,N,K", [(3, 50, 24576), (4, 50, 24608), (2, 40, 32768), (20, 70, 32768), (3, 40, 32800),
                                   (33, 100, 65600), (70, 30, 24608)])
def test_long_rows(M, N, K):
    """Around the lengths of K where few rows stop being quantised in the product's launch, and where they
    go to the tiles."""
    from lockstep_amd import moe_mxfp4 as X
    say("long rows", M, N, K)
    g = np.random.default_rng(M + N + K)
    x = torch.from_numpy(g.standard_normal((M, K)).astype(np.float32)).to(torch.bfloat16)
    cw, sw = _operand(g, N, K, 4)
    ca, sa = U.quantize(x.double().numpy())
    y, mag = U.product(ca, sa, cw, sw)
    w, ws = to_dev(U.pack(cw)), to_dev(sw)
    got = X.linear_mxfp4(x.to(dev()), w, ws, out_dtype=torch.float32)
    assert (np.abs(got.double().cpu().numpy() - y) <= U.bound(y, mag, K, 2.0 ** -24)).all()
    assert np.array_equal(bits(got), bits(_mm(ca, sa, cw, sw)))
    assert np.array_equal(bits(got[:1]), bits(X.linear_mxfp4(x[:1].to(dev()), w, ws, out_dtype=torch.float32)))


@pytest.mark.parametrize("M,N,K,out", [(1, 200, 3584, torch.bfloat16), (24, 129, 14336, torch.float32),
                                       (7, 64, 18944, torch.float16), (150, 300, 2880, torch.float32),
                                       (300, 513, 2048, torch.bfloat16), (64, 2000, 1056, torch.float32)])
def test_product_wide_scales(M, N, K, out):
    say("product wide", M, N, K, out)
    g = np.random.default_rng(M + N + K)
    ca, sa = _operand(g, M, K, 5)
    cw, sw = _operand(g, N, K, 5)
    sa = (sa.astype(int) - 3).astype(np.uint8)
    bias = g.standard_normal(N).astype(np.float32)
    y, mag = U.product(ca, sa, cw, sw, bias)
    got = _mm(ca, sa, cw, sw, bias, out).double().cpu().numpy()
    assert (np.abs(got - y) <= U.bound(y, mag, K, HALF[out])).all()


@pytest.mark.parametrize("M,N,K", [(24, 8400, 15200), (40, 4400, 15200), (16, 6000, 18944), (3, 9000, 5440)])
def test_long_rows_over_many_columns(M, N, K):
    """Long K over blocks of every number of columns: a column's bits are those of a product of its own."""
    g = np.random.default_rng(M + N + K)
    ca, sa = _operand(g, M, K, 5)
    w = torch.from_numpy(g.integers(0, 256, (N, K // 2), dtype=np.uint8)).to(dev())
    ws = torch.from_numpy(g.integers(120, 130, (N, K // 32), dtype=np.uint8)).to(dev())
    from lockstep_amd import moe_mxfp4 as X
    a, s = to_dev(U.pack(ca)), to_dev(sa)
    full = bits(X.mm_mxfp4(a, s, w, ws))
    for lo in (0, 1000, N - 33):
        cols = slice(lo, lo + 33)
        p = bits(w[cols])
        y, mag = U.product(ca, sa, np.stack((p & 15, p >> 4), -1).reshape(33, K), bits(ws[cols]))
        one = X.mm_mxfp4(a, s, w[cols], ws[cols])
        assert np.array_equal(bits(one), full[:, cols])
        assert (np.abs(one.double().cpu().numpy() - y) <= U.bound(y, mag, K, 2.0 ** -24)).all()


def test_product_rows_do_not_depend_on_the_batch():
    """The bits of a row are the same alone, in every batch and at every place in it."""
    g = np.random.default_rng(11)
    for N, K in ((200, 1088), (1040, 2880)):
        ca, sa = _operand(g, 600, K, 6)
        cw, sw = _operand(g, N, K, 6)
        full = bits(_mm(ca, sa, cw, sw))
        for lo, hi in ((0, 1), (3, 5), (7, 16), (100, 117), (30, 63), (5, 100), (590, 600), (10, 140), (0, 260), (99, 599)):
            assert np.array_equal(bits(_mm(ca[lo:hi], sa[lo:hi], cw, sw)), full[lo:hi]), (N, K, lo, hi)


def test_product_rows_do_not_depend_on_a_large_batch():
    """The same up to 256 x 256 tiles, and over every number of columns a block takes."""
    g = np.random.default_rng(13)
    M, N, K = 3600, 3600, 544
    ca, sa = _operand(g, M, K, 6)
    cw, sw = _operand(g, N, K, 6)
    full = bits(_mm(ca, sa, cw, sw))
    for lo, hi in ((0, 1), (17, 19), (300, 340), (3500, 3600), (1000, 1700), (900, 3000)):
        assert np.array_equal(bits(_mm(ca[lo:hi], sa[lo:hi], cw, sw)), full[lo:hi]), (lo, hi)
        assert np.array_equal(bits(_mm(ca[lo:hi], sa[lo:hi], cw[77:190], sw[77:190])), full[lo:hi, 77:190]), (lo, hi)


@pytest.mark.parametrize("M,N,K", [(3700, 3400, 224), (2050, 515, 128), (700, 4500, 1088), (300, 1030, 2880), (129, 255, 64)])
def test_product_rows_do_not_depend_on_the_batch_at_any_scale(M, N, K):
    """The same with scale bytes spread over up to 121 octaves in either operand, over all that a byte holds,
    and where products turn subnormal or overflow: few rows on one shape of the matrix instruction and many
    on the other sum alike."""
    g = np.random.default_rng(M + N + K)
    ca, cw = g.integers(0, 16, (M, K), dtype=np.uint8), g.integers(0, 16, (N, K), dtype=np.uint8)
    for lo, hi in ((107, 147), (67, 187), (40, 70), (180, 195), (0, 254)):
        say("scales", lo, hi)
        sa = g.integers(lo, hi + 1, (M, K // 32), dtype=np.uint8)
        sw = g.integers(lo, hi + 1, (N, K // 32), dtype=np.uint8)
        full = bits(_mm(ca, sa, cw, sw))
        for r0, r1 in ((0, 1), (5, 14), (60, 90), (0, min(M, 257)), (100, M)):
            assert np.array_equal(bits(_mm(ca[r0:r1], sa[r0:r1], cw, sw)), full[r0:r1]), (lo, hi, r0, r1)


def test_product_special_scales():
    """255 is a NaN for its row or column alone, also under zero codes; the largest scales overflow to
    infinity, the smallest reach zero or a subnormal; no neighbour changes."""
    for M, K, N in ((5, 96, 70), (40, 288, 70), (200, 160, 70), (600, 160, 900), (3600, 96, 3600)):
        g = np.random.default_rng(M)
        ca, sa = _operand(g, M, K, 1)
        cw, sw = _operand(g, N, K, 1)
        sa[2, 1], sw[33, 0] = 255, 255
        ca[2], cw[33, :32] = 0, 0
        y, _ = U.product(ca, sa, cw, sw)
        got = _mm(ca, sa, cw, sw).double().cpu().numpy()
        assert np.isnan(got[2]).all() and np.isnan(got[:, 33]).all()
        assert np.array_equal(got, y, equal_nan=True)
        ca[:], cw[:] = 2, 2
        sa[:], sw[:] = 254, 254
        assert np.isposinf(_mm(ca, sa, cw, sw).cpu().numpy()).all()
        sa[:], sw[:] = 0, 0
        assert (_mm(ca, sa, cw, sw).cpu().numpy() == 0).all()
        sw[:] = 110                                   # K products of 2^-144: subnormal and exact
        assert (_mm(ca, sa, cw, sw).double().cpu().numpy() == K * 2.0 ** -144).all()


def test_product_empty_and_layouts():
    from lockstep_amd import moe_mxfp4 as X
    g = np.random.default_rng(12)
    ca, sa = _operand(g, 20, 96, 1)
    cw, sw = _operand(g, 30, 96, 1)
    y, _ = U.product(ca, sa, cw, sw)
    a, s, w, t = (to_dev(v) for v in (U.pack(ca), sa, U.pack(cw), sw))
    bias = to_dev(g.standard_normal(30).astype(np.float32))
    assert X.mm_mxfp4(a[:0], s[:0], w, t).shape == (0, 30) and X.mm_mxfp4(a, s, w[:0], t[:0]).shape == (20, 0)
    none = X.mm_mxfp4(a[:, :0], s[:, :0], w[:, :0], t[:, :0], bias)          # K = 0: the bias alone
    assert torch.equal(none, bias.expand(20, 30))
    wide = torch.zeros((20, 100), dtype=torch.uint8, device=dev())
    wide[:, 7:55] = a                                                        # a misaligned, strided view
    assert np.array_equal(X.mm_mxfp4(wide[:, 7:55], s, w, t).double().cpu().numpy(), y)
    assert np.array_equal(X.mm_mxfp4(a[::2], s[::2], w, t).double().cpu().numpy(), y[::2])
    x = torch.randn((2, 3, 96), device=dev(), dtype=torch.bfloat16)
    assert X.linear_mxfp4(x, w, t, bias).shape == (2, 3, 30) and X.linear_mxfp4(x[:0], w, t).shape == (0, 3, 30)
    for bad in (lambda: X.mm_mxfp4(a, s, w[:, :32], t[:, :2]), lambda: X.mm_mxfp4(a, s[:, :2], w, t),
                lambda: X.mm_mxfp4(a.to(torch.int32), s, w, t), lambda: X.mm_mxfp4(a, s, w, t, bias[:29]),
                lambda: X.mm_mxfp4(a, s, w, t, out_dtype=torch.int32), lambda: X.linear_mxfp4(x[..., :64], w, t),
                lambda: X.linear_mxfp4(x.to(torch.int32), w, t)):
        with pytest.raises((ValueError, TypeError)):
            bad()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1, 100, 3584), (2, 130, 96), (4, 64, 2880), (3, 9001, 160), (1, 25001, 64), (16, 333, 1024), (15, 90, 32),
                                   (13, 20000, 96), (16, 9000, 160), (17, 100, 96), (9, 77, 448), (40, 300, 1024),
                                   (130, 260, 288), (300, 300, 512), (600, 900, 288), (601, 900, 512), (65, 5500, 96)])
def test_linear_is_the_product_of_the_quantised_rows(M, N, K, dtype):
    from lockstep_amd import moe_mxfp4 as X
    say("linear", M, N, K, dtype)
    g = torch.Generator().manual_seed(M + N + K)
    x = torch.randn((M, K + 3), generator=g).to(dtype).to(dev())
    w, ws = X.quantize_mxfp4(torch.randn((N, K), generator=g).to(dev()))
    bias = torch.randn((N,), generator=g).to(dev())
    for v in (x[:, :K].contiguous(), x[:, 3:]):
        a, s = X.quantize_mxfp4(v)
        assert np.array_equal(bits(X.linear_mxfp4(v, w, ws, bias)), bits(X.mm_mxfp4(a, s, w, ws, bias, dtype)))
        assert np.array_equal(bits(X.linear_mxfp4(v, w, ws, out_dtype=torch.float32)), bits(X.mm_mxfp4(a, s, w, ws)))
    bad = x[:, :K].contiguous()
    bad[0, 5] = float("inf")
    y = X.linear_mxfp4(bad, w, ws)
    assert y[0].isnan().all() and not y[1:].isnan().any()


# ---------------------------------------------------------------- by expert
def _experts(g, E, H, I, bias):
    ex, host = [], []
    for _ in range(E):
        c13, s13 = _operand(g, 2 * I, H, 1)
        c2, s2 = _operand(g, H, I, 1)
        b13 = g.standard_normal(2 * I).astype(np.float32) if bias else None
        b2 = g.standard_normal(H).astype(np.float32) if bias else None
        host.append({"w13": (c13, s13, b13), "w2": (c2, s2, b2)})
        ex.append(((to_dev(U.pack(c13)), to_dev(s13)), (to_dev(U.pack(c2)), to_dev(s2)),
                   None if b13 is None else to_dev(b13), None if b2 is None else to_dev(b2)))
    from lockstep_amd import moe_ref as MR
    return MR.ExpertTablesMX(ex, packed=True), host


def _check_grouped(tables, host, which, R, offs, g, dt):
    from lockstep_amd import moe_ref as MR
    K = tables.H if which == "w13" else tables.I
    ca, sa = _operand(g, R, K, 1)
    out = MR.grouped_linear_mxfp4(tables, which, to_dev(U.pack(ca)), to_dev(sa), to_dev(np.asarray(offs, np.int32)), dt)
    co = np.minimum(np.maximum.accumulate(np.maximum(offs, 0)), R)
    got = bits(out)
    for e, h in enumerate(host):
        r0, r1 = co[e], co[e + 1]
        if r1 > r0:
            cw, sw, b = h[which]
            y, _ = U.product(ca[r0:r1], sa[r0:r1], cw, sw)
            y = y.astype(np.float32) if b is None else y.astype(np.float32) + b
            assert np.array_equal(got[r0:r1], bits(torch.from_numpy(y).to(dt))), (which, e)


@pytest.mark.parametrize("R,E,H,I,bias,dt", [(1, 3, 64, 32, True, torch.bfloat16), (4, 32, 160, 96, True, torch.bfloat16),
                                             (50, 6, 288, 64, False, torch.float32), (256, 32, 96, 160, True, torch.bfloat16),
                                             (700, 5, 128, 256, False, torch.float16), (1500, 70, 64, 96, True, torch.bfloat16),
                                             (900, 2, 320, 544, True, torch.float32), (4000, 20, 96, 640, True, torch.bfloat16),
                                             (800, 40, 96, 640, False, torch.bfloat16), (400, 130, 64, 1024, True, torch.float32),
                                             (9000, 130, 32, 256, True, torch.float16), (96, 4, 96, 2272, True, torch.bfloat16),
                                             (512, 6, 96, 4448, False, torch.float32), (64, 32, 64, 1024, True, torch.bfloat16), (720, 8, 96, 4384, True, torch.bfloat16),
                                             (720, 8, 1696, 3680, True, torch.bfloat16)])
def test_grouped(R, E, H, I, bias, dt):
    say("grouped", R, E, H, I, bias, dt)
    g = np.random.default_rng(R + E)
    tables, host = _experts(g, E, H, I, bias)
    p = 1.0 / np.arange(1, E + 1) ** 1.1
    p[g.integers(0, E, max(1, E // 4))] = 0                        # experts without a row
    p = np.full(E, 1.0) if p.sum() == 0 else p
    offs = np.concatenate([[0], np.cumsum(g.multinomial(R, p / p.sum()))])
    for which in ("w13", "w2"):
        _check_grouped(tables, host, which, R, offs, g, dt)


@pytest.mark.parametrize("I", [64, 992])
def test_grouped_bad_offsets(I):
    g = np.random.default_rng(21)
    tables, host = _experts(g, 6, 96, I, False)
    for offs in ([0, 100, 80, 300, 700, 650, 900], [-5, -2, 10, 10, 9, 400, 499], [500] * 7, [0] * 7, [7, 7, 8, 500, 500, 501, 2]):
        _check_grouped(tables, host, "w13", 500, offs, g, torch.float32)


def test_grouped_some_biases_and_refused_experts():
    from lockstep_amd import moe_ref as MR
    g = np.random.default_rng(25)
    ex, host = [], []
    for e in range(3):
        c13, s13 = _operand(g, 64, 96, 1)
        c2, s2 = _operand(g, 96, 32, 1)
        b = g.standard_normal(64).astype(np.float32) if e == 1 else None
        host.append({"w13": (c13, s13, b)})
        ex.append(((to_dev(U.pack(c13)), to_dev(s13)), (to_dev(U.pack(c2)), to_dev(s2)), None if b is None else to_dev(b), None))
    tables = MR.ExpertTablesMX(ex, packed=True)
    for R, offs in ((30, [0, 4, 20, 30]), (100, [0, 1, 60, 100])):
        _check_grouped(tables, host, "w13", R, offs, g, torch.float32)
    a, s, o = to_dev(np.zeros((2, 48), np.uint8)), to_dev(np.zeros((2, 3), np.uint8)), torch.zeros(4, dtype=torch.int32, device=dev())
    moved = torch.zeros((64 * 48 + 1,), dtype=torch.uint8, device=dev())[1:].view(64, 48)
    other = (to_dev(np.zeros((32, 48), np.uint8)), to_dev(np.zeros((32, 3), np.uint8)))
    for bad in ((moved, ex[2][0][1]), other):
        with pytest.raises(ValueError):
            MR.grouped_linear_mxfp4(MR.ExpertTablesMX(ex[:2] + [(bad,) + ex[2][1:]], packed=True), "w13", a, s, o)
    for args in ((tables, "w3", a, s, o), (tables, "w13", a, s, o[:3]), (tables, "w13", a, s, o.long()),
                 (tables, "w2", a, s, o), (tables, "w13", a, s[:, :2], o)):
        with pytest.raises(ValueError):
            MR.grouped_linear_mxfp4(*args)


@pytest.mark.parametrize("I", [64, 1024])
def test_grouped_leaves_other_rows_alone(I):
    """Rows of no expert keep what the buffer held."""
    from lockstep_amd import _lib as L
    g = np.random.default_rng(22)
    tables, host = _experts(g, 3, 64, I, False)
    N = 2 * I
    for R, offs in ((40, [3, 10, 10, 30]), (600, [5, 200, 300, 580])):
        ca, sa = _operand(g, R, 64, 1)
        a, s, o = to_dev(U.pack(ca)), to_dev(sa), to_dev(np.asarray(offs, np.int32))
        out = torch.full((R, N), 7.0, device=dev())
        need = L.load().lsk_grouped_gemm_mxfp4_workspace(R, 3, N, 64)
        work = torch.empty((max(need, 1),), dtype=torch.uint8, device=dev())
        L.call("lsk_grouped_gemm_mxfp4", L.ptr(a), L.ptr(s), L.ptr(o), 3, R, L.ptr(tables.w13), tables.ldw13,
               L.ptr(tables.ws13), tables.lds13, None, N, 64, L.ptr(out), L.LSK_F32, N, L.ptr(work), need,
               L.stream_of(a))
        assert (out[:offs[0]] == 7).all() and (out[offs[3]:] == 7).all()
        y, _ = U.product(ca[offs[0]:offs[1]], sa[offs[0]:offs[1]], *host[0]["w13"][:2])
        assert np.array_equal(out[offs[0]:offs[1]].double().cpu().numpy(), y)


@pytest.mark.parametrize("I", [96, 736])
def test_grouped_rows_are_the_dense_products(I):
    from lockstep_amd import moe_mxfp4 as X, moe_ref as MR
    g = np.random.default_rng(23)
    E, H, R = 4, 2880, 777
    tables, host = _experts(g, E, H, I, True)
    ca, sa = _operand(g, R, H, 7)
    offs = [0, 1, 40, 41, 777]
    a, s = to_dev(U.pack(ca)), to_dev(sa)
    out = MR.grouped_linear_mxfp4(tables, "w13", a, s, to_dev(np.asarray(offs, np.int32)))
    for e in range(E):
        cw, sw, b = host[e]["w13"]
        r = slice(offs[e], offs[e + 1])
        one = X.mm_mxfp4(a[r], s[r], to_dev(U.pack(cw)), to_dev(sw), to_dev(b), torch.bfloat16)
        assert np.array_equal(bits(out[r]), bits(one)), e


# ---------------------------------------------------------------- together, streams, graphs
def test_moe_block_of_mxfp4_rows():
    """Router -> rows sorted by expert -> gate/up -> activation -> down -> weighted sum, every product
    in MXFP4, against the same steps in 64 bits on the kernels' own quantised rows."""
    from lockstep_amd import contract_common as CC, moe_mxfp4 as X, moe_ref as MR
    g = np.random.default_rng(31)
    T, E, k, H, I = 45, 8, 2, 96, 64
    tables, host = _experts(g, E, H, I, True)
    x = torch.from_numpy(g.standard_normal((T, H)).astype(np.float32) * 0.05).to(torch.bfloat16).to(dev())
    idx, wt, _ = MR.router_from_logits(torch.from_numpy(g.standard_normal((T, E)).astype(np.float32)).to(dev()), k, True,
                                       CC.table_on(dev()))
    order = idx.reshape(-1).argsort(stable=True)
    offs = torch.searchsorted(idx.reshape(-1)[order].contiguous(), torch.arange(E + 1, device=dev())).to(torch.int32)
    a, s = X.quantize_mxfp4(x[order // k])
    y13 = MR.grouped_linear_mxfp4(tables, "w13", a, s, offs)
    h = MR.act_silu(y13[:, :I].float(), y13[:, I:].float())
    a2, s2 = X.quantize_mxfp4(h)
    y2 = MR.grouped_linear_mxfp4(tables, "w2", a2, s2, offs, torch.float32)
    y = torch.zeros((T, H), device=dev()).index_add_(0, order // k, y2 * wt.reshape(-1)[order].float()[:, None])
    o, od = offs.cpu().numpy(), order.cpu().numpy()
    unpack = lambda p: np.stack((p & 15, p >> 4), -1).reshape(p.shape[0], -1)  # noqa: E731
    ca2, sa2 = U.quantize(h.double().cpu().numpy())
    assert np.array_equal(bits(a2), U.pack(ca2)) and np.array_equal(bits(s2), sa2)
    ref, mag = np.zeros((T, H)), np.zeros((T, H))
    for e in range(E):
        r = slice(o[e], o[e + 1])
        cw, sw, b = host[e]["w13"]
        v, m = U.product(unpack(bits(a)[r]), bits(s)[r], cw, sw, b)
        assert (np.abs(y13[r].double().cpu().numpy() - v) <= U.bound(v, m, H, 2.0 ** -8)).all()
        cw, sw, b = host[e]["w2"]
        v, m = U.product(ca2[r], sa2[r], cw, sw, b)
        f = wt.reshape(-1).double().cpu().numpy()[od[r]][:, None]
        for i, t in enumerate(od[r] // k):
            ref[t] += f[i] * v[i]
            mag[t] += f[i] * m[i]
    # the products' bound, and one unit for each of the weighting, and the additions of k terms
    assert (np.abs(y.double().cpu().numpy() - ref) <= (I // 32 + 2 + k) * 2.0 ** -23 * mag + 1e-30).all()


def test_head_and_penalties():
    """The MXFP4 head variant, and its logits through the penalties."""
    from lockstep_amd import moe_mxfp4 as X, t16h_lmvariants as TH
    g = np.random.default_rng(32)
    W = torch.from_numpy(g.standard_normal((1001, 224)).astype(np.float32)).to(torch.bfloat16).to(dev())
    head = TH.build("mxfp4").prepare(W)
    assert head.n_out() == 1001 and head.nbytes() == 1001 * (112 + 7)
    x = torch.from_numpy(g.standard_normal((6, 224)).astype(np.float32)).to(dev())
    l = head.logits(x)
    w, ws = X.quantize_mxfp4(W)
    assert l.dtype == torch.float32 and torch.equal(l, X.linear_mxfp4(x, w, ws))
    cw, sw = U.quantize(W.double().cpu().numpy())
    ca, sa = U.quantize(x.double().cpu().numpy())
    y, mag = U.product(ca, sa, cw, sw)
    assert (np.abs(l.double().cpu().numpy() - y) <= U.bound(y, mag, 224, 2.0 ** -24)).all()
    out = g.integers(0, 1001, (6, 30))
    rep, pres = np.full(6, 1.3, np.float32), np.full(6, 0.5, np.float32)
    got = TH.penalize_logits(l, output=to_dev(out), repetition=to_dev(rep), presence=to_dev(pres))
    want = U.penalize(l.cpu().numpy(), output=out, repetition=rep, presence=pres)
    assert np.array_equal(bits(got), bits(torch.from_numpy(want)))


def test_other_streams():
    from lockstep_amd import moe_mxfp4 as X
    g = torch.Generator().manual_seed(1)
    w, ws = X.quantize_mxfp4(torch.randn((520, 1024), generator=g).to(dev()))
    xs = [torch.randn((m, 1024), generator=g).to(dev()) for m in (1, 20, 300, 1100)]
    want = [X.linear_mxfp4(x, w, ws) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append(X.linear_mxfp4(x, w, ws))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("M", [1, 12, 40, 300, 1700])
def test_captured_and_replayed(M):
    from lockstep_amd import moe_mxfp4 as X, moe_ref as MR, t16h_lmvariants as TH
    g = np.random.default_rng(41)
    E, H, I = 5, 288, 704
    tables, _ = _experts(g, E, H, I, True)
    w, ws = X.quantize_mxfp4(torch.from_numpy(g.standard_normal((330, H)).astype(np.float32)).to(dev()))
    x = torch.zeros((M, H), device=dev(), dtype=torch.bfloat16)
    offs = torch.zeros((E + 1,), dtype=torch.int32, device=dev())
    tok = torch.zeros((M, 20), dtype=torch.int64, device=dev())
    pres = torch.full((M,), 0.25, device=dev())

    def step():
        l = X.linear_mxfp4(x, w, ws, out_dtype=torch.float32)
        a, s = X.quantize_mxfp4(x)
        y = MR.grouped_linear_mxfp4(tables, "w13", a, s, offs)
        return l, y, TH.penalize_logits(l, output=tok, presence=pres)

    def fill(seed):
        h = np.random.default_rng(seed)
        x.copy_(torch.from_numpy(h.standard_normal((M, H)).astype(np.float32)))
        c = h.multinomial(M, np.full(E, 1 / E))
        offs.copy_(torch.from_numpy(np.concatenate([[0], np.cumsum(c)]).astype(np.int32)))
        tok.copy_(torch.from_numpy(h.integers(0, 330, (M, 20))))
    fill(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(1, 5):
        fill(seed)
        graph.replay()
        got = [t.clone() for t in outs]
        torch.cuda.synchronize()
        want = step()
        assert all(np.array_equal(bits(a), bits(b)) for a, b in zip(got, want)), seed
