"""The block-scaled fp8 quantisers and products (lockstep_fullstack.quantize_rows_fp8 / quantize_weight_fp8 /
dequant_fp8 / mm_fp8 / linear_fp8, moe_ref.grouped_linear_fp8) against a plain 64-bit statement (fp8_util).

Codes and scales are compared bit for bit.  Products whose every partial sum is a binary32 number are compared bit
for bit; the others within a bound that counts every rounding (fp8_util.bound), and in the 2-norm."""
import numpy as np
import pytest
import torch

import fp8_util as U
from gpu_util import bits, dev, say, to_dev

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import lockstep_amd._lib as L
    L.load()


def _bytes(q):
    return q.view(torch.uint8).cpu().numpy()


def _f8(code):
    return to_dev(code).view(F8)


def _values(g, M, K):
    x = g.standard_normal((M, K)) * np.exp2(g.integers(-6, 7, (M, K)))
    x[g.random((M, K)) < 0.02] = 0
    return x.astype(np.float32)


def _same_codes(q, scale, want):
    c, s = want
    assert np.array_equal(bits(scale.contiguous()), s.view(np.uint32))
    assert np.array_equal(_bytes(q), c)


# ---------------------------------------------------------------- the quantisers
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", [(1, 16), (1, 1040), (2, 128), (3, 272), (5, 6000), (17, 144), (37, 2880), (129, 4096), (300, 512)])
def test_quantize(M, K, dtype):
    from lockstep_amd import lockstep_fullstack as FS
    say("quantize", M, K, dtype)
    x = torch.from_numpy(_values(np.random.default_rng(M + K), M, K)).to(dtype)
    for weight, quantize in ((False, FS.quantize_rows_fp8), (True, FS.quantize_weight_fp8)):
        q, scale = quantize(x.to(dev()))
        want = U.quantize(x.double().numpy(), weight)
        _same_codes(q, scale, want)
        for odt in HALF:
            back = FS.dequant_fp8(q, scale, odt).cpu()
            exact = torch.from_numpy(U.values(*want, weight).astype(np.float32))  # one product of 28 bits, one rounding
            assert torch.equal(back, exact.to(odt))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_every_border(dtype):
    """Every midpoint between two codes and its neighbours in the input type, of both signs, with 448 beside them
    so that the scale is a power of two; zeros of both signs, the smallest and largest numbers, zero blocks."""
    from lockstep_amd import lockstep_fullstack as FS
    mids = torch.from_numpy(U.MID)
    rows = []
    for e in (0, -3, 5) if dtype != torch.float16 else (0, -3):
        base = (mids * 2.0 ** e).to(dtype)
        v = torch.cat([base, torch.nextafter(base, torch.full_like(base, float("inf"))),
                       torch.nextafter(base, torch.zeros_like(base)), torch.tensor([0.0, -0.0], dtype=dtype)])
        v = torch.nn.functional.pad(v, (0, -v.numel() % 127))
        v = torch.cat([v.reshape(-1, 127), torch.full((v.numel() // 127, 1), 448.0 * 2.0 ** e, dtype=dtype)], 1)
        rows += [v, -v]
    fi = torch.finfo(dtype)
    odd = torch.zeros(5, 128, dtype=dtype)
    odd[1] = -0.0
    odd[2] = fi.max
    odd[3, 5] = torch.nextafter(torch.tensor(0.0, dtype=dtype), torch.tensor(1.0, dtype=dtype))
    odd[4, ::3] = fi.tiny
    x = torch.cat(rows + [odd])
    _same_codes(*FS.quantize_rows_fp8(x.to(dev())), U.quantize(x.double().numpy()))


def test_quantize_infinities_and_nans():
    from lockstep_amd import lockstep_fullstack as FS
    x = np.random.default_rng(5).standard_normal((4, 400)).astype(np.float32)
    x[0, 3], x[1, 140], x[2, 399], x[3, 256] = np.inf, -np.inf, np.nan, -np.nan
    for weight, quantize in ((False, FS.quantize_rows_fp8), (True, FS.quantize_weight_fp8)):
        q, scale = quantize(to_dev(x))
        c, s = U.quantize(x, weight)
        assert np.isnan(s).sum() == 4
        bad = np.isnan(s)
        got = scale.cpu().numpy()
        assert np.array_equal(np.isnan(got), bad) and np.array_equal(got[~bad], s[~bad])
        nan = (c & 0x7f) == 0x7f
        assert np.array_equal(np.isnan(U.E4M3[_bytes(q)]), nan) and np.array_equal(_bytes(q)[~nan], c[~nan])
        back = FS.dequant_fp8(q, scale, torch.float32).cpu().numpy()
        assert np.array_equal(np.isnan(back), nan)


def test_quantize_strides_shapes_and_empty():
    from lockstep_amd import lockstep_fullstack as FS
    g = np.random.default_rng(6)
    big = torch.from_numpy(_values(g, 40, 320)).to(dev())
    for view in (big[:, 32:192], big[:, 1:257], big[::3, :64], big[3:4, 5:149], big.t()[:304].t(), big[:32].t()[:, :32],
                 big.to(torch.bfloat16)[:, 3:147], big[:1].expand(5, 320)):
        for weight, quantize in ((False, FS.quantize_rows_fp8), (True, FS.quantize_weight_fp8)):
            _same_codes(*quantize(view), U.quantize(view.double().cpu().numpy(), weight))
    q, s = FS.quantize_rows_fp8(big.reshape(4, 10, 320))
    assert q.shape == (4, 10, 320) and s.shape == (4, 10, 3)
    q2, s2 = FS.quantize_rows_fp8(big)
    assert torch.equal(q.reshape(40, 320).view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s.reshape(40, 3), s2)
    assert torch.equal(FS.dequant_fp8(q, s), FS.dequant_fp8(q2, s2).reshape(4, 10, 320))
    assert torch.equal(FS.dequant_fp8(q2[5:17, 128:256], s2[5:17, 1:2]), FS.dequant_fp8(q2, s2)[5:17, 128:256])
    q1, s1 = FS.quantize_rows_fp8(big[0])
    assert q1.shape == (320,) and s1.shape == (3,) and torch.equal(s1, s2[0])
    assert [t.shape for t in FS.quantize_rows_fp8(big[:0])] == [(0, 320), (0, 3)]
    assert [t.shape for t in FS.quantize_rows_fp8(big[:, :0])] == [(40, 0), (40, 0)]
    assert [t.shape for t in FS.quantize_weight_fp8(big[:, :0])] == [(40, 0), (1, 0)]
    assert FS.dequant_fp8(*FS.quantize_rows_fp8(big[:0])).shape == (0, 320)
    q64, _ = FS.quantize_rows_fp8(big[:2].double())
    assert torch.equal(q64.view(torch.uint8), q2[:2].view(torch.uint8))
    for bad in (big[:, :40], big.to(torch.int32)):
        with pytest.raises((ValueError, TypeError)):
            FS.quantize_rows_fp8(bad)
        with pytest.raises((ValueError, TypeError)):
            FS.quantize_weight_fp8(bad)


# ---------------------------------------------------------------- the product
SMALL = np.array([0.0, 1.0, 1.5, 2.0, 3.0, -1.0, -1.5, -2.0, -3.0])   # products: multiples of 1/4 up to 9


def _exact_operand(g, rows, K, octaves, weight):
    code = U.nearest(SMALL[g.integers(0, 9, (rows, K))])
    down = (rows + 127) // 128 if weight else rows
    return code, np.exp2(g.integers(-octaves, octaves + 1, (down, (K + 127) // 128))).astype(np.float32)


def _mm(qa, sa, qw, sw, bias=None, out_dtype=torch.float32):
    from lockstep_amd import lockstep_fullstack as FS
    return FS.mm_fp8(_f8(qa), to_dev(sa), _f8(qw), to_dev(sw), None if bias is None else to_dev(bias), out_dtype)


SIZES = [(1, 1, 16), (1, 17, 128), (2, 48, 144), (5, 33, 256), (16, 16, 400), (17, 100, 384), (31, 64, 512), (33, 257, 272),
         (64, 130, 1024), (65, 129, 640), (100, 300, 656), (129, 255, 256), (200, 520, 480), (257, 260, 544), (300, 1030, 128),
         (513, 512, 96), (600, 900, 32), (65, 5500, 64), (1100, 480, 96), (129, 3301, 160), (2000, 280, 1056), (3, 700, 4096),
         (20, 200, 5008), (40, 4200, 2064), (260, 516, 4128), (600, 1290, 1552)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_exact(M, N, K):
    """Every term is a multiple of 2^-2 (of 2^-6 with scales an octave up or down) and of a magnitude up to 9 (144), and
    9 K < 2^22 (144 K < 2^18 for K < 1820), so every partial sum is a binary32 number; eight products at a time lie
    within 2^6 of each other, far from what the fp8 instruction drops."""
    say("product exact", M, N, K)
    g = np.random.default_rng(M * N + K)
    octaves = 1 if K < 1820 else 0
    qa, sa = _exact_operand(g, M, K, octaves, False)
    qw, sw = _exact_operand(g, N, K, octaves, True)
    y, _ = U.product(qa, sa, qw, sw)
    assert np.array_equal(_mm(qa, sa, qw, sw).double().cpu().numpy(), y)
    bias = g.standard_normal(N).astype(np.float32)
    want = torch.from_numpy(y.astype(np.float32) + bias)            # one binary32 addition
    for odt in HALF:
        got = _mm(qa, sa, qw, sw, bias, odt)
        assert got.dtype == odt and torch.equal(got.cpu(), want.to(odt))


# sizes that between them reach every launch a product may take, one expert's and (below) several experts'
LAUNCHES = [(6278, 1934, 16), (2100, 3900, 400), (579, 10033, 16), (1500, 2050, 656), (278, 13067, 16), (500, 2050, 272),
            (1, 16, 16), (700, 2050, 144), (1419, 20, 560), (78, 13670, 2656), (1, 17, 1056), (15, 4078, 688), (4175, 17, 480),
            (17, 8206, 16), (224, 18, 432), (2118, 21, 1792), (2433, 18, 848), (6689, 17, 1632)]


@pytest.mark.parametrize("M,N,K", LAUNCHES)
def test_product_exact_on_every_launch(M, N, K):
    """As above; the largest sizes' rows in 64 bits are the same few, so that the oracle's product stays small."""
    say("product exact", M, N, K)
    g = np.random.default_rng(M + N * K)
    R, octaves = min(M, 300), 1 if K < 1820 else 0
    qa, sa = _exact_operand(g, R, K, octaves, False)
    qw, sw = _exact_operand(g, N, K, octaves, True)
    pick = g.integers(0, R, M)
    y = U.product(qa, sa, qw, sw)[0][pick]
    for odt in HALF:
        got = _mm(qa[pick], sa[pick], qw, sw, None, odt)
        assert torch.equal(got.cpu(), torch.from_numpy(y.astype(np.float32)).to(odt))


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1, 300, 4096), (7, 513, 2880), (32, 256, 14336), (50, 1000, 400), (150, 700, 3584),
                                   (333, 300, 1040), (700, 1100, 912)])
def test_product(M, N, K, out_dtype):
    say("product", M, N, K, out_dtype)
    g = np.random.default_rng(M + N + K)
    x = g.standard_normal((M, K))
    x[g.random((M, K)) < 0.001] *= 20
    qa, sa = U.quantize(x)
    qw, sw = U.quantize(g.standard_normal((N, K)) / np.sqrt(K), True)
    bias = g.standard_normal(N).astype(np.float32)
    y, mag = U.product(qa, sa, qw, sw, bias)
    got = _mm(qa, sa, qw, sw, bias, out_dtype).double().cpu().numpy()
    exact = out_dtype == torch.float32
    assert (np.abs(got - y) <= U.bound(y, mag, K, HALF[out_dtype], exact)).all()
    # in the 2-norm: half a step (an error is no larger than that of any value), and 2^-13 for what fp8 drops or
    # K / 32 + K / 64 roundings of 2^-24 of the largest partial sum, which is at most twice the result's size here
    off = np.linalg.norm(got - y) / np.linalg.norm(y)
    assert off <= HALF[out_dtype] + (K * 3 / 64 * 2.0 ** -23 if exact else 2.0 ** -13), off


def test_product_scales_of_any_stride():
    from lockstep_amd import lockstep_fullstack as FS
    g = np.random.default_rng(3)
    M, N, K = 70, 200, 700 // 16 * 16
    qa, sa = U.quantize(g.standard_normal((M, K)))
    qw, sw = U.quantize(g.standard_normal((N, K)), True)
    a, s, w, ws = _f8(qa), to_dev(sa), _f8(qw), to_dev(sw)
    for odt in (torch.float32, torch.bfloat16):
        want = FS.mm_fp8(a, s, w, ws, out_dtype=odt)
        wide = torch.full((2 * M, 3 * s.shape[1] + 5), float("nan"), device=dev())
        wide[::2, 2:2 + 2 * s.shape[1]:2] = s
        for other in (s.t().contiguous().t(), wide[::2, 2:2 + 2 * s.shape[1]:2]):
            assert not other.is_contiguous() and torch.equal(FS.mm_fp8(a, other, w, ws, out_dtype=odt), want)
        one = torch.full((1, 1), 0.25, device=dev()).expand(M, s.shape[1])
        assert torch.equal(FS.mm_fp8(a, one, w, ws, out_dtype=odt), FS.mm_fp8(a, one.contiguous(), w, ws, out_dtype=odt))
        # one row, and one block, of a tensor whose strides no product could step by
        far = s[:1].contiguous().as_strided((1, s.shape[1]), (1 << 40, 1))
        assert torch.equal(FS.mm_fp8(a[:1], far, w, ws, out_dtype=odt), want[:1])
        far = s[:, :1].as_strided((M, 1), (s.stride(0), 1 << 40))
        assert torch.equal(FS.mm_fp8(a[:, :128].contiguous(), far, w[:, :128], ws[:, :1], out_dtype=odt),
                           FS.mm_fp8(a[:, :128].contiguous(), s[:, :1], w[:, :128], ws[:, :1], out_dtype=odt))
        # codes and weight scales as views: copied
        big = torch.zeros((M, 2 * K), dtype=torch.uint8, device=dev()).view(F8)
        big.view(torch.uint8)[:, 8:8 + K] = a.view(torch.uint8)
        assert torch.equal(FS.mm_fp8(big[:, 8:8 + K], s, w, ws.t().contiguous().t(), out_dtype=odt), want)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K", [(130, 1040), (4200, 272), (1030, 2880)])
def test_a_row_is_the_same_bits_in_every_batch(N, K, out_dtype):
    """Codes over all of e4m3, so that the order of additions and what the instruction drops show."""
    from lockstep_amd import lockstep_fullstack as FS
    g = np.random.default_rng(N)
    M = 1100
    qa = g.integers(0, 256, (M, K), dtype=np.uint8)
    qa[(qa & 127) == 127] = 5
    qw = g.integers(0, 256, (N, K), dtype=np.uint8)
    qw[(qw & 127) == 127] = 9
    sa = np.exp(g.standard_normal((M, (K + 127) // 128))).astype(np.float32)
    sw = np.exp(g.standard_normal(((N + 127) // 128, (K + 127) // 128))).astype(np.float32)
    a, s, w, ws = _f8(qa), to_dev(sa), _f8(qw), to_dev(sw)
    full = FS.mm_fp8(a, s, w, ws, out_dtype=out_dtype)
    for m in (1, 2, 4, 7, 16, 17, 32, 33, 64, 65, 100, 128, 200, 256, 300, 520, 1000):
        say("rows", m, "of", N, K, out_dtype)
        for at in (0, M - m):
            got = FS.mm_fp8(a[at:at + m], s[at:at + m], w, ws, out_dtype=out_dtype)
            assert np.array_equal(bits(got), bits(full[at:at + m]))


def test_nans_stay_in_their_rows_and_columns():
    from lockstep_amd import lockstep_fullstack as FS
    g = np.random.default_rng(8)
    for M in (3, 40, 300):
        x = g.standard_normal((M, 400)).astype(np.float32)
        W = g.standard_normal((300, 400)).astype(np.float32)
        qw, sw = FS.quantize_weight_fp8(to_dev(W))
        for odt in (torch.float32, torch.bfloat16):
            clean = FS.linear_fp8(to_dev(x), qw, sw, out_dtype=odt)
            y = x.copy()
            y[1, 399], y[2, 0] = np.nan, np.inf
            got = FS.linear_fp8(to_dev(y), qw, sw, out_dtype=odt)
            assert torch.isnan(got[1:3]).all()
            keep = [0] + list(range(3, M))
            assert torch.equal(got[keep], clean[keep])
            V = W.copy()
            V[130, 7] = np.inf                        # rows 128 to 255 share the block
            got = FS.linear_fp8(to_dev(x), *FS.quantize_weight_fp8(to_dev(V)), out_dtype=odt)
            assert torch.isnan(got[:, 128:256]).all()
            assert torch.equal(got[:, :128], clean[:, :128]) and torch.equal(got[:, 256:], clean[:, 256:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1, 100, 512), (1, 64, 20000), (3, 130, 1040), (16, 64, 512), (16, 300, 2880), (40, 200, 144),
                                   (300, 520, 656)])
def test_linear_is_mm_of_the_quantised_rows(M, N, K, dtype):
    from lockstep_amd import lockstep_fullstack as FS
    say("linear", M, N, K, dtype)
    g = np.random.default_rng(M + N)
    x = torch.from_numpy(_values(g, M, K)).to(dtype).to(dev())
    w, ws = FS.quantize_weight_fp8(torch.from_numpy(_values(g, N, K)).to(dev()))
    bias = to_dev(g.standard_normal(N).astype(np.float32))
    for b in (None, bias):
        for odt in (None, torch.float32, torch.bfloat16):
            got = FS.linear_fp8(x, w, ws, b, odt)
            want = FS.mm_fp8(*FS.quantize_rows_fp8(x), w, ws, b, odt or dtype)
            assert got.dtype == (odt or dtype) and np.array_equal(bits(got), bits(want))
    odd = torch.zeros((M, K + 3), dtype=dtype, device=dev())
    odd[:, 1:K + 1] = x
    assert np.array_equal(bits(FS.linear_fp8(odd[:, 1:K + 1], w, ws)), bits(FS.linear_fp8(x, w, ws)))


@pytest.mark.parametrize("M,N,K", [(17, 100, 512), (64, 2048, 512), (200, 500, 1024), (33, 17, 16), (130, 260, 656), (500, 16, 1024),
                                   (8192, 16, 32), (8193, 16, 32), (129, 1024, 144), (128, 1025, 144),
                                   (1, 4096, 20480), (1, 4097, 16400), (16, 4096, 1280), (16, 130, 1296), (13, 4097, 1264)])
def test_linear_of_rows_quantised_by_every_block(M, N, K):
    """Sizes on both sides of where a linear quantises its rows in the product's launch; rows at any place."""
    from lockstep_amd import lockstep_fullstack as FS
    say("linear", M, N, K)
    g = np.random.default_rng(M + N + K)
    w, ws = FS.quantize_weight_fp8(to_dev(_values(g, N, K)))
    bias = to_dev(g.standard_normal(N).astype(np.float32))
    wide = to_dev(np.concatenate([_values(g, M, K), _values(g, M, 5)], 1))
    for dtype in HALF:
        x = wide.to(dtype)
        for view in (x[:, :K].contiguous(), x[:, 3:3 + K]):
            for odt in (torch.float32, torch.bfloat16):
                want = FS.mm_fp8(*FS.quantize_rows_fp8(view), w, ws, bias, odt)
                assert np.array_equal(bits(FS.linear_fp8(view, w, ws, bias, odt)), bits(want))


def test_linear_shapes_and_empty():
    from lockstep_amd import lockstep_fullstack as FS
    g = np.random.default_rng(9)
    x = to_dev(_values(g, 6, 160))
    w, ws = FS.quantize_weight_fp8(to_dev(_values(g, 20, 160)))
    y = FS.linear_fp8(x, w, ws)
    assert torch.equal(FS.linear_fp8(x.reshape(2, 3, 160), w, ws), y.reshape(2, 3, 20))
    assert torch.equal(FS.linear_fp8(x[2], w, ws), y[2])
    assert FS.linear_fp8(x[:0], w, ws).shape == (0, 20)
    assert FS.linear_fp8(x, w[:0], ws[:0]).shape == (6, 0)
    bias = to_dev(g.standard_normal(20).astype(np.float32))
    empty = w.view(torch.uint8)[:, :0].view(F8)
    for M in (6, 300):
        x0 = torch.zeros((M, 0), device=dev())
        assert torch.equal(FS.linear_fp8(x0, empty, ws[:, :0], bias), bias.expand(M, 20))
        assert torch.equal(FS.linear_fp8(x0, empty, ws[:, :0]), torch.zeros((M, 20), device=dev()))


# ---------------------------------------------------------------- by expert
def _experts(g, E, H, I, bias):
    from lockstep_amd import lockstep_fullstack as FS
    out = []
    for _ in range(E):
        w13, w2 = (FS.quantize_weight_fp8(to_dev(g.standard_normal(s).astype(np.float32))) for s in ((2 * I, H), (H, I)))
        b = [to_dev(g.standard_normal(n).astype(np.float32)) if bias else None for n in (2 * I, H)]
        out.append((w13, w2, *b))
    return out


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts,H,I,bias", [([1], 128, 64, False), ([0, 3, 0, 1], 144, 80, True), ([5, 0, 17, 40, 2], 288, 192, False),
                                             ([64, 65, 130, 0, 1, 300], 272, 144, True), ([700, 3, 200], 512, 336, False),
                                             ([2] * 70 + [0] * 20 + [90], 128, 48, True)])
def test_grouped_is_mm_of_each_expert(counts, H, I, bias, out_dtype):
    from lockstep_amd import lockstep_fullstack as FS, moe_ref
    say("grouped", counts[:8], H, I, out_dtype)
    g = np.random.default_rng(H + I)
    ex = _experts(g, len(counts), H, I, bias)
    t = moe_ref.ExpertTablesFP8(ex)
    offs = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    R = int(offs[-1])
    for which, K, j in (("w13", H, 0), ("w2", I, 1)):
        a, s = FS.quantize_rows_fp8(to_dev(g.standard_normal((R, K)).astype(np.float32)))
        for scale in (s, s.contiguous()):
            got = moe_ref.grouped_linear_fp8(t, which, a, scale, to_dev(offs), out_dtype)
            for e in range(len(counts)):
                rows = slice(offs[e], offs[e + 1])
                want = FS.mm_fp8(a[rows], s[rows], *ex[e][j], ex[e][2 + j], out_dtype)
                assert np.array_equal(bits(got[rows]), bits(want)), (which, e)


@pytest.mark.parametrize("R,N,K,E", [(1880, 6048, 272, 6), (443, 9920, 16, 6), (10, 13504, 16, 6), (1, 16, 16, 6), (1185, 32, 528, 6),
                                     (362, 2560, 2896, 6), (1, 16, 1040, 6), (3, 13856, 32, 6), (9, 3648, 16, 6), (357, 16, 416, 6),
                                     (4593, 16, 1360, 6), (3682, 16, 784, 6), (70, 1104, 1024, 6), (3235, 1408, 16, 40),
                                     (56, 2144, 16, 40), (50, 544, 16, 40), (541, 144, 1088, 40)])
def test_grouped_exact_on_every_launch(R, N, K, E):
    """Random counts, some experts empty, rows behind the last expert: those stay what they were."""
    from lockstep_amd import _lib as L
    say("grouped exact", R, N, K, E)
    g = np.random.default_rng(R * E + N)
    octaves = 1 if K < 1820 else 0
    qa, sa = _exact_operand(g, min(R, 300), K, octaves, False)
    pick = g.integers(0, len(qa), R)
    qa, sa = qa[pick], sa[pick]
    weights = [_exact_operand(g, N, K, octaves, True) for _ in range(min(E, 7))]
    held = [(to_dev(q), to_dev(s)) for q, s in weights]
    part = g.random(E) * (g.random(E) < 0.8) + 1e-9
    offs = np.concatenate([[0], np.cumsum(part) / part.sum() * R * (0.9 if R > 20 else 1)]).astype(np.int32)
    y = np.full((R, N), 7.0)
    for e in range(E):
        rows = slice(offs[e], offs[e + 1])
        y[rows] = U.product(qa[rows], sa[rows], *weights[e % len(weights)])[0]
    a, s, o = to_dev(qa), to_dev(sa), to_dev(offs)
    wp, sp = (to_dev(np.array([held[e % len(held)][j].data_ptr() for e in range(E)], np.int64)) for j in (0, 1))
    for odt in (torch.float32, torch.bfloat16):
        out = torch.full((R, N), 7.0, dtype=odt, device=dev())
        L.call("lsk_grouped_gemm_fp8", a.data_ptr(), s.data_ptr(), s.stride(0), s.stride(1), o.data_ptr(), E, R, wp.data_ptr(), K,
               sp.data_ptr(), (K + 127) // 128, None, N, K, out.data_ptr(), L.LSK_F32 if odt == torch.float32 else L.LSK_BF16, N,
               L.stream_of(a))
        assert torch.equal(out.cpu(), torch.from_numpy(y.astype(np.float32)).to(odt))


def test_grouped_offsets_out_of_order_and_rows_of_no_expert():
    """Offsets as min(R, max(0, the largest so far)); rows before the first and behind the last expert keep what lay there."""
    from lockstep_amd import _lib as L, lockstep_fullstack as FS, moe_ref
    g = np.random.default_rng(12)
    H, I, R = 256, 128, 90
    ex = _experts(g, 4, H, I, False)
    t = moe_ref.ExpertTablesFP8(ex)
    a, s = FS.quantize_rows_fp8(to_dev(g.standard_normal((R, H)).astype(np.float32)))
    for offs in ([0, 20, 10, 50, 70], [-5, 30, 200, 90, 90], [7, 7, 40, 41, 60], [0, 0, 0, 0, 0], [90, 95, 100, 90, 91], [500, 0, 0, 1, 2]):
        say("offsets", offs)
        eff = np.clip(np.maximum.accumulate(np.clip(offs, 0, R)), 0, R)
        out = torch.full((R, 2 * I), 7.0, dtype=torch.bfloat16, device=dev())
        o = to_dev(np.array(offs, np.int32))
        L.call("lsk_grouped_gemm_fp8", a.data_ptr(), s.data_ptr(), s.stride(0), s.stride(1), o.data_ptr(), 4, R,
               t.w13.data_ptr(), H, t.ws13.data_ptr(), 2, None, 2 * I, H, out.data_ptr(), L.LSK_BF16, 2 * I, L.stream_of(a))
        want = torch.full_like(out, 7.0)
        for e in range(4):
            rows = slice(int(eff[e]), int(eff[e + 1]))
            want[rows] = FS.mm_fp8(a[rows], s[rows], *ex[e][0], None, torch.bfloat16)
        assert np.array_equal(bits(out), bits(want))
    assert moe_ref.grouped_linear_fp8(t, "w13", a[:0], s[:0], to_dev(np.zeros(5, np.int32))).shape == (0, 2 * I)


def test_grouped_refusals():
    from lockstep_amd import lockstep_fullstack as FS, moe_ref
    g = np.random.default_rng(13)
    ex = _experts(g, 2, 128, 64, False)
    t = moe_ref.ExpertTablesFP8(ex)
    a, s = FS.quantize_rows_fp8(to_dev(g.standard_normal((4, 128)).astype(np.float32)))
    offs = to_dev(np.array([0, 2, 4], np.int32))
    for bad in (lambda: moe_ref.grouped_linear_fp8(t, "w3", a, s, offs), lambda: moe_ref.grouped_linear_fp8(ex, "w13", a, s, offs),
                lambda: moe_ref.grouped_linear_fp8(t, "w13", a, s, offs.long()),
                lambda: moe_ref.grouped_linear_fp8(t, "w13", a, s, offs[:2]),
                lambda: moe_ref.grouped_linear_fp8(t, "w2", a, s, offs), lambda: moe_ref.grouped_linear_fp8(t, "w13", a, s[:3], offs),
                lambda: moe_ref.grouped_linear_fp8(t, "w13", a.view(torch.uint8), s, offs),
                lambda: moe_ref.ExpertTablesFP8([]), lambda: moe_ref.ExpertTablesFP8([ex[0], _experts(g, 1, 144, 64, False)[0]]),
                lambda: moe_ref.ExpertTablesFP8([ex[0][:2] + (to_dev(np.zeros(128, np.float32)), None), ex[1]])):
        with pytest.raises((ValueError, TypeError)):
            bad()


# ---------------------------------------------------------------- how programs call them
def test_other_stream_and_graph():
    from lockstep_amd import lockstep_fullstack as FS
    g = np.random.default_rng(14)
    w, ws = FS.quantize_weight_fp8(to_dev(_values(g, 300, 656)))
    for M in (1, 9, 40, 400):
        x = to_dev(_values(g, M, 656)).to(torch.bfloat16)
        want = FS.linear_fp8(x, w, ws)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = FS.linear_fp8(x, w, ws)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        xs = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = FS.linear_fp8(xs, w, ws)
        for i in range(4):
            xs.copy_(x * (i + 1) if i % 2 else x - i)
            graph.replay()
            eager = FS.linear_fp8(xs, w, ws)
            torch.cuda.synchronize()
            assert torch.equal(y, eager)


def test_offsets_beyond_32_bits():
    """The last rows of tensors past 2^32 elements, as the same rows alone give them."""
    from lockstep_amd import lockstep_fullstack as FS, moe_ref, t16n_ref
    g = np.random.default_rng(15)
    M, K, n = 2 ** 20 + 5, 4096, 7
    x = torch.zeros((M, K), dtype=torch.bfloat16, device=dev())
    x[-n:] = torch.from_numpy(_values(g, n, K)).to(torch.bfloat16)
    few = x[-n:].clone()
    say("quantise", M, K)
    q, s = FS.quantize_rows_fp8(x)
    qf, sf = FS.quantize_rows_fp8(few)
    assert torch.equal(q[-n:].view(torch.uint8), qf.view(torch.uint8)) and torch.equal(s[-n:], sf)
    w, ws = FS.quantize_weight_fp8(to_dev(_values(g, 40, K)))
    say("products", M, K)
    for odt in (torch.bfloat16, torch.float32):
        assert torch.equal(FS.mm_fp8(q, s, w, ws, out_dtype=odt)[-n:], FS.mm_fp8(qf, sf, w, ws, out_dtype=odt))
        assert torch.equal(FS.linear_fp8(x, w, ws, out_dtype=odt)[-n:], FS.linear_fp8(few, w, ws, out_dtype=odt))
    say("by expert", M, K)
    I = 32
    tables = moe_ref.ExpertTablesFP8([tuple(FS.quantize_weight_fp8(to_dev(_values(g, *shape))) for shape in ((2 * I, K), (K, I)))
                                      for _ in range(2)])
    offs = torch.tensor([0, M - n - 1, M], dtype=torch.int32, device=dev())
    last = torch.tensor([0, 0, n], dtype=torch.int32, device=dev())
    y = moe_ref.grouped_linear_fp8(tables, "w13", q, s, offs)
    assert torch.equal(y[-n:], moe_ref.grouped_linear_fp8(tables, "w13", qf, sf, last))
    act, acts = FS.quantize_rows_fp8(y[:, :I].contiguous())
    y = moe_ref.grouped_linear_fp8(tables, "w2", act, acts, offs)
    assert torch.equal(y[-n:], moe_ref.grouped_linear_fp8(tables, "w2", act[-n:], acts[-n:], last))
    del y
    say("dequantise", M, K)
    assert torch.equal(FS.dequant_fp8(q, s)[-n:], FS.dequant_fp8(qf, sf))
    del q, s
    say("norm", M, K)
    gain = to_dev(_values(g, 1, K)[0])
    for a, b in zip(t16n_ref.add_rmsnorm_fp8(x, x, gain, want_out=True), t16n_ref.add_rmsnorm_fp8(few, few, gain, want_out=True)):
        assert np.array_equal(bits(a[-n:].contiguous().view(torch.uint8)) if a.dtype == F8 else bits(a[-n:].contiguous()),
                              bits(b.contiguous().view(torch.uint8)) if b.dtype == F8 else bits(b.contiguous()))
    del x
    say("outputs", 70000, 65536)
    a, s = FS.quantize_rows_fp8(to_dev(_values(g, 70000, 16)))
    w, ws = FS.quantize_weight_fp8(to_dev(_values(g, 65536, 16)))
    for odt in (torch.bfloat16, torch.float32):
        out = FS.mm_fp8(a, s, w, ws, out_dtype=odt)
        assert torch.equal(out[-n:], FS.mm_fp8(a[-n:], s[-n:], w, ws, out_dtype=odt))
        del out
    say("route", 2 ** 22 + 3, 1024)
    z = torch.zeros((2 ** 22 + 3, 1024), device=dev())
    z[-n:] = to_dev(_values(g, n, 1024))
    for a, b in zip(moe_ref.route_experts(z, 8), moe_ref.route_experts(z[-n:].clone(), 8)):
        assert torch.equal(a[-n:], b)


def test_two_streams_at_once():
    """Products of two streams side by side, each with a workspace of its own."""
    from lockstep_amd import lockstep_fullstack as FS
    g = np.random.default_rng(16)
    w, ws = FS.quantize_weight_fp8(to_dev(_values(g, 2000, 2048)))
    xs = [to_dev(_values(g, m, 2048)).to(torch.bfloat16) for m in (300, 300, 1, 40)]
    want = [FS.linear_fp8(x, w, ws) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(24):
        with torch.cuda.stream(streams[i % 2]):
            got.append((i % 4, FS.linear_fp8(xs[i % 4], w, ws)))
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[i])
