"""t16n_ref.add_rmsnorm_fp8 against its parts: the addition rounded once, the contract's norm of it (its sum and its
bf16 output are pinned by the published digests), and fp8 rows of the norm's binary32 steps, all bit for bit."""
import numpy as np
import pytest
import torch

import fp8_util as U
from gpu_util import bits, dev, say, to_dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import lockstep_amd._lib as L
    L.load()


def _expect(h, gain, eps):
    """(codes, scales) by the declared binary32 steps from the row sums."""
    from lockstep_amd import t16n_ref as N
    n = h.shape[-1]
    S = N.row_sum_float(h).cpu().numpy().astype(np.float32)
    ne = np.float32(N.eps_term(n, eps))
    S = S + ne if eps else S
    S = np.where(S < np.float32(2.0 ** -126), np.float32(2.0 ** -126), S)
    rs = np.float32(N.sqrt_n(n)) / np.sqrt(S)
    with np.errstate(all="ignore"):
        y = h.float().cpu().numpy() * rs[:, None]
        y = y * gain.float().cpu().numpy()[None]
    assert y.dtype == np.float32
    return U.quantize(y)


def _check(x, residual, gain, eps):
    from lockstep_amd import t16n_ref as N
    q, s, h, out = N.add_rmsnorm_fp8(x, residual, gain, eps=eps, want_out=True)
    want_h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    assert np.array_equal(bits(h), bits(want_h))
    assert np.array_equal(bits(out), bits(N.rmsnorm_float(h, gain, eps=eps)))
    c, sc = _expect(h, gain, eps)
    assert np.array_equal(bits(s.contiguous()), sc.view(np.uint32)) and np.array_equal(q.view(torch.uint8).cpu().numpy(), c)
    q2, s2, h2, none = N.add_rmsnorm_fp8(x, residual, gain, eps=eps)
    assert none is None and torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s) and torch.equal(h2, h)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,N", [(1, 16), (3, 128), (2, 144), (5, 512), (4, 528), (1, 3584), (33, 2880), (3, 4096), (2, 8208), (2, 18944),
                                 (1, 40000), (1, 65536)])
def test_against_its_parts(R, N, dtype):
    say("norm", R, N, dtype)
    g = np.random.default_rng(R + N)
    x = to_dev(g.standard_normal((R, N)).astype(np.float32)).to(dtype)
    r = to_dev((4 * g.standard_normal((R, N))).astype(np.float32)).to(dtype)
    gain = to_dev((1 + 0.2 * g.standard_normal(N)).astype(np.float32))
    _check(x, r, gain, 1e-6)
    _check(x, None, gain.to(dtype), 0.0)
    _check(x, r, gain.to(torch.bfloat16), 1e-5)


def test_many_rows():
    g = torch.Generator(device="cuda").manual_seed(1)
    x, r = (torch.randn((1500, 1040), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    _check(x, r, torch.ones(1040, device="cuda"), 1e-6)


def test_strides_shapes_and_empty():
    from lockstep_amd import t16n_ref as N
    g = torch.Generator(device="cuda").manual_seed(2)
    big, other = (torch.randn((12, 600), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    gain = torch.rand(272, generator=g, device="cuda")
    want = [N.add_rmsnorm_fp8(a.contiguous(), b.contiguous(), gain, eps=1e-6) for a, b in ((big[:, 1:273], other[:, 8:280]),)][0]
    for a, b in ((big[:, 1:273], other[:, 8:280]), (big[:, 1:273].t().contiguous().t(), other[:, 8:280]),
                 (big[:, 1:273].contiguous(), other[:, 8:280])):
        got = N.add_rmsnorm_fp8(a, b, gain, eps=1e-6)
        assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
        assert torch.equal(got[2], want[2])
    q, s, h, _ = N.add_rmsnorm_fp8(big[:, 1:273].reshape(3, 4, 272), other[:, 8:280].reshape(3, 4, 272), gain, eps=1e-6)
    assert q.shape == h.shape == (3, 4, 272) and s.shape == (3, 4, 3)
    assert torch.equal(s.reshape(12, 3), want[1]) and torch.equal(h.reshape(12, 272), want[2])
    one = N.add_rmsnorm_fp8(big[2, 1:273], other[2, 8:280], gain, eps=1e-6)
    assert torch.equal(one[0].view(torch.uint8), want[0].view(torch.uint8)[2]) and torch.equal(one[1], want[1][2])
    q, s, h, out = N.add_rmsnorm_fp8(big[:0, :32], other[:0, :32], gain[:32], want_out=True)
    assert q.shape == h.shape == out.shape == (0, 32) and s.shape == (0, 1)
    for bad in (lambda: N.add_rmsnorm_fp8(big[:, :40], None, gain[:40]), lambda: N.add_rmsnorm_fp8(big, other[:, :592], gain),
                lambda: N.add_rmsnorm_fp8(big[:, :272], other[:, :272].float(), gain), lambda: N.add_rmsnorm_fp8(big.int(), None, gain),
                lambda: N.add_rmsnorm_fp8(big[:, :272], None, gain[:100])):
        with pytest.raises((ValueError, TypeError)):
            bad()


def test_nonfinite_and_zero_rows():
    from lockstep_amd import t16n_ref as N
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((5, 400), generator=g, device="cuda")
    x[1, 7], x[2, 399], x[3] = float("nan"), float("inf"), 0.0
    gain = torch.ones(400, device="cuda")
    q, s, h, _ = N.add_rmsnorm_fp8(x, torch.zeros_like(x), gain, eps=1e-6)
    assert torch.isnan(s[1]).all() and torch.isnan(q[1].float()).all()
    # an infinity: rs = 0, so the row is 0 but for its own place, which is NaN and takes its block along
    assert torch.isnan(s[2, 3]) and not torch.isnan(s[2, :3]).any() and (q[2, :384].float() == 0).all()
    assert (q[3].float() == 0).all() and not torch.isnan(s[3]).any()
    ref = N.add_rmsnorm_fp8(x[[0, 4]], None, gain, eps=1e-6)
    assert torch.equal(q.view(torch.uint8)[[0, 4]], ref[0].view(torch.uint8)) and torch.equal(s[[0, 4]], ref[1])


def test_in_place_residual_through_c():
    """h may be the residual's own memory."""
    from lockstep_amd import _lib as L, t16n_ref as N
    g = torch.Generator(device="cuda").manual_seed(4)
    x, r = (torch.randn((20, 1040), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    gain = torch.ones(1040, device="cuda")
    q, s, h, _ = N.add_rmsnorm_fp8(x, r, gain, eps=1e-6)
    q2, s2 = torch.empty_like(q), torch.empty((9, 20), device="cuda")
    L.call("lsk_add_rmsnorm_fp8", x.data_ptr(), L.LSK_BF16, 1040, r.data_ptr(), 1040, 20, 1040, gain.data_ptr(), L.LSK_F32, 0.0,
           1e-6, r.data_ptr(), 1040, q2.data_ptr(), s2.data_ptr(), 1, 20, None, L.stream_of(x))
    assert torch.equal(r, h) and torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2.t(), s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,N", [(2050, 2064), (2048, 4096), (3000, 8208)])
def test_a_row_is_the_same_in_every_batch(R, N, dtype):
    """However many groups a lane holds; NaNs and infinities among the rows."""
    from lockstep_amd import t16n_ref as T
    say("norm", R, N, dtype)
    g = torch.Generator(device="cuda").manual_seed(R)
    x, r = ((3 * torch.randn((R, N), generator=g, device="cuda")).to(dtype) for _ in range(2))
    x[5, 7], x[5, 9], x[R - 1, N - 1], r[9, 3], x[9, 3] = float("nan"), -float("nan"), float("nan"), -float("inf"), float("inf")
    gain = (1 + 0.1 * torch.randn(N, generator=g, device="cuda")).to(dtype)
    full = T.add_rmsnorm_fp8(x, r, gain, eps=1e-6, want_out=True)
    for rows in (slice(0, 1), slice(4, 12), slice(R - 3, R)):
        few = T.add_rmsnorm_fp8(x[rows], r[rows], gain, eps=1e-6, want_out=True)
        for a, b in zip(full, few):
            a, b = a[rows].contiguous(), b.contiguous()
            if dtype == torch.float32 and a.dtype == torch.float32:
                a, b = a.nan_to_num(nan=1e30, posinf=2e30), b.nan_to_num(nan=1e30, posinf=2e30)
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_h_without_a_residual_through_c():
    """h is then x, a NaN of bf16 as every conversion to it gives one."""
    from lockstep_amd import _lib as L
    for dt, code in ((torch.bfloat16, L.LSK_BF16), (torch.float16, L.LSK_F16), (torch.float32, L.LSK_F32)):
        x = torch.randn((7, 1040), device="cuda").to(dt)
        gain = torch.ones(1040, device="cuda")
        h, q, s = torch.zeros_like(x), torch.empty((7, 1040), dtype=torch.uint8, device="cuda"), torch.empty((9, 7), device="cuda")
        L.call("lsk_add_rmsnorm_fp8", x.data_ptr(), code, 1040, None, 0, 7, 1040, gain.data_ptr(), L.LSK_F32, 0.0, 1e-6,
               h.data_ptr(), 1040, q.data_ptr(), s.data_ptr(), 1, 7, None, L.stream_of(x))
        assert torch.equal(h, x)
