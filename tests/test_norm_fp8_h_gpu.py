"""lsk_add_rmsnorm_fp8 without a residual but with an h: x itself, whatever it holds, at every number of groups a lane holds."""
import numpy as np
import pytest
import torch

from gpu_util import bits

pytestmark = pytest.mark.gpu

NAN = {torch.bfloat16: (0x7f80, 0x7f), torch.float16: (0x7c00, 0x3ff), torch.float32: (0x7f800000, 0x7fffff)}   # exponent, payload


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R,N", [(7, 1040), (2050, 2064), (5, 16400), (5, 32768), (4, 65520)])     # 1, 2 (1 in binary32), 4, 4 and 8 groups
def test_h_without_a_residual(R, N, dtype):
    from lockstep_amd import _lib as L, t16n_ref
    print("h without a residual", R, N, dtype, flush=True)
    g = torch.Generator(device="cuda").manual_seed(N)
    x = torch.randn((R, N), generator=g, device="cuda").to(dtype)
    raw = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
    top, payload = NAN[dtype]
    sign = -1 << (31 if dtype == torch.float32 else 15)
    for i, p in enumerate((1, payload, (payload + 1) // 2, payload // 2, 3)):      # signalling and quiet ones of both signs
        raw[1, 11 + 37 * i] = top | p
        raw[R - 1, N - 1 - 50 * i] = (top | p) + sign
    raw[2, 5], raw[2, N - 3], raw[0, 1], raw[0, N - 9], raw[0, 40] = top, top + sign, sign, 1, 1 + sign
    gain = torch.ones(N, device="cuda")
    nb = (N + 127) // 128
    h, q, s = torch.zeros_like(x), torch.empty((R, N), dtype=torch.uint8, device="cuda"), torch.empty((nb, R), device="cuda")
    L.call("lsk_add_rmsnorm_fp8", x.data_ptr(), L.dtype_code(dtype), N, None, 0, R, N, gain.data_ptr(), L.LSK_F32, 0.0, 1e-6,
           h.data_ptr(), N, q.data_ptr(), s.data_ptr(), 1, R, None, L.stream_of(x))
    nan = torch.isnan(x).cpu().numpy()
    assert nan.sum() == 10
    got, want = bits(h), bits(x)
    assert np.array_equal(got[~nan], want[~nan])
    if dtype == torch.bfloat16:                       # as every conversion to bf16 gives one
        assert (got[nan] == 0x7fc0).all()
    elif dtype == torch.float32:
        assert np.array_equal(got[nan], want[nan])
    else:
        assert torch.isnan(h).cpu().numpy()[nan].all()
    # and the rows are those of a call without an h
    q2, s2, same, _ = t16n_ref.add_rmsnorm_fp8(x, None, gain, eps=1e-6)
    assert same is x and torch.equal(q2.view(torch.uint8), q) and np.array_equal(bits(s2.t()), bits(s))
