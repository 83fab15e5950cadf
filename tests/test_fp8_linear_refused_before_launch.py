"""linear_fp8 looks over everything it may refuse before its first launch: what it refuses has started nothing, so that
the workspace is as it was."""
from lockstep_amd import _lib as L

P = 1 << 20      # a plausible, 256-byte aligned address: every call here is refused before it is used


def _linear(M, N, K, odt=L.LSK_BF16):
    lib = L.load()
    rc = lib.lsk_linear_fp8(P, L.LSK_BF16, K, M, K, P, P, N, None, P, odt, N, P, lib.lsk_linear_fp8_workspace(M, N, K), None)
    return rc, lib.lsk_last_error()


def test_scales_beyond_reach():
    rc, err = _linear(1 << 22, 64, 16384)        # 2^22 rows of 128 scales, 2^31 bytes
    assert rc == 1 and b"31-bit offsets" in err, (rc, err)


def test_products_beyond_a_grid():
    for odt in (L.LSK_BF16, L.LSK_F32):
        rc, err = _linear(1 << 24, (1 << 31) - 1, 2048, odt)
        assert rc == 1 and b"grid too large" in err, (rc, err)


def test_rows_beyond_the_quantisers_grid():
    rc, err = _linear(1 << 29, 16, 16)
    assert rc == 1 and b"grid too large" in err, (rc, err)
