"""What the MXFP4 and logits entry points refuse, at the C boundary and in Python, without a GPU."""
import pytest
import torch

from lockstep_amd import _lib as L
from lockstep_amd import moe_mxfp4, moe_ref, t16h_lmvariants

P = 1 << 20      # a plausible, 256-byte aligned address: every call here is refused before it is used


def _refused(rc, word):
    lib = L.load()
    assert rc == 1 and word in lib.lsk_last_error(), (rc, lib.lsk_last_error())


def test_quantize_refusals():
    q = L.load().lsk_quantize_mxfp4
    _refused(q(P, L.LSK_I8, 1, 32, 32, P, P, None), b"x_dtype")
    _refused(q(P, L.LSK_F32, 1, 33, 33, P, P, None), b"multiple of 32")
    _refused(q(P, L.LSK_F32, -1, 32, 32, P, P, None), b"multiple of 32")
    _refused(q(P, L.LSK_F32, 2, 64, 32, P, P, None), b"ldx")
    _refused(q(None, L.LSK_F32, 2, 64, 64, P, P, None), b"null")
    _refused(q(P, L.LSK_F32, 2, 64, 64, P + 2, P, None), b"aligned")
    assert q(None, L.LSK_F32, 0, 64, 64, None, None, None) == 0
    assert q(None, L.LSK_F32, 5, 0, 0, None, None, None) == 0


def test_product_refusals():
    lib = L.load()

    def gemm(M=4, K=64, N=8, odt=L.LSK_F32, ldo=8, a=P, w=P, out=P):
        return lib.lsk_gemm_mxfp4(a, P, M, K, w, P, N, None, out, odt, ldo, None, 0, None)
    _refused(gemm(K=48), b"multiple of 32")
    _refused(gemm(M=-1), b"bad sizes")
    _refused(gemm(odt=L.LSK_I32), b"out_dtype")
    _refused(gemm(ldo=7), b"ldo")
    _refused(gemm(a=P + 8), b"16-byte")
    _refused(gemm(w=P + 4), b"16-byte")
    _refused(gemm(a=None), b"null")
    _refused(gemm(out=None), b"null")
    _refused(gemm(M=1 << 32), b"31 bits")
    assert gemm(M=0, a=None, w=None, out=None) == 0
    assert gemm(N=0, ldo=0, a=None, w=None, out=None) == 0
    need = lib.lsk_linear_mxfp4_workspace(17, 8, 64)
    assert need > 0
    _refused(lib.lsk_linear_mxfp4(P, L.LSK_F32, 64, 17, 64, P, P, 8, None, P, L.LSK_F32, 8, P, need - 1, None), b"workspace")
    _refused(lib.lsk_linear_mxfp4(P, L.LSK_F32, 64, 17, 64, P, P, 8, None, P, L.LSK_F32, 8, P + 16, need, None), b"workspace")
    _refused(lib.lsk_linear_mxfp4(P, L.LSK_I32, 64, 5, 64, P, P, 8, None, P, L.LSK_F32, 8, P, need, None), b"x_dtype")


def test_grouped_refusals():
    lib = L.load()

    def grouped(E=2, R=4, ldw=32, lds=2, N=8, K=64, ldo=8, offs=P, odt=L.LSK_BF16):
        need = lib.lsk_grouped_gemm_mxfp4_workspace(R, E, N, K)
        return lib.lsk_grouped_gemm_mxfp4(P, P, offs, E, R, P, ldw, P, lds, None, N, K, P, odt, ldo, P, need, None)
    _refused(grouped(E=0), b"E=0")
    _refused(grouped(ldw=24), b"strides")
    _refused(grouped(ldw=40), b"strides")
    _refused(grouped(lds=1), b"strides")
    _refused(grouped(offs=None), b"null")
    _refused(grouped(K=63), b"multiple of 32")
    _refused(grouped(odt=L.LSK_I32), b"out_dtype")
    assert grouped(R=0) == 0


def test_logits_refusals():
    lib = L.load()

    def pen(dtype=L.LSK_F32, B=2, V=100, ldl=100, ldo=100, Lp=0, Lo=0, logits=P, out=P):
        return lib.lsk_penalize_logits(logits, dtype, ldl, B, V, P, Lp, Lp, None, P, Lo, Lo, None, 0, None, None, None,
                                       None, 0, None, 0, out, ldo, None)
    _refused(pen(dtype=L.LSK_I32), b"dtype")
    _refused(pen(B=-1), b"bad sizes")
    _refused(pen(ldl=99), b"strides")
    _refused(pen(ldo=99), b"strides")
    _refused(pen(Lp=-1), b"history")
    _refused(pen(logits=None), b"null")
    assert pen(B=0, logits=None, out=None) == 0
    assert pen(V=0, ldl=0, ldo=0, logits=None, out=None) == 0


def test_cpu_tensors_are_refused():
    x, u = torch.zeros(2, 64), torch.zeros(2, 32, dtype=torch.uint8)
    s = torch.zeros(2, 2, dtype=torch.uint8)
    for call in (lambda: moe_mxfp4.quantize_mxfp4(x), lambda: moe_mxfp4.mm_mxfp4(u, s, u, s),
                 lambda: moe_mxfp4.linear_mxfp4(x, u, s), lambda: t16h_lmvariants.penalize_logits(x),
                 lambda: t16h_lmvariants.build("mxfp4").prepare(x)):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()
    with pytest.raises(ValueError):
        moe_ref.grouped_linear_mxfp4([], "w13", u, s, torch.zeros(3, dtype=torch.int32))


def test_head_variant_names():
    assert t16h_lmvariants.build(" mxfp4 ").kind == "mxfp4"
    assert t16h_lmvariants.build("mxfp4").gemms() == 0 and t16h_lmvariants.build("mxfp4").nbytes() == 0
    with pytest.raises(ValueError):
        t16h_lmvariants.build("mxfp6")


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where no launch can start")
def test_dequant_beyond_one_grid():
    """The quad kernel takes a launch of fewer than 2^32 threads (2^36 values); a larger tensor goes to the
    kernel that strides over its grid.  Without a GPU each says which one it tried to launch."""
    lib = L.load()
    for rows, kernel in ((1, b"dequant_mxfp4_4_kernel:"), ((1 << 30) - 64, b"dequant_mxfp4_4_kernel:"),
                         ((1 << 30), b"dequant_mxfp4_kernel:"), ((1 << 34), b"dequant_mxfp4_kernel:")):
        for odt in (L.LSK_BF16, L.LSK_F32):
            assert lib.lsk_dequant_mxfp4(P, P, rows, 64, 32, P, odt, None) == 2
            assert kernel in lib.lsk_last_error(), (rows, lib.lsk_last_error())


def test_grids_beyond_hip_are_refused():
    """HIP launches fewer than 2^32 threads along a grid: what would take more is refused before anything is
    launched."""
    lib = L.load()

    def pen(B, V):
        return lib.lsk_penalize_logits(P, L.LSK_F32, V, B, V, None, 0, 0, None, None, 0, 0, None, 0, None, None, None,
                                       None, 0, None, 0, P, V, None)
    _refused(pen(1 << 24, 1), b"grid too large")             # a block of 256 threads a row
    _refused(pen(1 << 22, 8192), b"grid too large")          # of 1024
    _refused(pen((1 << 31) - 1, 33), b"grid too large")
    for M, N in ((1, (1 << 31) - 1), (1 << 21, 1 << 21), ((1 << 29) - 1, 2000)):
        need = lib.lsk_gemm_mxfp4_workspace(M, N, 32)
        _refused(lib.lsk_gemm_mxfp4(P, P, M, 32, P, P, N, None, P, L.LSK_BF16, N, P, need, None), b"grid too large")
    need = lib.lsk_linear_mxfp4_workspace(1 << 28, 64, 128)  # 16 rows a block of the quantiser
    _refused(lib.lsk_linear_mxfp4(P, L.LSK_BF16, 128, 1 << 28, 128, P, P, 64, None, P, L.LSK_BF16, 64, P, need, None),
             b"grid too large")
    E = 1 << 20
    need = lib.lsk_grouped_gemm_mxfp4_workspace(E, E, 8192, 32)
    _refused(lib.lsk_grouped_gemm_mxfp4(P, P, P, E, E, P, 16, P, 1, None, 8192, 32, P, L.LSK_BF16, 8192, P, need, None),
             b"grid too large")


def test_logits_in_place_needs_one_stride():
    """In place with two row strides, a row's output lies in another row's input."""
    lib = L.load()

    def pen(B, ldl, ldo):
        return lib.lsk_penalize_logits(P, L.LSK_F32, ldl, B, 100, None, 0, 0, None, None, 0, 0, None, 0, None, None, None,
                                       None, 0, None, 0, P, ldo, None)
    _refused(pen(2, 128, 100), b"in place")
    _refused(pen(2, 100, 128), b"in place")
