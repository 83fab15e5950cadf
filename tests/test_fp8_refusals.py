"""What the fp8, residual norm and routing entry points refuse, at the C boundary and in Python, without a GPU."""
import pytest
import torch

from lockstep_amd import _lib as L
from lockstep_amd import lockstep_fullstack as FS, moe_ref, t16n_ref

P = 1 << 20      # a plausible, 256-byte aligned address: every call here is refused before it is used


def _refused(rc, word):
    lib = L.load()
    assert rc == 1 and word in lib.lsk_last_error(), (rc, lib.lsk_last_error())


def test_quantiser_refusals():
    lib = L.load()

    def rows(x=P, dt=L.LSK_F32, M=2, K=64, ldx=64, q=P, s=P):
        return lib.lsk_quantize_rows_fp8(x, dt, M, K, ldx, q, s, 1, M, None)

    def weight(x=P, dt=L.LSK_F32, M=2, K=64, ldx=64, q=P, s=P):
        return lib.lsk_quantize_weight_fp8(x, dt, M, K, ldx, q, s, None)
    for f in (rows, weight):
        _refused(f(dt=L.LSK_I8), b"x_dtype")
        _refused(f(K=40), b"multiple of 16")
        _refused(f(M=-1), b"bad sizes")
        _refused(f(K=1 << 24, ldx=1 << 24), b"2^24")
        _refused(f(ldx=48), b"ldx")
        _refused(f(x=None), b"null")
        _refused(f(s=None), b"null")
        _refused(f(q=P + 8), b"aligned")
        _refused(f(M=1 << 38, K=65536, ldx=65536), b"grid too large")
        assert f(M=0, x=None, q=None, s=None) == 0
        assert f(K=0, ldx=0, x=None, q=None, s=None) == 0

    def deq(q=P, s=P, rows=1, M=2, K=64, out=P, odt=L.LSK_BF16):
        return lib.lsk_dequant_fp8(q, s, 1, 2, rows, M, K, out, odt, None)
    _refused(deq(odt=L.LSK_I32), b"out_dtype")
    _refused(deq(K=24), b"multiple of 16")
    _refused(deq(rows=64), b"128 rows")
    _refused(deq(out=P + 8), b"aligned")
    _refused(deq(q=None), b"null")
    assert deq(M=0, q=None, s=None, out=None) == 0


def test_product_refusals():
    lib = L.load()

    def gemm(M=4, K=64, N=8, odt=L.LSK_F32, ldo=8, a=P, w=P, out=P, sm=1, sb=4):
        return lib.lsk_gemm_fp8(a, P, sm, sb, M, K, w, P, N, None, out, odt, ldo, None)
    _refused(gemm(K=40), b"multiple of 16")
    _refused(gemm(M=-1), b"bad sizes")
    _refused(gemm(odt=L.LSK_I32), b"out_dtype")
    _refused(gemm(ldo=7), b"ldo")
    _refused(gemm(a=P + 8), b"16-byte")
    _refused(gemm(w=P + 4), b"16-byte")
    _refused(gemm(a=None), b"null")
    _refused(gemm(out=None), b"null")
    _refused(gemm(M=1 << 32), b"31 bits")
    _refused(gemm(K=1 << 22), b"2^22")
    _refused(gemm(sm=-1), b"scale strides")
    _refused(gemm(sb=-1), b"scale strides")
    _refused(gemm(M=100, sm=1 << 30), b"31-bit offsets")
    _refused(gemm(K=1280, sb=1 << 27), b"31-bit offsets")
    assert gemm(M=0, a=None, w=None, out=None) == 0
    assert gemm(N=0, ldo=0, a=None, w=None, out=None) == 0
    need = lib.lsk_linear_fp8_workspace(17, 8, 2048)
    assert need > 0
    lin = lambda x=P, dt=L.LSK_F32, ldx=2048, work=P, nbytes=need: lib.lsk_linear_fp8(x, dt, ldx, 17, 2048, P, P, 8, None, P, L.LSK_F32, 8, work, nbytes, None)  # noqa: E731,E501
    _refused(lin(nbytes=need - 1), b"workspace")
    _refused(lin(work=P + 16), b"workspace")
    _refused(lin(work=None), b"workspace")
    _refused(lin(dt=L.LSK_I32), b"x_dtype")
    _refused(lin(ldx=2047), b"ldx")


def test_grouped_refusals():
    lib = L.load()

    def grouped(E=2, R=4, ldw=64, lds=1, N=8, K=64, ldo=8, offs=P, odt=L.LSK_BF16, a=P):
        return lib.lsk_grouped_gemm_fp8(a, P, 1, R, offs, E, R, P, ldw, P, lds, None, N, K, P, odt, ldo, None)
    _refused(grouped(E=0), b"E=0")
    _refused(grouped(ldw=48), b"strides")
    _refused(grouped(ldw=72), b"strides")
    _refused(grouped(lds=0), b"strides")
    _refused(grouped(offs=None), b"null")
    _refused(grouped(a=P + 8), b"16-byte")
    _refused(grouped(K=56, ldw=64), b"multiple of 16")
    _refused(grouped(odt=L.LSK_I32), b"out_dtype")
    assert grouped(R=0) == 0


def test_products_beyond_a_grid_are_refused():
    lib = L.load()
    most = 2 ** 31 - 1
    for odt in (L.LSK_F32, L.LSK_BF16):
        for K in (0, 16, 4096):
            _refused(lib.lsk_gemm_fp8(P, P, 1, 1, most, K, P, P, most, None, P, odt, most, None), b"grid too large")
            _refused(lib.lsk_grouped_gemm_fp8(P, P, 1, 1, P, 8, most, P, K, P, (K + 127) // 128, None, most, K, P, odt, most, None),
                     b"grid too large")


def test_norm_refusals():
    lib = L.load()

    def norm(x=P, dt=L.LSK_BF16, ldx=64, r=P, ldr=64, R=4, N=64, gdt=L.LSK_F32, h=P, ldh=64, q=P, s=P, out=None):
        return lib.lsk_add_rmsnorm_fp8(x, dt, ldx, r, ldr, R, N, P, gdt, 8.0, 1e-6, h, ldh, q, s, 1, R, out, None)
    _refused(norm(dt=L.LSK_I8), b"x_dtype")
    _refused(norm(gdt=L.LSK_I8), b"gain")
    _refused(norm(N=72, ldx=72, ldr=72, ldh=72), b"multiple of 16")
    _refused(norm(N=65552, ldx=65552, ldr=65552, ldh=65552), b"65536")
    _refused(norm(ldx=63), b"leading dimension")
    _refused(norm(ldr=63), b"leading dimension")
    _refused(norm(ldh=63), b"leading dimension")
    _refused(norm(x=None), b"null")
    _refused(norm(q=None), b"null")
    _refused(norm(q=P + 8), b"aligned")
    _refused(norm(out=P + 8), b"aligned")
    _refused(norm(h=P + 8), b"aligned")
    _refused(norm(ldh=68), b"aligned")
    _refused(norm(R=1 << 31), b"grid too large")
    assert norm(R=0, x=None) == 0


def test_route_refusals():
    lib = L.load()

    def route(g=P, dt=L.LSK_F32, ldg=64, T=4, E=64, k=8, groups=1, keep=1, top=1, wdt=L.LSK_F32, idx=P):
        return lib.lsk_route_experts(g, dt, ldg, T, E, k, 0, None, groups, keep, top, 1, 1.0, idx, P, wdt, None)
    _refused(route(dt=L.LSK_I8), b"logits")
    _refused(route(wdt=L.LSK_I8), b"weights")
    _refused(route(E=0), b"E in")
    _refused(route(E=1025), b"E in")
    _refused(route(T=-1), b"T=-1")
    _refused(route(k=0), b"k=0")
    _refused(route(k=65, E=128, ldg=128), b"k=65")
    _refused(route(k=17, groups=8, keep=2, top=2), b"k=17")
    _refused(route(groups=7), b"groups")
    _refused(route(groups=4, keep=5), b"groups")
    _refused(route(groups=4, keep=0), b"groups")
    _refused(route(E=128, ldg=128, groups=128, keep=8), b"groups")
    _refused(route(groups=4, keep=2, top=3), b"counts")
    _refused(route(groups=64, keep=8, top=2), b"counts")
    _refused(route(g=None), b"null")
    _refused(route(idx=None), b"null")
    _refused(route(ldg=63), b"ldg")
    _refused(route(T=1 << 39), b"grid too large")
    assert route(T=0, g=None) == 0


def test_cpu_tensors_and_wrong_operands_are_refused():
    x, q = torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.zeros(2, 1)
    for call in (lambda: FS.quantize_rows_fp8(x), lambda: FS.quantize_weight_fp8(x), lambda: FS.dequant_fp8(q, s),
                 lambda: FS.mm_fp8(q, s, q, s[:1]), lambda: FS.linear_fp8(x, q, s[:1]), lambda: t16n_ref.add_rmsnorm_fp8(x, x, x[0]),
                 lambda: moe_ref.route_experts(x, 2), lambda: moe_ref.ExpertTablesFP8([((q, s), (q, s))])):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()
    with pytest.raises(TypeError):
        moe_ref.grouped_linear_fp8([], "w13", q, s, torch.zeros(3, dtype=torch.int32))
