"""Every launch a block-scaled fp8 product may take, at one, two, three and many stages of K, dense and by expert.

The sizes come from the rule itself (lsk_fp8_launch, a host function): for each launch and each K the cheapest M and N of a
grid that the rule sends there, so a change of the rule moves the sizes along.  What is computed: products whose every
partial sum is a binary32 number, against 64 bits bit for bit; and products over all of e4m3, bit for bit against the
same rows alone, which take other launches."""
import functools

import pytest
import torch

import test_fp8_gpu as T
from lockstep_amd import _lib as L

# a stage's values of K and how many stages are in flight, by launch
SPAN = [128] * 6 + [512, 256, 256, 512, 512, 256, 512]
RING = [2, 2, 2, 2, 4, 4, 4, 3, 2, 6, 4, 3, 4]
LAUNCHES = range(13)
OUT = {torch.bfloat16: L.LSK_BF16, torch.float16: L.LSK_F16, torch.float32: L.LSK_F32}


def _spread(lo, hi, n=60):
    return sorted({min(hi, max(lo, round(lo * (hi / lo) ** (i / (n - 1))))) for i in range(n)})


GRID = [(m, n) for m in _spread(1, 8192) for n in _spread(16, 16384)]


def _lengths(c):
    """K of 1, 2, 3, 2 RING + 1, 16 and 33 stages; all but the first end inside a stage and inside a block of 128."""
    return [(s, 16 if s == 1 else s * SPAN[c] - 48) for s in (1, 2, 3, 2 * RING[c] + 1, 16, 33)]


@functools.lru_cache(None)
def _cheapest(K, E, code):
    """{launch: (M, N)} of the grid at this K."""
    best, fn = {}, L.load().lsk_fp8_launch
    for M, N in GRID:
        c, cost = fn(M, N, K, E, code), M * N * K + 10 * (M + N * max(1, E)) * K
        if cost < best.get(c, (1 << 62,))[0]:
            best[c] = cost, (M, N)
    return {c: v for c, (_, v) in best.items()}


def _sizes(c, E, out_dtype):
    for stages, K in _lengths(c):
        if c in _cheapest(K, E, OUT[out_dtype]):
            yield (stages, *_cheapest(K, E, OUT[out_dtype])[c], K)


def _none(c, out_dtype):
    return c == 0 and out_dtype == torch.float32      # (products kept whole need more registers than it has)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_the_sizes_below_reach_every_launch_at_many_stages(out_dtype):
    for c in LAUNCHES:
        reached = {s for E in (0, 6, 40) for s, *_ in _sizes(c, E, out_dtype)}
        if _none(c, out_dtype):
            assert not reached
        else:
            assert max(reached) > 2 * RING[c] and len(reached) >= 2, (c, reached)
    # the ordinary tiles of prompts, dense, at every number of stages
    for c in (1, 2, 3) + ((0,) if out_dtype == torch.bfloat16 else ()):
        assert [s for s, *_ in _sizes(c, 0, out_dtype)] == [s for s, _ in _lengths(c)]


def test_the_frozen_sizes_reach_every_launch():
    """The sizes of test_fp8_gpu that stand for the launches still do."""
    fn = L.load().lsk_fp8_launch
    assert {fn(M, N, K, 0, L.LSK_BF16) for M, N, K in T.LAUNCHES} == set(LAUNCHES)
    grouped = next(m for m in T.test_grouped_exact_on_every_launch.pytestmark if m.name == "parametrize").args[1]
    assert {fn(R, N, K, E, L.LSK_BF16) for R, N, K, E in grouped} == set(LAUNCHES)


def test_the_query_itself():
    fn = L.load().lsk_fp8_launch
    for bad in ((0, 16, 16, 0), (1, 0, 16, 0), (1, 16, -1, 0), (1, 16, 1 << 22, 0), (1, 16, 16, -1), (1 << 31, 16, 16, 0)):
        assert fn(*bad, L.LSK_BF16) == -1
    assert fn(1, 16, 24, 0, L.LSK_BF16) == fn(1, 16, 16, 0, L.LSK_I8) == -1
    assert fn((1 << 31) - 1, (1 << 31) - 1, 16, 0, L.LSK_BF16) == -1
    assert fn(5, 16, 0, 0, L.LSK_BF16) in range(6) and fn(1, 1, 16, 1 << 20, L.LSK_F32) in LAUNCHES


# ---------------------------------------------------------------- on the GPU
def _table(device):
    import fp8_util as U
    return torch.from_numpy(U.E4M3).to(device)


def _exact_operand(g, rows, K, weight):
    """Codes of 0 and +-1, 1.5, 2, 3; scales 1 or 2 (of a weight 1 or 1/2).  A term is then a multiple of 2^-3 up to 18 and
    18 K < 2^21 for K < 116508: every partial sum is a binary32 number.  Eight products of one block lie within 2^6 of
    each other, far from what the fp8 instruction drops."""
    small = torch.tensor([0x00, 0x38, 0x3c, 0x40, 0x44, 0xb8, 0xbc, 0xc0, 0xc4], dtype=torch.uint8, device="cuda")
    code = small[torch.randint(0, 9, (rows, K), generator=g, device="cuda")]
    s = torch.randint(0, 2, ((rows + 127) // 128 if weight else rows, (K + 127) // 128), generator=g, device="cuda")
    return code, (1.0 + s) / (2.0 if weight else 1.0)


def _any_operand(g, rows, K, weight):
    """Codes over all of e4m3 but its NaNs, scales over an octave or two; results within f16's range."""
    code = torch.randint(0, 256, (rows, K), generator=g, device="cuda").to(torch.uint8)
    code = torch.where((code & 127) == 127, code ^ 2, code)
    s = torch.randn(((rows + 127) // 128 if weight else rows, (K + 127) // 128), generator=g, device="cuda")
    return code, torch.exp(0.5 * s) * 2.0 ** -7


def _values(code, scale, weight):
    """In 64 bits."""
    v = _table(code.device)[code.long()]
    s = scale.double().repeat_interleave(128, 1)[:, :code.shape[1]]
    return v * (s.repeat_interleave(128, 0)[:code.shape[0]] if weight else s)


def _f8(code):
    return code.view(torch.float8_e4m3fn)


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("launch", LAUNCHES)
def test_dense(launch, out_dtype):
    from lockstep_amd import lockstep_fullstack as FS
    fn = L.load().lsk_fp8_launch
    for stages, M, N, K in _sizes(launch, 0, out_dtype):
        print("dense", launch, stages, M, N, K, out_dtype, flush=True)
        assert fn(M, N, K, 0, OUT[out_dtype]) == launch
        g = torch.Generator(device="cuda").manual_seed(launch * 100 + stages)
        (a, sa), (w, sw) = _exact_operand(g, M, K, False), _exact_operand(g, N, K, True)
        y = (_values(a, sa, False) @ _values(w, sw, True).t().contiguous()).float()
        assert torch.equal(FS.mm_fp8(_f8(a), sa, _f8(w), sw, out_dtype=out_dtype), y.to(out_dtype))
        del y
        (a, sa), (w, sw) = _any_operand(g, M, K, False), _any_operand(g, N, K, True)
        sa = sa.t().contiguous().t()
        full = FS.mm_fp8(_f8(a), sa, _f8(w), sw, out_dtype=out_dtype)
        assert torch.isfinite(full).all()
        others = set()
        for m in (1, 16, 40, 130, 300):
            if m < M:
                others.add(fn(m, N, K, 0, OUT[out_dtype]))
                for at in (0, M - m):
                    few = FS.mm_fp8(_f8(a[at:at + m]), sa[at:at + m], _f8(w), sw, out_dtype=out_dtype)
                    assert torch.equal(few, full[at:at + m]), (m, at)
        for n in (16, 128, 640):       # (on the scales' blocks)
            if n < N:
                others.add(fn(M, n, K, 0, OUT[out_dtype]))
                assert torch.equal(FS.mm_fp8(_f8(a), sa, _f8(w[:n]), sw[:(n + 127) // 128], out_dtype=out_dtype), full[:, :n])
        assert others - {launch} or (M == 1 and N <= 16), (others, launch)


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E", [6, 40])
@pytest.mark.parametrize("launch", LAUNCHES)
def test_by_expert(launch, E, out_dtype):
    """Random counts, some experts empty, rows behind the last expert, which stay what they were."""
    from lockstep_amd import lockstep_fullstack as FS
    fn = L.load().lsk_fp8_launch
    for stages, R, N, K in _sizes(launch, E, out_dtype):
        print("by expert", launch, stages, R, N, K, E, out_dtype, flush=True)
        assert fn(R, N, K, E, OUT[out_dtype]) == launch
        g = torch.Generator(device="cuda").manual_seed(launch * 100 + stages + E)
        part = torch.rand(E, generator=g, device="cuda") * (torch.rand(E, generator=g, device="cuda") < 0.8) + 1e-6
        ends = (part.cumsum(0) / part.sum() * R * (0.95 if R > 20 else 1.0)).round().int()
        offs = torch.cat([ends.new_zeros(1), ends])
        at = offs.tolist()
        for operand in (_exact_operand, _any_operand):
            a, sa = operand(g, R, K, False)
            held = [operand(g, N, K, True) for _ in range(min(E, 7))]
            wp, sp = (torch.tensor([held[e % len(held)][j].data_ptr() for e in range(E)], device="cuda") for j in (0, 1))
            out = torch.full((R, N), 7.0, dtype=out_dtype, device="cuda")
            L.call("lsk_grouped_gemm_fp8", a.data_ptr(), sa.data_ptr(), sa.stride(0), sa.stride(1), offs.data_ptr(), E, R,
                   wp.data_ptr(), K, sp.data_ptr(), (K + 127) // 128, None, N, K, out.data_ptr(), OUT[out_dtype], N, L.stream_of(a))
            want = torch.full_like(out, 7.0)
            for e in range(E):
                rows, (w, sw) = slice(at[e], at[e + 1]), held[e % len(held)]
                if operand is _exact_operand:
                    want[rows] = (_values(a[rows], sa[rows], False) @ _values(w, sw, True).t().contiguous()).float().to(out_dtype)
                elif at[e] < at[e + 1]:
                    want[rows] = FS.mm_fp8(_f8(a[rows]), sa[rows], _f8(w), sw, out_dtype=out_dtype)
            assert torch.equal(out, want)


# N on both sides of each number of columns a block takes when it quantises its rows itself (16, 32, 64), and K of one, two,
# three, seven and more stages of that launch (of 512, 256 and 256 values)
FUSED = [(N, K) for N in (17, 4800, 4801, 25600, 25601, 40000) for K in (16, 464, 720, 1232, 1744, 3536, 8144, 16384)]


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", FUSED)
def test_rows_quantised_in_the_launch(N, K):
    from lockstep_amd import lockstep_fullstack as FS
    g = torch.Generator(device="cuda").manual_seed(N + K)
    w, sw = _any_operand(g, N, K, True)
    b = torch.randn(N, generator=g, device="cuda")
    wide = torch.randn((16, K + 8), generator=g, device="cuda")
    for M in (1, 2, 5, 16):
        if L.load().lsk_linear_fp8_workspace(M, N, K):
            continue
        print("quantised in the launch", M, N, K, flush=True)
        for dtype in OUT:
            for at in (0, 3):
                x = wide[:M, at:at + K].to(dtype) if at == 0 else wide.to(dtype)[:M, at:at + K]
                for odt in (torch.bfloat16, torch.float32):
                    want = FS.mm_fp8(*FS.quantize_rows_fp8(x), _f8(w), sw, b, odt)
                    assert torch.equal(FS.linear_fp8(x, _f8(w), sw, b, odt), want)


def test_rows_are_quantised_in_the_launch_at_those_sizes():
    fn = L.load().lsk_linear_fp8_workspace
    assert all(fn(1, N, K) == 0 for N, K in FUSED)
    assert [fn(16, N, 1232) > 0 for N in (4800, 4801)] == [True, True] and fn(16, 4800, 720) == fn(16, 40000, 720) == 0
