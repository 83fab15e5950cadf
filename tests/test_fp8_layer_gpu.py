"""The fp8 operators as a decoder layer runs them, one after the other: the residual norm into fp8 rows, a linear on
them, the choice of experts, both projections of every expert over rows sorted by expert, the weighted sum.  Against
the same in 64 bits with every rounding that is declared (h, the norm's fp8 rows, bf16 between the linears)."""
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


def _bf(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16).double().numpy()


def _layer(x, r, gain, gate, gbias, experts, tables, k, groups, keep):
    """x, r [T, H] bf16 -> (h, idx, w, y) with the framework's operators."""
    from lockstep_amd import lockstep_fullstack as FS, moe_ref, t16n_ref
    q, s, h, _ = t16n_ref.add_rmsnorm_fp8(x, r, gain, eps=1e-6)
    g = FS.mm_fp8(q, s, *gate)                                   # f32 logits
    idx, w = moe_ref.route_experts(g, k, "sigmoid", bias=gbias, groups=groups, keep_groups=keep, scale=2.5)
    T = x.shape[0]
    flat = idx.reshape(-1)
    order = flat.sort(stable=True).indices
    offs = torch.searchsorted(flat[order], torch.arange(tables.E + 1, device=x.device)).to(torch.int32)
    rows = order // k
    a = moe_ref.grouped_linear_fp8(tables, "w13", q.view(torch.uint8)[rows].view(q.dtype), s[rows], offs)
    act = moe_ref.act_silu(a[:, :tables.I].contiguous(), a[:, tables.I:].contiguous()).to(torch.bfloat16)
    b = moe_ref.grouped_linear_fp8(tables, "w2", *FS.quantize_rows_fp8(act), offs)
    y = torch.zeros((T, tables.H), device=x.device).index_add_(0, rows, b.float() * w.reshape(-1)[order, None])
    return h, g, idx, w, act, order, offs, y


@pytest.mark.parametrize("T,E,k,H,I,groups,keep", [(1, 8, 2, 256, 144, 1, 1), (7, 16, 4, 400, 192, 4, 2), (150, 32, 6, 512, 272, 8, 3)])
def test_a_layer(T, E, k, H, I, groups, keep):
    from lockstep_amd import lockstep_fullstack as FS, moe_ref
    say("layer", T, E, k, H, I)
    g = np.random.default_rng(T + E)
    x, r = (to_dev(g.standard_normal((T, H)).astype(np.float32)).to(torch.bfloat16) for _ in range(2))
    gain = to_dev((1 + 0.1 * g.standard_normal(H)).astype(np.float32))
    weight = lambda n, m: FS.quantize_weight_fp8(to_dev((g.standard_normal((n, m)) / np.sqrt(m)).astype(np.float32)))  # noqa: E731
    gate = weight(E, H)
    gbias = to_dev((0.05 * g.standard_normal(E)).astype(np.float32))
    experts = [(weight(2 * I, H), weight(H, I)) for _ in range(E)]
    tables = moe_ref.ExpertTablesFP8(experts)
    h, lg, idx, w, act, order, offs, y = _layer(x, r, gain, gate, gbias, experts, tables, k, groups, keep)

    host = lambda t: (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t).cpu().numpy()  # noqa: E731
    held = lambda p: U.values(host(p[0]), host(p[1]), True)  # noqa: E731
    # the norm: fp8 rows of 64-bit values may differ by a step of e4m3 (2^-3) where a value lies next to a border
    want_h = _bf(host(x.float()).astype(np.float64) + host(r.float()))
    assert np.array_equal(host(h.float()).astype(np.float64), want_h)
    n = want_h / np.sqrt((want_h ** 2).mean(1, keepdims=True) + 1e-6) * host(gain)
    q64 = U.values(*U.quantize(n.astype(np.float32)))
    logits = q64 @ held(gate).T
    off = np.linalg.norm(host(lg) - logits) / np.linalg.norm(logits)
    assert off < 1e-4, off           # few such steps: each moves a logit by 2^-3 of one of H terms
    i, v = U.route(host(lg), k, "sigmoid", host(gbias), groups, keep, 2, True, 2.5)
    assert np.array_equal(host(idx), i) and np.allclose(host(w), v, rtol=2.0 ** -23, atol=0)
    # the experts, from the rows as they are: bf16 after w13 and after the activation (2^-8 each at most, and the
    # activation's slope is at most 1.1), fp8 rows of it (2^-4), bf16 after w2
    y64 = np.zeros((T, H))
    a64 = np.zeros((T * k, I))
    o = host(order)
    for pos, slot in enumerate(o):
        t, e = slot // k, i[slot // k, slot % k]
        z = q64[t] @ held(experts[e][0]).T
        gt, up = z[:I], z[I:]
        a64[pos] = gt / (1 + np.exp(-gt)) * up
        y64[t] += v[t, slot % k] * (U.values(*U.quantize(a64[pos][None])) @ held(experts[e][1]).T)[0]
    got = host(act.float()).astype(np.float64)
    assert np.linalg.norm(got - a64) / np.linalg.norm(a64) < 3 * 2.0 ** -8
    # the fp8 rows of activations that far apart differ by up to a step, most not at all: 2^-4 bounds the 2-norm
    assert np.linalg.norm(host(y) - y64) / np.linalg.norm(y64) < 2.0 ** -4


def test_a_layer_in_a_graph():
    """Captured once and replayed on other rows: the same bits as eagerly."""
    from lockstep_amd import lockstep_fullstack as FS, moe_ref, t16n_ref
    g = torch.Generator(device="cuda").manual_seed(5)
    T, E, k, H, I = 24, 16, 4, 512, 256
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, r, gain = rnd(T, H).to(torch.bfloat16), rnd(T, H).to(torch.bfloat16), 1 + 0.1 * rnd(H)
    wq, wo = FS.quantize_weight_fp8(rnd(700, H) / 22), FS.quantize_weight_fp8(rnd(E, H) / 22)
    tables = moe_ref.ExpertTablesFP8([(FS.quantize_weight_fp8(rnd(2 * I, H) / 22), FS.quantize_weight_fp8(rnd(H, I) / 16))
                                      for _ in range(E)])
    offs = torch.arange(0, T * k + 1, T * k // E, device="cuda", dtype=torch.int32)

    def step():
        q, s, h, _ = t16n_ref.add_rmsnorm_fp8(x, r, gain, eps=1e-6)
        z = FS.mm_fp8(q, s, *wq, out_dtype=torch.bfloat16)
        l = FS.linear_fp8(x, *wo, out_dtype=torch.float32)
        idx, w = moe_ref.route_experts(l, k, groups=4, keep_groups=2)
        a = moe_ref.grouped_linear_fp8(tables, "w13", *FS.quantize_rows_fp8(h.repeat_interleave(k, 0)), offs)
        return h, z, l, idx, w, a
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(torch.roll(x, 3, 1))
        r.mul_(-1)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert np.array_equal(bits(a), bits(b))
