"""moe_ref.route_experts against a plain 64-bit statement (fp8_util.route): the same experts in the same order, the
weights within half a step of their type (and what two 64-bit exponentials may differ by)."""
import numpy as np
import pytest
import torch

import fp8_util as U
from gpu_util import dev, say, to_dev

pytestmark = pytest.mark.gpu

STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8 + 2.0 ** -24, torch.float16: 2.0 ** -11 + 2.0 ** -24}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import lockstep_amd._lib as L
    L.load()


def _compare(g, k, scoring="softmax", bias=None, groups=1, keep_groups=None, group_top=2, renormalize=True, scale=1.0,
             out_dtype=torch.float32):
    from lockstep_amd import moe_ref
    idx, w = moe_ref.route_experts(g.to(dev()), k, scoring, bias=None if bias is None else to_dev(bias), groups=groups,
                                   keep_groups=keep_groups, group_top=group_top, renormalize=renormalize, scale=scale,
                                   out_dtype=out_dtype)
    assert idx.dtype == torch.int64 and w.dtype == out_dtype
    i, v = U.route(g.double().numpy(), k, scoring, bias, groups, keep_groups, group_top, renormalize, scale)
    assert np.array_equal(idx.cpu().numpy(), i)
    got = w.double().cpu().numpy()
    nan = np.isnan(v)
    assert np.array_equal(np.isnan(got), nan)
    tiny = float(torch.finfo(out_dtype).smallest_normal) * STEP[out_dtype]      # (half a subnormal step)
    assert (np.abs(got - v)[~nan] <= (STEP[out_dtype] * (1 + 1e-6) * np.abs(v) + tiny + 1e-46)[~nan]).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 8), (3, 7, 2), (37, 64, 6), (5, 65, 1), (50, 128, 8), (9, 100, 64), (33, 256, 8),
                                   (4, 500, 10), (6, 1024, 16), (700, 160, 6)])
def test_route(T, E, k, scoring):
    say("route", T, E, k, scoring)
    g = np.random.default_rng(T + E)
    l = torch.from_numpy((2 * g.standard_normal((T, E))).astype(np.float32))
    bias = (0.1 * g.standard_normal(E)).astype(np.float32)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for b in (None, bias):
            for renorm in (True, False):
                _compare(l.to(dtype), k, scoring, b, renormalize=renorm, scale=2.5 if renorm else 1.0)
    _compare(l, k, scoring, bias, out_dtype=torch.bfloat16)
    _compare(l, k, scoring, None, out_dtype=torch.float16)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,groups,keep,top", [(5, 16, 2, 4, 2, 2), (40, 64, 6, 8, 3, 1), (30, 256, 8, 8, 4, 2), (7, 60, 20, 3, 2, 2),
                                                   (6, 1024, 8, 64, 5, 2), (9, 64, 4, 64, 4, 1), (20, 100, 5, 5, 5, 2),
                                                   (300, 160, 6, 8, 3, 1), (3, 384, 64, 2, 1, 2)])
def test_groups(T, E, k, groups, keep, top, scoring):
    say("groups", T, E, k, groups, keep, top)
    g = np.random.default_rng(T + E + k)
    l = torch.from_numpy((2 * g.standard_normal((T, E))).astype(np.float32))
    bias = (0.2 * g.standard_normal(E)).astype(np.float32)
    for b in (None, bias):
        _compare(l, k, scoring, b, groups, keep, top)
        _compare(l.to(torch.bfloat16), k, scoring, b, groups, keep, top)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_ties_go_to_the_lower_index(scoring):
    g = np.random.default_rng(1)
    l = torch.from_numpy(g.integers(0, 3, (60, 96)).astype(np.float32))
    flat = np.zeros(96, np.float32)
    for b in (None, flat, (0.5 * g.integers(0, 2, 96)).astype(np.float32)):
        _compare(l, 12, scoring, b)
        _compare(l, 12, scoring, b, 6, 3, 2)
        _compare(l, 5, scoring, b, 48, 7, 1)
    _compare(torch.zeros((4, 200)), 9, scoring)
    _compare(torch.zeros((4, 200)), 9, scoring, None, 4, 2, 2)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_scores_that_binary32_does_not_tell_apart(scoring):
    """Logits and biases a few binary32 units apart, whose scores round to the same binary32 number."""
    g = np.random.default_rng(2)
    T, E = 200, 128
    l = (1.0 + g.integers(0, 6, (T, E)) * 2.0 ** -23).astype(np.float32)
    bias = (0.25 + g.integers(0, 6, E) * 2.0 ** -25).astype(np.float32)
    for b in (None, bias):
        _compare(torch.from_numpy(l), 8, scoring, b)
        _compare(torch.from_numpy(l), 8, scoring, b, 8, 4, 2)
        _compare(torch.from_numpy(l), 6, scoring, b, 8, 2, 1)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_infinities_nans_and_rows_without_an_expert(scoring):
    g = np.random.default_rng(3)
    E = 48
    l = g.standard_normal((9, E)).astype(np.float32)
    l[0] = -np.inf
    l[1, 5:] = -np.inf
    l[2, 3] = np.nan
    l[3] = np.nan
    l[4, 7] = np.inf
    l[5, [1, 40]] = np.inf
    l[6] = np.finfo(np.float32).min
    l[7, ::2] = np.finfo(np.float32).min
    l[8, 0] = 3e38
    bias = (0.1 * g.standard_normal(E)).astype(np.float32)
    banned = bias.copy()
    banned[10:] = -np.inf
    both = bias.copy()
    both[[0, 9, 17]], both[[1, 2, 16, 18]] = np.inf, -np.inf
    for b in (None, bias, banned, both):
        for renorm in (True, False):
            _compare(torch.from_numpy(l), 8, scoring, b, renormalize=renorm)
        _compare(torch.from_numpy(l), 8, scoring, b, 6, 2, 2)
        _compare(torch.from_numpy(l), 8, scoring, b, 6, 2, 1)


def test_strides_stream_graph_and_empty():
    from lockstep_amd import moe_ref
    g = np.random.default_rng(4)
    big = to_dev(g.standard_normal((30, 200)).astype(np.float32))
    want = moe_ref.route_experts(big[:, 3:131].contiguous(), 8, "sigmoid")
    for view in (big[:, 3:131], big[:, 3:131].t().contiguous().t()):
        got = moe_ref.route_experts(view, 8, "sigmoid")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    some = moe_ref.route_experts(big[::3, 3:131], 8, "sigmoid")
    assert torch.equal(some[0], want[0][::3]) and torch.equal(some[1], want[1][::3])
    idx, w = moe_ref.route_experts(big[:0], 4)
    assert idx.shape == w.shape == (0, 4)
    l = big[:, :128].contiguous()
    graph = torch.cuda.CUDAGraph()
    moe_ref.route_experts(l, 6, "softmax", groups=4, keep_groups=2)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = moe_ref.route_experts(l, 6, "softmax", groups=4, keep_groups=2)
    for i in range(4):
        l.copy_(torch.roll(l, i + 1, 1))
        graph.replay()
        eager = moe_ref.route_experts(l, 6, "softmax", groups=4, keep_groups=2)
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def test_into_a_layer():
    """(idx, w) as moe_forward takes them: the same layer as with the same routing made by hand."""
    from lockstep_amd import contract_common as CC, moe_ref, workloads as WL
    T, E, k, H, I = 24, 8, 2, 256, 128
    x, experts, logits = WL.moe_inputs(T, E, k, H, I, seed=3)
    ex = [(to_dev(w13).t(), to_dev(ws13), to_dev(w2).t(), to_dev(ws2)) for (w13, ws13, w2, ws2, _, _) in experts]
    xd = to_dev(x).to(torch.bfloat16)
    l = to_dev(np.asarray(logits, np.float32))
    idx, w = moe_ref.route_experts(l, k, "sigmoid", out_dtype=torch.bfloat16)
    run = lambda r: moe_ref.moe_forward(xd, None, ex, k, True, CC.table_on(dev()), 0, moe_ref.act_silu, routing=r)[0]  # noqa: E731
    p = torch.sigmoid(l.double().cpu())
    v, i = p.sort(dim=-1, descending=True, stable=True)
    by_hand = (v[:, :k] / v[:, :k].sum(-1, keepdim=True)).float().to(torch.bfloat16).to(dev())
    assert torch.equal(idx.cpu(), i[:, :k]) and torch.equal(w, by_hand)
    assert torch.equal(run((idx, w)), run((i[:, :k].to(dev()), by_hand)))
