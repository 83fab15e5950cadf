"""t16h_lmvariants.penalize_logits against its declared steps, each one binary32 operation, bit for
bit (fp4_util.penalize)."""
import numpy as np
import pytest
import torch

import fp4_util as U
from gpu_util import bits, dev, say, to_dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import lockstep_amd._lib as L
    L.load()


def _case(g, B, V, Lp, Lo, dtype, tok=np.int64):
    l = torch.from_numpy((3 * g.standard_normal((B, V))).astype(np.float32)).to(dtype)
    p = g.integers(-2, V + 3, (B, Lp)).astype(tok)
    o = np.minimum(g.geometric(0.02, (B, Lo)), V + 1).astype(tok) - 1
    c = dict(prompt=p, prompt_lens=g.integers(0, Lp + 1, B).astype(np.int32), output=o,
             output_lens=g.integers(-1, Lo + 3, B).astype(np.int64), repetition=g.uniform(0.7, 1.6, B).astype(np.float32),
             frequency=g.uniform(-0.5, 0.9, B).astype(np.float32), presence=g.uniform(-0.5, 0.9, B).astype(np.float32),
             bias=g.standard_normal(V).astype(np.float32),
             mask=g.integers(-2 ** 31, 2 ** 31, (B, (V + 31) // 32)).astype(np.int32))
    return l, c


def _run(l, c, **kw):
    from lockstep_amd import t16h_lmvariants as TH
    return TH.penalize_logits(l.to(dev()), **{k: to_dev(v) for k, v in c.items()}, **kw)


def _check(l, c):
    want = torch.from_numpy(U.penalize(l.float().numpy(), **c)).to(l.dtype)
    assert np.array_equal(bits(_run(l, c)), bits(want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,V,Lp,Lo", [(1, 1, 1, 1), (1, 65536, 300, 100), (3, 1000, 40, 60), (2, 33, 5, 700),
                                       (5, 16391, 1, 257), (17, 8193, 90, 30), (300, 77, 10, 10), (2, 152064, 2000, 900)])
def test_all_steps(B, V, Lp, Lo, dtype):
    say("logits", B, V, Lp, Lo, dtype)
    l, c = _case(np.random.default_rng(B + V), B, V, Lp, Lo, dtype, np.int32 if V % 2 else np.int64)
    _check(l, c)


@pytest.mark.parametrize("left", [(), ("prompt", "prompt_lens"), ("output", "output_lens"), ("mask",), ("bias",),
                                  ("repetition",), ("frequency", "presence"), ("prompt_lens", "output_lens"),
                                  ("prompt", "prompt_lens", "output", "output_lens")])
def test_each_part_may_be_left_out(left):
    l, c = _case(np.random.default_rng(7), 4, 5003, 60, 50, torch.bfloat16)
    _check(l, {k: v for k, v in c.items() if k not in left})
    _check(l, {k: v for k, v in c.items() if k in left and k.replace("_lens", "") in left})   # (lengths need tokens)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_histories(dtype):
    """Counts of 2^15 and more, and one token over the whole of a long output."""
    g = np.random.default_rng(11)
    for Lo in (32767, 32768, 70000):
        l, c = _case(g, 2, 40003, 3, Lo, dtype)
        c["output"][0] = 40002
        c["output_lens"][0], c["prompt"][0], c["prompt_lens"][0] = Lo, 40002, 1
        _check(l, c)


def test_many_rows():
    l, c = _case(np.random.default_rng(12), 1500, 2100, 5, 9, torch.bfloat16)
    _check(l, c)


def test_special_values():
    """Infinite and NaN logits, also in masked and penalised places, and a row whose mask allows nothing."""
    g = np.random.default_rng(8)
    l, c = _case(g, 4, 3000, 500, 400, torch.float32)
    flat = l.view(-1)
    for i, v in enumerate((float("inf"), float("-inf"), float("nan"), 0.0, -0.0, torch.finfo(torch.float32).min)):
        flat[torch.from_numpy(g.integers(0, flat.numel(), 300))] = v
    c["mask"][2] = 0
    c["mask"][3] = -1
    c["bias"][::7] = -np.inf
    got = _run(l, c).cpu().numpy()
    want = U.penalize(l.numpy(), **c)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(got)].view(np.uint32), want[~np.isnan(want)].view(np.uint32))
    assert np.isneginf(got[2]).all()


def test_layouts_and_in_place():
    from lockstep_amd import t16h_lmvariants as TH
    g = np.random.default_rng(9)
    B, V = 5, 2050
    l, c = _case(g, B, V, 64, 64, torch.bfloat16)
    want = bits(torch.from_numpy(U.penalize(l.float().numpy(), **c)).to(l.dtype))
    d = {k: to_dev(v) for k, v in c.items()}
    for off in (0, 1, 3, 8):
        wide = torch.zeros((B, V + 11), dtype=l.dtype, device=dev())
        wide[:, off:off + V] = l.to(dev())
        view = wide[:, off:off + V]
        assert np.array_equal(bits(TH.penalize_logits(view, **d)), want)
        guard = wide.clone()
        out = guard[:, off:off + V]
        assert TH.penalize_logits(out, **d, out=out) is out
        assert np.array_equal(bits(out), want)
        assert torch.equal(guard[:, :off], wide[:, :off]) and torch.equal(guard[:, off + V:], wide[:, off + V:])
    assert np.array_equal(bits(TH.penalize_logits(l.to(dev()).t().contiguous().t(), **d)), want)
    assert np.array_equal(bits(TH.penalize_logits(l.to(dev()), **{**d, "bias": d["bias"].expand(B, V)})), want)
    many = to_dev(g.standard_normal((B, V)).astype(np.float32))
    one = torch.from_numpy(U.penalize(l.float().numpy(), **{**c, "bias": many.cpu().numpy(), "mask": c["mask"][1:2].repeat(B, 0)}))
    got = TH.penalize_logits(l.to(dev()), **{**d, "bias": many, "mask": d["mask"][1:2]})
    assert np.array_equal(bits(got), bits(one.to(l.dtype)))
    got = TH.penalize_logits(l.to(dev()), **{**d, "prompt": d["prompt"].t().contiguous().t(), "mask": d["mask"].expand(B, -1)})
    assert np.array_equal(bits(got), want)
    assert TH.penalize_logits(torch.zeros((0, V), device=dev())).shape == (0, V)
    assert TH.penalize_logits(torch.zeros((B, 0), device=dev())).shape == (B, 0)
    z = torch.zeros((B, 0), dtype=torch.int64, device=dev())
    assert np.array_equal(bits(TH.penalize_logits(l.to(dev()), prompt=z, output=z)), bits(l))


def test_bad_arguments():
    from lockstep_amd import t16h_lmvariants as TH
    l, c = _case(np.random.default_rng(10), 3, 100, 8, 8, torch.float32)
    d = {k: to_dev(v) for k, v in c.items()}
    l = l.to(dev())
    bad = [dict(prompt=d["prompt"].float()), dict(prompt=d["prompt"][:2]), dict(prompt_lens=d["prompt_lens"]),
           dict(output=d["output"], output_lens=d["output_lens"].float()), dict(repetition=d["repetition"][:2]),
           dict(frequency=d["frequency"].double()), dict(bias=d["bias"][:99]), dict(mask=d["mask"][:, :3]),
           dict(mask=d["mask"].to(torch.int64)), dict(out=torch.empty((3, 101), device=dev())),
           dict(out=l.to(torch.bfloat16)), dict(out=l[:1].expand(3, 100)), dict(presence=d["presence"].cpu())]
    for kw in bad:
        with pytest.raises(ValueError):
            TH.penalize_logits(l, **kw)
    with pytest.raises(ValueError):
        TH.penalize_logits(l[0])
    with pytest.raises(ValueError):
        TH.penalize_logits(l.to(torch.int32))


@pytest.mark.parametrize("Lo", [6, 32768])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_untouched_tokens_keep_their_bits(dtype, Lo):
    """Without bias and mask a token outside the history keeps its bits, a NaN's payload too, whatever the
    row's alignment and its neighbours (every 16-bit pattern; binary32 ones of every exponent)."""
    from lockstep_amd import t16h_lmvariants as TH
    g = np.random.default_rng(21)
    B, V = 3, 65536 + 11
    raw = np.arange(B * V, dtype=np.uint32)
    if dtype == torch.float32:
        raw = ((raw << 16) ^ g.integers(0, 1 << 16, raw.size, dtype=np.uint32)).view(np.int32)
    else:
        raw = raw.astype(np.uint16).view(np.int16)
    l = torch.from_numpy(raw).view(dtype).view(B, V)
    out_tok = g.integers(0, V, (B, Lo))
    out_tok[:, :6] = np.array([0x7f81, 0x7fff, 0xffc1, 0x7c01, 0xfe00, V - 1]) + np.arange(B)[:, None]   # (some past V)
    kw = dict(output=out_tok, output_lens=np.full(B, 6), repetition=np.full(B, 1.25, np.float32),
              presence=np.full(B, 0.5, np.float32))
    seen = U.counts(out_tok, kw["output_lens"], V) > 0
    with np.errstate(invalid="ignore"):
        want = torch.from_numpy(U.penalize(l.float().numpy(), **kw)).to(dtype)
    d = {k: to_dev(v) for k, v in kw.items()}
    for off, to in ((0, 0), (1, 1), (5, 5), (0, 1), (3, 0)):
        wide, out = (torch.zeros((B, V + 8), dtype=dtype, device=dev()) for _ in range(2))
        wide[:, off:off + V].copy_(l)
        assert np.array_equal(bits(wide[:, off:off + V]), bits(l))      # (the copy there kept them)
        got = TH.penalize_logits(wide[:, off:off + V], **d, out=out[:, to:to + V])
        assert np.array_equal(bits(got)[~seen], bits(l)[~seen]), (off, to)
        nan = want.isnan().numpy()
        assert np.array_equal(got.isnan().cpu().numpy(), nan) and np.array_equal(bits(got)[~nan], bits(want)[~nan])
        if off == to:
            TH.penalize_logits(wide[:, off:off + V], **d, out=wide[:, off:off + V])
            assert np.array_equal(bits(wide[:, off:off + V]), bits(got)), off


def test_a_frequency_of_infinity_or_nan_reaches_counted_tokens_only():
    """The frequency step, as the presence step, is for tokens that stand in the output: the others keep
    their logits (and a zero its sign) under any frequency."""
    g = np.random.default_rng(22)
    l, c = _case(g, 4, 3000, 50, 40, torch.float32)
    c["frequency"] = np.array([np.inf, -np.inf, np.nan, -0.5], np.float32)
    l[:, ::5] = -0.0
    for left in ((), ("bias", "mask")):
        kw = {k: v for k, v in c.items() if k not in left}
        got, want = _run(l, kw).cpu().numpy(), U.penalize(l.numpy(), **kw)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[~np.isnan(got)].view(np.uint32), want[~np.isnan(want)].view(np.uint32))
        no = U.counts(kw["output"], kw["output_lens"], 3000) == 0
        assert not np.isnan(got[no]).any()
