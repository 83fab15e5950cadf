"""What the MXFP4 and logits operators are timed on: activations quantised to MXFP4 and multiplied with
MXFP4 weights (one linear, or one projection of every expert over rows sorted by expert), the
quantisation itself, and the penalties, biases and masks on a head's logits.

Kinds of case:
  quantize  moe_mxfp4.quantize_mxfp4, given back as the values it holds (moe_mxfp4.dequant_mxfp4)
  linear    moe_mxfp4.linear_mxfp4, rows in, the same type out
  grouped   moe_ref.grouped_linear_mxfp4 over rows quantised beforehand
  logits    t16h_lmvariants.penalize_logits

`own` chooses between the framework's operators and their plain form in elementary torch operations.
"""
from __future__ import annotations

import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 32


def _linear(M, N, K, bias, dtype="bf16"):
    return {"kind": "linear", "M": M, "N": N, "K": K, "bias": bias, "dtype": dtype}


def _grouped(R, E, H, I, which, bias):
    return {"kind": "grouped", "R": R, "E": E, "H": H, "I": I, "which": which, "bias": bias}


def _logits(B, V, prompt, output, dtype, bias, mask):
    return {"kind": "logits", "B": B, "V": V, "prompt": prompt, "output": output, "dtype": dtype, "bias": bias,
            "mask": mask}


def listed():
    named = {
        # the rows of a small decode batch on their way into an expert
        "quantize_rows_37": {"kind": "quantize", "M": 37, "K": 2880, "dtype": "f32"},
        # a whole gate/up weight brought to MXFP4 when a model is loaded
        "quantize_weight": {"kind": "quantize", "M": 28672, "K": 4096, "dtype": "bf16"},
        # one user's decode step: the QKV projection with its bias, all latency
        "linear_decode_1": _linear(1, 4608, 3584, True),
        # a serving batch on the down projection: long rows, few columns
        "linear_decode_24": _linear(24, 4096, 14336, False),
        # a busy server's decode batch: more rows than a stream of the weight wants, fewer than a prompt
        "linear_decode_200": _linear(200, 3584, 18944, False, "f16"),
        # a ragged prompt chunk through the QKV projection, binary32 in and out
        "linear_chunk_777": _linear(777, 4608, 3584, True, "f32"),
        # a prompt on the widest projection (the largest call)
        "linear_prefill_4096": _linear(4096, 28672, 4096, False),
        # one token's four experts
        "grouped_decode_4": _grouped(4, 32, 2880, 2880, "w13", True),
        # a decode batch's rows over all experts, few rows each
        "grouped_decode_256": _grouped(256, 32, 2880, 2880, "w2", True),
        # a prompt's rows over many small experts, unevenly
        "grouped_prefill_16384": _grouped(16384, 128, 2048, 768, "w13", False),
        # one user's logits after a short answer, with a bias for every token
        "logits_1": _logits(1, 65536, 300, 100, "f32", True, False),
        # a server's batch under a grammar, long prompts
        "logits_128": _logits(128, 152064, 2048, 700, "bf16", False, True),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    most = 2 * 4096 * 28672 * 4096 / 2    # half the largest listed case's flops
    kind = rng.choice(("quantize", "linear", "linear", "linear", "grouped", "grouped", "logits", "logits"))
    if kind == "quantize":
        return {"kind": kind, "M": _spread(rng, 1, 16384), "K": 32 * _spread(rng, 1, 224),
                "dtype": rng.choice(("bf16", "f32", "f16"))}
    if kind == "linear":
        M, N, K = _spread(rng, 1, 4096), _spread(rng, 17, 28672), 32 * _spread(rng, 1, 592)
        while 2 * M * N * K > most:
            M = max(1, M // 2)
        return _linear(M, N, K, rng.random() < 0.5, rng.choice(("bf16", "bf16", "f32", "f16")))
    if kind == "grouped":
        return _grouped(_spread(rng, 1, 16384), _spread(rng, 2, 128), 32 * _spread(rng, 4, 90), 32 * _spread(rng, 4, 48),
                        rng.choice(("w13", "w2")), rng.random() < 0.5)
    return _logits(_spread(rng, 1, 160), _spread(rng, 1000, 152064), _spread(rng, 1, 4096), _spread(rng, 1, 2048),
                   rng.choice(("f32", "bf16", "f16")), rng.random() < 0.5, rng.random() < 0.5)


# ---------------------------------------------------------------- inputs
def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _activations(g, M, K, dtype):
    """Hidden rows: N(0, 1) with one value in a thousand at +-20."""
    x = _normal(g, (M, K))
    far = torch.rand((M, K), generator=g, device="cuda") < 0.001
    return torch.where(far, 20.0 * torch.sign(x), x).to(dtype)


def _pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).contiguous()


def _weight(g, shape):
    """A normal weight of 1 / sqrt(K) as packed codes and scales."""
    code, scale = _codes(_normal(g, shape) / math.sqrt(shape[-1]))
    return _pack(code), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "quantize":
        return {"kind": kind, "x": _activations(g, case["M"], case["K"], DT[case["dtype"]])}
    if kind == "linear":
        w, ws = _weight(g, (case["N"], case["K"]))
        return {"kind": kind, "x": _activations(g, case["M"], case["K"], DT[case["dtype"]]), "w": w, "ws": ws,
                "bias": _normal(g, (case["N"],)) if case["bias"] else None}
    if kind == "grouped":
        return _prepare_grouped(case, g)
    B, V = case["B"], case["V"]
    s = {"kind": kind, "logits": (3.0 * _normal(g, (B, V))).to(DT[case["dtype"]])}
    for name in ("prompt", "output"):
        L = case[name]
        # text repeats itself: tokens by a falling law, rows of unequal length, padded with -1
        u = torch.rand((B, L), generator=g, device="cuda", dtype=torch.float64)
        tok = (V ** u - 1.0).long().clamp(0, V - 1)
        lens = torch.randint(L // 2, L + 1, (B,), generator=g, device="cuda")
        s[name] = torch.where(torch.arange(L, device="cuda") < lens[:, None], tok, -1)
        s[name + "_lens"] = lens
    rand = torch.rand((3, B), generator=g, device="cuda")
    s["repetition"], s["frequency"], s["presence"] = 1.0 + 0.5 * rand[0], 0.6 * rand[1], 0.6 * rand[2]
    s["bias"] = _normal(g, (V,)) if case["bias"] else None
    words = -(-V // 32)
    s["mask"] = (torch.randint(-2 ** 31, 2 ** 31, (B, words), generator=g, device="cuda").to(torch.int32)
                 if case["mask"] else None)
    return s


def _prepare_grouped(case, g):
    """Expert weights, their tables (which a program keeps with its weights), and expert-sorted rows."""
    R, E, H, I, which = case["R"], case["E"], case["H"], case["I"], case["which"]
    N, K = (2 * I, H) if which == "w13" else (H, I)
    w, ws = _weight(g, (E, N, K))
    bias = _normal(g, (E, N)) if case["bias"] else None
    # rows fall on experts with a skew of about five to one
    p = torch.exp(-1.6 * torch.rand((E,), generator=g, device="cuda"))
    expert = torch.multinomial(p, R, replacement=True, generator=g).sort().values
    offs = torch.searchsorted(expert, torch.arange(E + 1, device="cuda")).to(torch.int32)
    code, scale = _codes(_activations(g, R, K, torch.bfloat16))
    s = {"kind": "grouped", "which": which, "w": w, "ws": ws, "bias": bias, "a": _pack(code), "a_scale": scale,
         "offs": offs, "most": int((offs[1:] - offs[:-1]).max())}
    if own:
        from lockstep_amd import moe_ref
        # the layer's other projection is not called here: one of zeros stands in its place
        other = (H, I) if which == "w13" else (2 * I, H)
        z = (torch.zeros((other[0], other[1] // 2), dtype=torch.uint8, device="cuda"),
             torch.full((other[0], other[1] // BLOCK), 127, dtype=torch.uint8, device="cuda"))
        one = lambda e: (w[e], ws[e])  # noqa: E731
        bias_of = lambda e: None if bias is None else bias[e]  # noqa: E731
        s["tables"] = moe_ref.ExpertTablesMX(
            [(one(e), z, bias_of(e), None) if which == "w13" else (z, one(e), None, bias_of(e)) for e in range(E)],
            packed=True)
    return s


# ---------------------------------------------------------------- the plain form
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _codes(x):
    """x [..., K] -> (E2M1 codes [..., K], E8M0 bytes [..., K / 32]): the block's largest magnitude in
    [4, 8) of its scale, rounded to nearest with ties to the even code, above 6 to 6."""
    xb = x.float().unflatten(-1, (-1, BLOCK))
    top = xb.abs().amax(-1)
    e = torch.frexp(top).exponent - 3
    scale = torch.where(top > 0, e + 127, 0).clamp(0, 254)
    v = torch.ldexp(xb, 127 - scale.unsqueeze(-1))
    a = v.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code.to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    return code.flatten(-2), scale.to(torch.uint8)


def _unpack(packed):
    return torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)


def _values(code, scale, dtype=torch.float32):
    """The values that codes [..., K] and scales [..., K / 32] stand for."""
    tab = torch.tensor(E2M1, dtype=dtype, device=code.device)
    v = tab[code.long()].unflatten(-1, (-1, BLOCK))
    return (v * torch.exp2(scale.to(dtype) - 127.0).unsqueeze(-1)).flatten(-2)


def _padded(rows, offs, most):
    """Expert-sorted rows [R, K] at [E, most, K], and where each went."""
    E, R = offs.numel() - 1, rows.shape[0]
    p = torch.arange(R, device=rows.device)
    e = torch.searchsorted(offs[1:].long(), p, right=True)
    at = e * most + p - offs.long()[e]
    full = torch.zeros((E * most, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    full[at] = rows
    return full.unflatten(0, (E, most)), at, e


def _grouped_product(s, dtype):
    a = _values(_unpack(s["a"]), s["a_scale"], dtype)
    wt = _values(_unpack(s["w"]), s["ws"], dtype).transpose(1, 2).contiguous()
    full, at, e = _padded(a, s["offs"], s["most"])
    y = torch.bmm(full, wt).flatten(0, 1)[at]
    return y if s["bias"] is None else y + s["bias"].to(dtype)[e]


def _counts(tokens, lens, V, like):
    """How often each token below V stands in the first lens tokens of each row."""
    L = tokens.shape[1]
    ok = (torch.arange(L, device=tokens.device) < lens[:, None]) & (tokens >= 0) & (tokens < V)
    n = torch.zeros((tokens.shape[0], V), dtype=like, device=tokens.device)
    return n.scatter_add_(1, torch.where(ok, tokens, 0), ok.to(like))


def _penalized(s, dtype):
    l = s["logits"].to(dtype)
    V = l.shape[1]
    if s["bias"] is not None:
        l = l + s["bias"].to(dtype)
    n = _counts(s["output"], s["output_lens"], V, dtype)
    seen = (n > 0) | (_counts(s["prompt"], s["prompt_lens"], V, dtype) > 0)
    r, f, p = (s[k].to(dtype)[:, None] for k in ("repetition", "frequency", "presence"))
    l = torch.where(seen, torch.where(l > 0, l / r, l * r), l)
    l = l - f * n
    l = torch.where(n > 0, l - p, l)
    if s["mask"] is not None:
        v = torch.arange(V, device=l.device)
        l = torch.where(((s["mask"][:, v // 32] >> (v % 32)) & 1) != 0, l, -math.inf)
    return l


def run(state):
    s = state
    kind = s["kind"]
    if own:
        from lockstep_amd import moe_mxfp4, moe_ref, t16h_lmvariants
        if kind == "quantize":
            return moe_mxfp4.dequant_mxfp4(*moe_mxfp4.quantize_mxfp4(s["x"]))
        if kind == "linear":
            return moe_mxfp4.linear_mxfp4(s["x"], s["w"], s["ws"], s["bias"])
        if kind == "grouped":
            return moe_ref.grouped_linear_mxfp4(s["tables"], s["which"], s["a"], s["a_scale"], s["offs"])
        return t16h_lmvariants.penalize_logits(
            s["logits"], prompt=s["prompt"], prompt_lens=s["prompt_lens"], output=s["output"],
            output_lens=s["output_lens"], repetition=s["repetition"], frequency=s["frequency"],
            presence=s["presence"], bias=s["bias"], mask=s["mask"])
    if kind == "quantize":
        return _values(*_codes(s["x"])).to(torch.bfloat16)
    if kind == "linear":
        y = _values(*_codes(s["x"])) @ _values(_unpack(s["w"]), s["ws"]).t()
        return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)
    if kind == "grouped":
        return _grouped_product(s, torch.float32).to(torch.bfloat16)
    return _penalized(s, torch.float32).to(s["logits"].dtype)


# ---------------------------------------------------------------- 64 bits, from the definition
def _near(x):
    """x [..., K] in 64 bits rounded to what MXFP4 holds: of the signed E2M1 values times the block's
    power of two the nearest, of two as near the one with the even code."""
    xb = x.double().unflatten(-1, (-1, BLOCK))
    top = xb.abs().amax(-1, keepdim=True)
    step = torch.where(top > 0, torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -149))) - 2.0), 1.0)
    v = (xb / step).clamp(-6.0, 6.0)
    a = v.abs()
    # the spacing of E2M1 is 0.5 below 2, 1 below 4, 2 to 6; torch.round goes to the even multiple
    d = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).double()
    return (torch.round(v / d) * d * step).flatten(-2)


def _held(packed, scale):
    """The values of packed codes from their fields: sign, two bits of exponent, one of mantissa."""
    c = torch.stack((packed % 16, packed // 16), dim=-1).flatten(-2).double()
    sign = torch.where(c >= 8, -1.0, 1.0).double()
    c = c % 8
    ex, man = torch.floor(c / 2), c % 2
    mag = torch.where(ex == 0, man / 2, (1.0 + man / 2) * torch.exp2(ex - 1.0))
    return (sign * mag).unflatten(-1, (-1, BLOCK)).mul_(torch.exp2(scale.double() - 127.0).unsqueeze(-1)).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "quantize":
        return _near(s["x"])
    if kind == "linear":
        y = torch.matmul(_near(s["x"]), _held(s["w"], s["ws"]).t())
        return y if s["bias"] is None else y + s["bias"].double()
    if kind == "grouped":
        offs = s["offs"].tolist()
        y = torch.empty((case["R"], s["w"].shape[1]), dtype=torch.float64, device="cuda")
        for e in range(case["E"]):
            rows = slice(offs[e], offs[e + 1])
            y[rows] = _held(s["a"][rows], s["a_scale"][rows]) @ _held(s["w"][e], s["ws"][e]).t()
            if s["bias"] is not None:
                y[rows] += s["bias"][e].double()
        return y
    l = s["logits"].double()
    B, V = l.shape
    if s["bias"] is not None:
        l += s["bias"].double()
    hist = {}
    for name in ("prompt", "output"):
        L = s[name].shape[1]
        live = torch.arange(L, device="cuda")[None] < s[name + "_lens"][:, None]
        row = torch.arange(B, device="cuda")[:, None].expand(B, L)
        hist[name] = torch.bincount((row * V + s[name])[live], minlength=B * V).reshape(B, V)
    rep = s["repetition"].double()[:, None].expand(B, V)
    rep = torch.where(l > 0, 1.0 / rep, rep)
    l = torch.where(hist["prompt"] + hist["output"] > 0, l * rep, l)
    l -= s["frequency"].double()[:, None] * hist["output"]
    l -= s["presence"].double()[:, None] * (hist["output"] > 0)
    if s["mask"] is not None:
        bit = torch.arange(32, device="cuda")
        allowed = ((s["mask"].long()[..., None] >> bit) % 2).flatten(-2)[:, :V]
        l[allowed == 0] = -math.inf
    return l


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        n = case["M"] * case["K"]
        return {"bytes": n * (SIZE[case["dtype"]] + 2), "flops": 2 * n}
    if kind == "linear":
        M, N, K, size = case["M"], case["N"], case["K"], SIZE[case["dtype"]]
        return {"bytes": size * M * (K + N) + N * K * (1 / 2 + 1 / 32) + 4 * N * case["bias"], "flops": 2 * M * N * K}
    if kind == "grouped":
        R, E, H, I = case["R"], case["E"], case["H"], case["I"]
        N, K = (2 * I, H) if case["which"] == "w13" else (H, I)
        # experts that get a row, were all as likely
        live = E * (1.0 - (1.0 - 1.0 / E) ** R)
        return {"bytes": (R + live * N) * K * (1 / 2 + 1 / 32) + 2 * R * N + 4 * live * N * case["bias"],
                "flops": 2 * R * N * K}
    B, V, size = case["B"], case["V"], SIZE[case["dtype"]]
    hist = 0.75 * 8 * B * (case["prompt"] + case["output"])
    return {"bytes": 2 * size * B * V + hist + 4 * V * case["bias"] + B * V / 8 * case["mask"], "flops": 6 * B * V}
