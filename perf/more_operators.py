"""What the fp8 and routing operators are timed on: rows and weights in 8-bit floating point (e4m3) with a
binary32 scale for each block of 128 values, the norm that feeds them, the linears that multiply them
(dense, and one projection of every expert over rows sorted by expert), and the choice of experts.

Kinds of case:
  quantize  lockstep_fullstack.quantize_rows_fp8 (a scale for 128 values of a row) or quantize_weight_fp8
            (for 128 x 128), given back as the values they hold (dequant_fp8)
  norm      t16n_ref.add_rmsnorm_fp8: the residual's addition, the norm and its fp8 rows
  linear    lockstep_fullstack.linear_fp8, rows in, the same type out
  grouped   moe_ref.grouped_linear_fp8 over rows quantised beforehand
  route     moe_ref.route_experts on a gate's logits

`own` chooses between the framework's operators and their plain form in elementary torch operations.
"""
from __future__ import annotations

import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 128
F8 = torch.float8_e4m3fn


def _quantize(M, K, weight, dtype="bf16"):
    return {"kind": "quantize", "M": M, "K": K, "weight": weight, "dtype": dtype}


def _norm(M, K, dtype="bf16"):
    return {"kind": "norm", "M": M, "K": K, "dtype": dtype}


def _linear(M, N, K, bias, dtype="bf16"):
    return {"kind": "linear", "M": M, "N": N, "K": K, "bias": bias, "dtype": dtype}


def _grouped(R, E, H, I, which, bias, by_block):
    return {"kind": "grouped", "R": R, "E": E, "H": H, "I": I, "which": which, "bias": bias, "by_block": by_block}


def _route(T, E, k, scoring, bias, groups, keep, dtype="f32"):
    return {"kind": "route", "T": T, "E": E, "k": k, "scoring": scoring, "bias": bias, "groups": groups, "keep": keep,
            "dtype": dtype}


def listed():
    named = {
        # the hidden rows of a small decode batch on their way into an expert
        "quantize_rows_37": _quantize(37, 2880, False, "f32"),
        # a whole gate/up weight brought to fp8 when a model is loaded
        "quantize_weight": _quantize(28672, 4096, True),
        # one user's decode step between two linears, all latency
        "norm_decode_1": _norm(1, 3584),
        # a long prompt's hidden rows before a gate/up projection
        "norm_prefill_8192": _norm(8192, 4096),
        # one user's decode step: the QKV projection with its bias, all latency
        "linear_decode_1": _linear(1, 4608, 3584, True),
        # a serving batch on the down projection: long rows, few columns
        "linear_decode_32": _linear(32, 4096, 14336, False),
        # a ragged prompt chunk through another model's down projection
        "linear_chunk_500": _linear(500, 3584, 18944, False, "f16"),
        # a prompt on the widest projection (the largest call)
        "linear_prefill_4096": _linear(4096, 28672, 4096, False),
        # a decode batch's rows over all experts, few rows each, K that ends inside a block, scales by row
        "grouped_decode_128": _grouped(128, 32, 2880, 2880, "w2", True, False),
        # a prompt's rows over many small experts, unevenly, scales as the quantiser lays them
        "grouped_prefill_32768": _grouped(32768, 128, 2048, 768, "w13", False, True),
        # a decode batch's choice among 128 experts
        "route_decode_32": _route(32, 128, 8, "softmax", False, 1, 1, "bf16"),
        # a prompt's choice with a balancing bias, half of eight groups kept
        "route_prefill_8192": _route(8192, 256, 8, "sigmoid", True, 8, 4),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    most = 2 * 4096 * 28672 * 4096 / 4    # a quarter of the largest listed case's flops
    kind = rng.choice(("quantize", "norm", "linear", "linear", "linear", "grouped", "grouped", "route"))
    dtype = rng.choice(("bf16", "bf16", "f32", "f16"))
    if kind == "quantize":
        return _quantize(_spread(rng, 1, 16384), 16 * _spread(rng, 1, 448), rng.random() < 0.5, dtype)
    if kind == "norm":
        return _norm(_spread(rng, 1, 8192), 16 * _spread(rng, 1, 448), dtype)
    if kind == "linear":
        M, N, K = _spread(rng, 1, 4096), _spread(rng, 17, 28672), 16 * _spread(rng, 1, 1184)
        while 2 * M * N * K > most:
            M = max(1, M // 2)
        return _linear(M, N, K, rng.random() < 0.5, dtype)
    if kind == "grouped":
        R, E, H, I = _spread(rng, 1, 32768), _spread(rng, 2, 128), 16 * _spread(rng, 8, 180), 16 * _spread(rng, 8, 96)
        while 4 * R * H * I > most:
            R = max(1, R // 2)
        return _grouped(R, E, H, I, rng.choice(("w13", "w2")), rng.random() < 0.5, rng.random() < 0.5)
    groups = rng.choice((1, 1, 2, 4, 8, 16))
    E = groups * max(_spread(rng, 4, 384) // groups, 2)
    keep = rng.randint(1, groups)
    return _route(_spread(rng, 1, 16384), E, rng.randint(1, min(16, E // groups * keep)),
                  rng.choice(("softmax", "sigmoid")), rng.random() < 0.6, groups, keep, dtype)


# ---------------------------------------------------------------- inputs
def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _activations(g, M, K, dtype):
    """Hidden rows: N(0, 1) with one value in a thousand at +-20."""
    x = _normal(g, (M, K))
    far = torch.rand((M, K), generator=g, device="cuda") < 0.001
    return torch.where(far, 20.0 * torch.sign(x), x).to(dtype)


def _weight(g, N, K):
    """A normal weight of 1 / sqrt(K) in fp8 with a scale for 128 x 128 values."""
    return _codes(_normal(g, (N, K)) / math.sqrt(K), True)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "quantize":
        return {"kind": kind, "weight": case["weight"], "x": _activations(g, case["M"], case["K"], DT[case["dtype"]])}
    if kind == "norm":
        M, K, dtype = case["M"], case["K"], DT[case["dtype"]]
        return {"kind": kind, "x": _activations(g, M, K, dtype), "residual": (4.0 * _normal(g, (M, K))).to(dtype),
                "gain": (1.0 + 0.2 * _normal(g, (K,))).to(dtype), "eps": 1e-6}
    if kind == "linear":
        w, ws = _weight(g, case["N"], case["K"])
        return {"kind": kind, "x": _activations(g, case["M"], case["K"], DT[case["dtype"]]), "w": w, "ws": ws,
                "bias": _normal(g, (case["N"],)) if case["bias"] else None}
    if kind == "grouped":
        return _prepare_grouped(case, g)
    T, E = case["T"], case["E"]
    return {"kind": kind, "logits": (1.5 * _normal(g, (T, E))).to(DT[case["dtype"]]),
            "bias": 0.1 * _normal(g, (E,)) if case["bias"] else None, "k": case["k"], "scoring": case["scoring"],
            "groups": case["groups"], "keep": case["keep"], "scale": 2.5 if case["scoring"] == "sigmoid" else 1.0}


def _prepare_grouped(case, g):
    """Expert weights, their tables (which a program keeps with its weights), and expert-sorted rows."""
    R, E, H, I, which = case["R"], case["E"], case["H"], case["I"], case["which"]
    N, K = (2 * I, H) if which == "w13" else (H, I)
    pairs = [_weight(g, N, K) for _ in range(E)]
    bias = _normal(g, (E, N)) if case["bias"] else None
    # rows fall on experts with a skew of about five to one
    p = torch.exp(-1.6 * torch.rand((E,), generator=g, device="cuda"))
    expert = torch.multinomial(p, R, replacement=True, generator=g).sort().values
    offs = torch.searchsorted(expert, torch.arange(E + 1, device="cuda")).to(torch.int32)
    a, scale = _codes(_activations(g, R, K, torch.bfloat16), False)
    if case["by_block"]:
        scale = scale.t().contiguous().t()
    s = {"kind": "grouped", "which": which, "w": torch.stack([w.view(torch.uint8) for w, _ in pairs]).view(F8),
         "ws": torch.stack([ws for _, ws in pairs]), "bias": bias, "a": a, "a_scale": scale, "offs": offs,
         "most": int((offs[1:] - offs[:-1]).max())}
    if own:
        from lockstep_amd import moe_ref
        # the layer's other projection is not called here: one of zeros stands in its place
        other = (H, I) if which == "w13" else (2 * I, H)
        z = (torch.zeros(other, dtype=torch.uint8, device="cuda").view(F8),
             torch.ones((-(-other[0] // BLOCK), -(-other[1] // BLOCK)), device="cuda"))
        one = lambda e: (s["w"][e], s["ws"][e])  # noqa: E731
        bias_of = lambda e: None if bias is None else bias[e]  # noqa: E731
        s["tables"] = moe_ref.ExpertTablesFP8(
            [(one(e), z, bias_of(e), None) if which == "w13" else (z, one(e), None, bias_of(e)) for e in range(E)])
    return s


# ---------------------------------------------------------------- the plain form
def _blocks(x, weight):
    """x [M, K] in blocks of 128 values of a row, or of 128 x 128, zeros past the end."""
    M, K = x.shape
    down = -M % BLOCK if weight else 0
    x = torch.nn.functional.pad(x, (0, -K % BLOCK, 0, down))
    return x.unflatten(1, (-1, BLOCK)).unflatten(0, (-1, BLOCK if weight else 1))    # [rows / b, b, blocks, 128]


def _codes(x, weight):
    """x [M, K] -> (e4m3 [M, K], scales f32 [M or ceil(M / 128), ceil(K / 128)]): the scale is the block's
    largest magnitude over 448, not below 2^-126, and a value is rounded times the scale's reciprocal."""
    M, K = x.shape
    xb = _blocks(x.float(), weight)
    top = xb.abs().amax((1, 3), keepdim=True)
    # (quotients by 64 bits: rounded once to 32 they are the correctly rounded ones of 32)
    scale = (top.double() / 448.0).float().clamp(min=2.0 ** -126)
    q = (xb * (1.0 / scale.double()).float()).to(F8)
    return q.flatten(2).flatten(0, 1)[:M, :K].contiguous(), scale[:, 0, :, 0].contiguous()


def _values(q, scale, weight):
    """What codes and scales stand for, in 32 bits."""
    M, K = q.shape
    v = _blocks(q.float(), weight) * scale[:, None, :, None]
    return v.flatten(2).flatten(0, 1)[:M, :K]


def _normed(s):
    h = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + s["eps"]) * s["gain"].float()
    return y, h


def _padded(rows, offs, most):
    """Expert-sorted rows [R, K] at [E, most, K], and where each went."""
    E, R = offs.numel() - 1, rows.shape[0]
    p = torch.arange(R, device=rows.device)
    e = torch.searchsorted(offs[1:].long(), p, right=True)
    at = e * most + p - offs.long()[e]
    full = torch.zeros((E * most, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    full[at] = rows
    return full.unflatten(0, (E, most)), at, e


def _grouped_product(s):
    E, N, K = s["w"].shape
    # (every expert's scales spread over its values: N need not be a multiple of 128)
    n, k = torch.arange(N, device="cuda") // BLOCK, torch.arange(K, device="cuda") // BLOCK
    wt = (s["w"].float() * s["ws"][:, n][:, :, k]).transpose(1, 2).contiguous()
    full, at, e = _padded(_values(s["a"], s["a_scale"], False), s["offs"], s["most"])
    y = torch.bmm(full, wt).flatten(0, 1)[at]
    return y if s["bias"] is None else y + s["bias"][e]


def _routed(s):
    """In 64 bits: which of two experts is chosen hangs on differences that 32 do not hold."""
    l = s["logits"].double()
    p = torch.exp(l - l.amax(-1, keepdim=True)) if s["scoring"] == "softmax" else 1.0 / (1.0 + torch.exp(-l))
    if s["scoring"] == "softmax":
        p = p / p.sum(-1, keepdim=True)
    c = p if s["bias"] is None else p + s["bias"].double()
    if s["groups"] > 1:
        cg = c.unflatten(-1, (s["groups"], -1))
        top = cg.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        order = top.sort(dim=-1, descending=True, stable=True).indices[:, :s["keep"]]
        kept = torch.zeros_like(top).scatter_(-1, order, 1.0) > 0
        c = torch.where(kept[..., None], cg, -math.inf).flatten(-2)
    idx = c.sort(dim=-1, descending=True, stable=True).indices[:, :s["k"]]
    w = p.gather(-1, idx)
    return idx, (w / w.sum(-1, keepdim=True) * s["scale"]).float()


def run(state):
    s = state
    kind = s["kind"]
    if own:
        from lockstep_amd import lockstep_fullstack as FS, moe_ref, t16n_ref
        if kind == "quantize":
            return FS.dequant_fp8(*(FS.quantize_weight_fp8 if s["weight"] else FS.quantize_rows_fp8)(s["x"]))
        if kind == "norm":
            q, scale, h, _ = t16n_ref.add_rmsnorm_fp8(s["x"], s["residual"], s["gain"], eps=s["eps"])
            return FS.dequant_fp8(q, scale), h
        if kind == "linear":
            return FS.linear_fp8(s["x"], s["w"], s["ws"], s["bias"])
        if kind == "grouped":
            return moe_ref.grouped_linear_fp8(s["tables"], s["which"], s["a"], s["a_scale"], s["offs"])
        return moe_ref.route_experts(s["logits"], s["k"], s["scoring"], bias=s["bias"], groups=s["groups"],
                                     keep_groups=s["keep"], renormalize=True, scale=s["scale"])
    if kind == "quantize":
        return _values(*_codes(s["x"], s["weight"]), s["weight"]).to(torch.bfloat16)
    if kind == "norm":
        y, h = _normed(s)
        return _values(*_codes(y, False), False).to(torch.bfloat16), h
    if kind == "linear":
        y = _values(*_codes(s["x"], False), False) @ _values(s["w"], s["ws"], True).t()
        return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)
    if kind == "grouped":
        return _grouped_product(s).to(torch.bfloat16)
    return _routed(s)


# ---------------------------------------------------------------- 64 bits, from the definition
def _spaced(v, dim):
    """`v` with each entry along dim repeated for its block."""
    return v.repeat_interleave(BLOCK, dim)


def _near(x, weight):
    """x [M, K] rounded to what fp8 holds, in 64 bits: of the multiples of e4m3's spacing the nearest, of two
    as near the even one.  The scale, its reciprocal and the value times it are numbers of 32 bits."""
    M, K = x.shape
    v = torch.zeros((-(-M // BLOCK) * BLOCK if weight else M, -(-K // BLOCK) * BLOCK), dtype=torch.float64, device="cuda")
    v[:M, :K] = x.double()
    top = v.abs().unfold(1, BLOCK, BLOCK).amax(-1)
    if weight:
        top = top.unfold(0, BLOCK, BLOCK).amax(-1)
    s = (top / 448.0).float().double().clamp(min=2.0 ** -126)
    inv = (1.0 / s).float().double()
    if weight:
        s, inv = _spaced(s, 0), _spaced(inv, 0)
    t = (v * _spaced(inv, 1)).float().double()
    e = torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6)))
    d = torch.exp2(e - 3.0)
    return ((torch.round(t / d) * d).clamp(-448.0, 448.0) * _spaced(s, 1))[:M, :K]


def _held(q, scale, weight):
    """The values of e4m3 bytes from their fields: sign, four bits of exponent, three of mantissa."""
    M, K = q.shape
    c = q.view(torch.uint8).double()
    sign = torch.where(c >= 128, -1.0, 1.0).double()
    c = c % 128
    ex, man = torch.floor(c / 8), c % 8
    mag = torch.where(ex == 0, man * 2.0 ** -9, (8.0 + man) * torch.exp2(ex - 10.0))
    s = _spaced(scale.double(), 1)
    if weight:
        s = _spaced(s, 0)
    return sign * mag * s[:M, :K]


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "quantize":
        return _near(s["x"], s["weight"])
    if kind == "norm":
        h = (s["x"].double() + s["residual"].double()).to(s["x"].dtype).double()
        rms = torch.sqrt((h * h).sum(-1, keepdim=True) / h.shape[1] + s["eps"])
        return _near(h / rms * s["gain"].double(), False), h
    if kind == "linear":
        y = torch.matmul(_near(s["x"], False), _held(s["w"], s["ws"], True).t())
        return y if s["bias"] is None else y + s["bias"].double()
    if kind == "grouped":
        offs = s["offs"].tolist()
        y = torch.empty((case["R"], s["w"].shape[1]), dtype=torch.float64, device="cuda")
        for e in range(case["E"]):
            rows = slice(offs[e], offs[e + 1])
            y[rows] = _held(s["a"][rows], s["a_scale"][rows], False) @ _held(s["w"][e], s["ws"][e], True).t()
            if s["bias"] is not None:
                y[rows] += s["bias"][e].double()
        return y
    p = s["logits"].double()
    p = torch.softmax(p, -1) if s["scoring"] == "softmax" else torch.sigmoid(p)
    T, E = p.shape
    c = p.clone() if s["bias"] is None else p + s["bias"].double()[None]
    size = E // s["groups"]
    if s["groups"] > 1:
        first = c.reshape(T, s["groups"], size)
        high = first.amax(-1)
        rest = first.scatter(-1, first.argmax(-1, keepdim=True), -math.inf)
        sums = high + rest.amax(-1)
        dead = torch.ones_like(sums, dtype=torch.bool)
        for _ in range(s["keep"]):
            best = sums.argmax(-1, keepdim=True)
            dead.scatter_(-1, best, False)
            sums.scatter_(-1, best, -math.inf)
        c[dead.repeat_interleave(size, -1)] = -math.inf
    w = []
    for _ in range(s["k"]):
        best = c.argmax(-1, keepdim=True)
        w.append(p.gather(-1, best))
        c.scatter_(-1, best, -math.inf)
    w = torch.cat(w, -1)
    return None, w * (s["scale"] / w.sum(-1, keepdim=True))


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        n = case["M"] * case["K"]
        return {"bytes": n * (SIZE[case["dtype"]] + 2), "flops": 4 * n}
    if kind == "norm":
        n, size = case["M"] * case["K"], SIZE[case["dtype"]]
        return {"bytes": n * (3 * size + 2) + size * case["K"], "flops": 8 * n}
    if kind == "linear":
        M, N, K, size = case["M"], case["N"], case["K"], SIZE[case["dtype"]]
        return {"bytes": size * M * (K + N) + N * K * (1 + 4 / BLOCK ** 2) + 4 * N * case["bias"], "flops": 2 * M * N * K}
    if kind == "grouped":
        R, E, H, I = case["R"], case["E"], case["H"], case["I"]
        N, K = (2 * I, H) if case["which"] == "w13" else (H, I)
        # experts that get a row, were all as likely
        live = E * (1.0 - (1.0 - 1.0 / E) ** R)
        return {"bytes": R * K * (1 + 4 / BLOCK) + live * N * K * (1 + 4 / BLOCK ** 2) + 2 * R * N
                + 4 * live * N * case["bias"], "flops": 2 * R * N * K}
    T, E = case["T"], case["E"]
    return {"bytes": T * E * SIZE[case["dtype"]] + 12 * T * case["k"], "flops": 10 * T * E}
