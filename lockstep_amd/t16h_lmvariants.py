"""Drop-in for the lm_head / linear arithmetic variants of reference/t16h_lmvariants.py, on MI355X.

Same names, signatures, dtypes and return values as the reference (device tensors only; the
arithmetic runs in the HIP kernels of liblockstep_amd.so):

    _int_mm(a8, b8)                 t16h_lmvariants.py:51-68    exact int8 GEMM -> int32
    _planes(a_i32, sh)              :71-77                      the two-plane int8 carrier
    _quant_rows(x2, abits)          :80-84                      per-row <abits>-bit quant
    quantize_weight_int8(W)         :87-92
    quantize_weight(W, wbits)       :95-103                    planes [(sh, [K, N] view)], ws
    smooth_scales(act_amax, W, a)   :106-112                    SmoothQuant per-input-channel scale
    _mm_planes(x2, wplanes, ws, abits)   :115-125               planes combined exactly in int64
    Variant, build(spec), needs_calibration(specs)              :128-201

and, with no counterpart there, the variant "mxfp4" (weight and rows in MXFP4, moe_mxfp4.linear_mxfp4)
and penalize_logits(logits, ...): penalties for repeated tokens, biases and allowed-token masks.

A <B>-bit value (B in 8, 11, 15) rides two int8 planes hi = a >> (B - 8), lo = a - (hi << (B - 8));
the plane products are exact int32 GEMMs and the combine is exact in int64, so the result is
fl32(fl32(fl32(s) * asc[m]) * ws[n]) of the exact integer s = sum_k a[m, k] * w[n, k].  On the
device the activation planes are stacked under each other and the weight planes side by side,
so one exact GEMM evaluates every plane product (the weight is read once per call), and one
kernel combines them with the epilogue.

`smooth_scales` (binary32 pow, a prepare-time artifact, not on the GEMM path) and the "bf16"
variant (the stock float lm_head, not a contract op) run as the reference writes them, in torch.
"""
from __future__ import annotations

import re

import torch

from . import _lib as L
from . import ops

INT8_MIN_ROWS = 17          # kept for API compatibility: the kernels take any row count


def _const(value: float, ref):
    """Device/dtype-resident scalar (the reference's tensor divisor helper)."""
    return torch.tensor(float(value), device=ref.device, dtype=ref.dtype)


def _int_mm(a8, b8):
    """int8 [M, K] x int8 [K, N] -> int32 [M, N], exact for any M."""
    return ops.gemm(a8, ops.weight_nk(b8), L.EPI_RAW, L.LSK_I32)


def _planes(a_i32, sh):
    """a = (hi << sh) + lo, hi in [-128, 127], lo in [0, 2^sh - 1]; sh = 0 -> one plane."""
    return ops.split_planes(a_i32, sh)


def _quant_rows(x2, abits):
    """amax_q = 2^(abits-1) - 1; asc = max(|x|, 1e-8) / amax_q; a = clamp(rint(x / asc)) (int32)."""
    return ops.quant_bits(x2, abits)


def quantize_weight_int8(W):
    """Per-out-channel int8 weight, contract_common.w8a8_linear semantics."""
    W8, ws = ops.rowquant(W.detach())
    return W8.contiguous(), ws.contiguous()


def quantize_weight(W, wbits):
    """Per-out-channel <wbits>-bit weight carried by 1 or 2 int8 planes; each plane is [K, N] with
    stride (1, K), a view into one stacked [P * N, K] buffer (hi plane rows first)."""
    w2, ws = ops.quant_planes(W.detach(), wbits)
    return _plane_views(w2, wbits, W.shape[0]), ws


def _plane_views(w2, wbits, N):
    if wbits == 8:
        return [(0, w2.t())]
    return [(wbits - 8, w2[:N].t()), (0, w2[N:].t())]


def _stacked(wplanes):
    """The stacked [P * N, K] weight buffer behind a planes list (a view when the planes came from
    quantize_weight, else one copy), with the weight width it implies."""
    nk = [p.t() for _, p in wplanes]
    if len(nk) == 1:
        return (nk[0] if nk[0].stride(-1) == 1 else nk[0].contiguous()), 8
    wbits = wplanes[0][0] + 8
    if wbits not in (11, 15) or wplanes[1][0] != 0 or len(nk) != 2:
        raise ValueError("weight planes must be [(wbits - 8, hi), (0, lo)] with wbits 11 or 15")
    hi, lo = nk
    N, K = hi.shape
    adjacent = (hi.is_contiguous() and lo.is_contiguous() and lo.data_ptr() == hi.data_ptr() + N * K)
    if adjacent:
        return hi.as_strided((2 * N, K), (K, 1)), wbits
    return torch.cat([hi, lo], 0).contiguous(), wbits


def smooth_scales(act_amax, W, alpha):
    """SmoothQuant per-IN-channel scale, folded once into the weight (prepare time)."""
    Wf = W.detach().float()
    w_amax = Wf.abs().amax(dim=0).clamp(min=1e-5)
    a_amax = act_amax.detach().float().to(Wf.device).clamp(min=1e-5)
    s = (a_amax ** float(alpha)) / (w_amax ** (1.0 - float(alpha)))
    return s.clamp(min=1e-5).contiguous()


def _mm_planes(x2, wplanes, ws, abits, sdiv=None):
    """x2 [rows, K] float -> [rows, N] float32: the <abits> row quant (after x / sdiv when given),
    every plane product exact, combined in int64, then fl32(fl32(fl32(s) * asc) * ws)."""
    w2, wbits = _stacked(wplanes)
    return ops.planes_linear(x2, w2, wbits, ws, abits, sdiv=sdiv)


class Variant:
    """name -> logits.  `prepare` is called once with the bf16 lm_head weight and (for the sq
    family) the calibrated per-in-channel activation amax."""

    def __init__(self, name, kind, abits=8, wbits=8, alpha=None):
        self.name, self.kind = name, kind
        self.abits, self.wbits, self.alpha = abits, wbits, alpha
        self.wplanes = self.ws = self.sdiv = self.W_bf16 = None
        self._w4 = None            # the MXFP4 variant's packed codes [N, K/2] (ws: its scales [N, K/32])
        self._w2 = None            # the stacked weight planes [P * N, K] the kernels read

    def prepare(self, W, act_amax=None):
        self.W_bf16 = W
        if self.kind == "bf16":
            return self
        if self.kind == "mxfp4":
            self._w4, self.ws = ops.quantize_mxfp4(W.detach())
            return self
        if self.alpha is not None:
            if act_amax is None:
                raise RuntimeError("variant %s needs a calibrated act_amax" % self.name)
            self.sdiv = smooth_scales(act_amax, W, self.alpha)
        # the fold W * sdiv[None, :] runs inside the weight quant kernel (the same binary32 product)
        fold = 0 if self.sdiv is None else 2
        self._w2, self.ws = ops.quant_planes(W.detach(), self.wbits, sdiv=self.sdiv, sdiv_op=fold)
        self.wplanes = _plane_views(self._w2, self.wbits, W.shape[0])
        # a wide head's decode batches read a copy of the planes: made here, with the planes, so that
        # logits() packs nothing (65536 x 3584 in 15 bits: 470 MB)
        ops.prepare_planes_pairs(self._w2, self.abits)
        return self

    def logits(self, x2):
        """x2 : [rows, K] float32 -> [rows, N] float32."""
        if self.kind == "bf16":
            return torch.nn.functional.linear(x2.to(self.W_bf16.dtype), self.W_bf16).float()
        if self.kind == "mxfp4":
            return ops.linear_mxfp4(x2, self._w4, self.ws, out_dtype=torch.float32)
        rows = x2.numel() // max(1, x2.shape[-1])
        return ops.planes_linear(x2, self._w2, self.wbits, self.ws, self.abits, sdiv=self.sdiv,
                                 w_pairs=ops.planes_pairs(self._w2, rows, self.abits))

    def n_out(self):
        return int(self.W_bf16.shape[0])

    def gemms(self):
        """int8 GEMMs per call: activation planes x weight planes (0 for the float and MXFP4 heads)."""
        if self.kind in ("bf16", "mxfp4"):
            return 0
        return (2 if self.abits > 8 else 1) * len(self.wplanes)

    def nbytes(self):
        """Bytes of the published constants: weight planes, smoothing vector, scales."""
        if self.kind == "mxfp4":
            return 0 if self._w4 is None else self._w4.numel() + self.ws.numel()
        parts = [p.numel() for _, p in (self.wplanes or [])]
        parts += [4 * t.numel() for t in (self.sdiv, self.ws) if t is not None]
        return sum(parts)


_SPEC = re.compile(r"(?:sq(?P<sq>\d*))?(?P<rest>.*)")
_AW = re.compile(r"(?:a(?P<a>\d+))?(?:w(?P<w>\d+))?")


def build(spec: str) -> Variant:
    """bf16 | mxfp4 | [sq<AA>][a<A>][w<W>].  e.g. a8  a15  a15w15  sq50  sq50a15  sq80a15w15"""
    s = spec.strip()
    if s in ("bf16", "mxfp4"):
        return Variant(s, s)
    head = _SPEC.fullmatch(s)
    alpha = None
    if s.startswith("sq"):
        if not head.group("sq"):
            raise ValueError("sq needs an alpha, e.g. sq50: %r" % spec)
        alpha = int(head.group("sq")) / 100.0
    aw = _AW.fullmatch(head.group("rest"))
    if aw is None:
        raise ValueError("unknown lm_head variant spec: %r" % spec)
    abits = int(aw.group("a") or 8)
    wbits = int(aw.group("w") or 8)
    for b, what in ((abits, "activation"), (wbits, "weight")):
        if b not in (8, 11, 15):
            raise ValueError("%s width %d not supported (8, 11, 15): %r" % (what, b, spec))
    return Variant(s, "planes", abits=abits, wbits=wbits, alpha=alpha)


def needs_calibration(specs) -> bool:
    return any(sp.strip().startswith("sq") for sp in specs)


def penalize_logits(logits, prompt=None, prompt_lens=None, output=None, output_lens=None, repetition=None, frequency=None,
                    presence=None, bias=None, mask=None, out=None):
    """What a sampler does to a head's logits [B, V] before it draws, in one pass (ops.penalize_logits):
    bias, the repetition penalty over prompt and output tokens, the frequency and presence penalties
    over output tokens, then -inf where the allowed-token bits of `mask` are 0."""
    return ops.penalize_logits(logits, prompt, prompt_lens, output, output_lens, repetition, frequency, presence, bias,
                               mask, out)
