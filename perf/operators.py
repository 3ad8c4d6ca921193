"""The calls that the operators of one MoE layer at decode, and the stages in front of the experts, are measured on.

  norm     residual addition + root-mean-square norm, to 16 bits and / or to MX codes with E8M0 scales (``ops.rms_norm``,
           ``ops.rms_norm_quant``)
  gating   routing to experts: softmax or sigmoid scores, a bias for balance, expert groups, top-k, renormalised weights
           (``ops.moe_gating``)
  gemv     a few rows of activations times MXFP4 weights (``ops.mxfp4_gemv``)
  ffn      the routed FFN of a few tokens on MXFP4 expert weights, activations in 16 bits (``ops.mxfp4_moe_ffn``)

``own`` false: the operators from elementary torch operations, 32 bits throughout (the gate's scores in 64, because its choices hang
on values that may lie next to each other), one rounding at the end.  ``own`` true: the calls of this package.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ops = None


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the norm in front of a layer at decode: one token, only latency
        {"name": "norm token", "op": "norm", "rows": 1, "cols": 7168, "x": "bf16", "w": "bf16", "residual": True, "fmt": "none", "want_y": True},
        # the same at prefill: codes for the MX matmuls, bf16 for the gate and the dispatch
        {"name": "norm prefill", "op": "norm", "rows": 8192, "cols": 7168, "x": "bf16", "w": "bf16", "residual": True, "fmt": "E4M3", "want_y": True},
        # rows that end inside an MX block (the reference's own odd test width), fp16, codes alone
        {"name": "norm ragged", "op": "norm", "rows": 777, "cols": 1000, "x": "fp16", "w": "fp32", "residual": False, "fmt": "E5M2", "want_y": False},
        # one token's gate: sigmoid scores, balance bias, 4 of 8 groups, top-8 of 256
        {"name": "gating token", "op": "gating", "tokens": 1, "experts": 256, "top_k": 8, "x": "fp32", "score": "sigmoid", "bias": True, "groups": 8,
         "top_groups": 4, "group_best": 2, "renormalize": True},
        # prefill: softmax, top-8 of 256, renormalised (the FFN configuration's own routing)
        {"name": "gating prefill", "op": "gating", "tokens": 8192, "experts": 256, "top_k": 8, "x": "fp32", "score": "softmax", "bias": False, "groups": 1,
         "top_groups": 1, "group_best": 1, "renormalize": True},
        # a batch of long prompts, the grouped form on bf16 logits
        {"name": "gating long", "op": "gating", "tokens": 32768, "experts": 256, "top_k": 8, "x": "bf16", "score": "sigmoid", "bias": True, "groups": 8,
         "top_groups": 4, "group_best": 2, "renormalize": True},
        # one projection of one token: a matrix-vector product, 15.6 MB of weights
        {"name": "gemv token", "op": "gemv", "m": 1, "n": 4096, "k": 7168, "x": "bf16", "out": "bf16"},
        # the same for a decode batch
        {"name": "gemv batch", "op": "gemv", "m": 16, "n": 4096, "k": 7168, "x": "bf16", "out": "bf16"},
        # an odd small projection in 32 bits
        {"name": "gemv ragged", "op": "gemv", "m": 3, "n": 1000, "k": 960, "x": "fp32", "out": "fp32"},
        # the experts of one token, top-8 of 256
        {"name": "ffn token", "op": "ffn", "tokens": 1, "experts": 256, "top_k": 8, "k": 7168, "n": 4096},
        # a decode step of 32 tokens: about 163 experts get a row
        {"name": "ffn batch", "op": "ffn", "tokens": 32, "experts": 256, "top_k": 8, "k": 7168, "n": 4096},
        # an odd number of tokens, experts that share many, sizes that are no multiple of any tile
        {"name": "ffn ragged", "op": "ffn", "tokens": 45, "experts": 16, "top_k": 3, "k": 992, "n": 1088},
    ]


def _log_int(rng, lo, hi):
    """A whole number from [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _step(rng, lo, hi, by):
    """A multiple of `by` from [lo, hi], its logarithm uniform."""
    return min(hi // by * by, max(-(-lo // by) * by, round(_log_int(rng, lo, hi) / by) * by))


def draw(rng):
    op = rng.choice(("norm", "gating", "gemv", "ffn"))
    if op == "norm":
        cols = _log_int(rng, 64, 16384)
        if rng.random() < 0.5:                                   # hidden sizes are mostly whole MX blocks
            cols = max(64, cols // 32 * 32)
        fmt = rng.choice(("none", "E4M3", "E4M3", "E5M2"))
        x = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        return {"op": op, "rows": min(_log_int(rng, 1, 8192), 8192 * 7168 // cols), "cols": cols, "x": x, "w": rng.choice((x, "fp32")),
                "residual": rng.random() < 0.7, "fmt": fmt, "want_y": fmt == "none" or rng.random() < 0.6}
    if op == "gating":
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * _log_int(rng, 4, 512 // groups)
        top_groups = rng.randint(1, groups)
        return {"op": op, "tokens": _log_int(rng, 1, 32768), "experts": experts, "top_k": rng.randint(1, min(16, experts // groups * top_groups)),
                "x": rng.choice(("bf16", "fp16", "fp32")), "score": rng.choice(("softmax", "sigmoid")), "bias": rng.random() < 0.5, "groups": groups,
                "top_groups": top_groups, "group_best": rng.choice((1, 2)), "renormalize": rng.random() < 0.8}
    if op == "gemv":
        k = _step(rng, 64, 16384, 32)
        return {"op": op, "m": _log_int(rng, 1, 64), "n": _log_int(rng, 64, min(32768, 8192 * 8192 // k)), "k": k,
                "x": rng.choice(("bf16", "bf16", "fp16", "fp32")), "out": rng.choice(("bf16", "fp16", "fp32"))}
    experts = rng.choice((8, 16, 32, 64, 128, 256))
    top_k = rng.randint(1, 8)
    k, n = _step(rng, 256, 7168, 32), _step(rng, 256, 4096, 64)
    # as many routes as the largest listed case has work for
    tokens = min(_log_int(rng, 1, 96), max(1, 32 * 8 * 7168 * 4096 // (top_k * k * n)))
    return {"op": op, "tokens": tokens, "experts": experts, "top_k": top_k, "k": k, "n": n}


# ------------------------------------------------------------------------------------------------ their inputs
def _activations(gen, rows, cols, dtype):
    """N(0, 1) with 0.1 % outliers thirty times as large, as activations have them."""
    x = torch.randn((rows, cols), generator=gen, device=DEV)
    x.mul_(1.0 + 29.0 * (torch.rand((rows, cols), generator=gen, device=DEV) < 1e-3))
    return x.to(dtype)


def _mxfp4_weights(gen, experts, n, k):
    """[experts, n, k] of N(0, 0.02) as E2M1 codes [experts, n, k / 2] (even column in the low nibble) with E8M0 scales
    [experts, n, k / 32 rounded up to an even count]."""
    nb = k // 32
    codes = torch.empty((experts, n, k // 2), dtype=torch.uint8, device=DEV)
    scales = torch.full((experts, n, nb + nb % 2), 127, dtype=torch.uint8, device=DEV)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    for e in range(experts):
        w = torch.randn((n, nb, 32), generator=gen, device=DEV).mul_(0.02)
        exp = torch.frexp(w.abs().amax(dim=2)).exponent - 3                  # floor(log2) - 2
        w = torch.ldexp(w, -exp[:, :, None])
        c = torch.bucketize(w.abs(), borders).to(torch.uint8) | ((w < 0).to(torch.uint8) << 3)
        codes[e] = (c[:, :, 0::2] | (c[:, :, 1::2] << 4)).view(n, k // 2)
        scales[e, :, :nb] = (exp + 127).to(torch.uint8)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    c, s = case, {"case": case}
    if c["op"] == "norm":
        s["x"] = _activations(gen, c["rows"], c["cols"], DTYPE[c["x"]])
        s["residual"] = _activations(gen, c["rows"], c["cols"], DTYPE[c["x"]]) if c["residual"] else None
        s["weight"] = (1.0 + 0.2 * torch.randn(c["cols"], generator=gen, device=DEV)).to(DTYPE[c["w"]])
    elif c["op"] == "gating":
        s["logits"] = torch.randn((c["tokens"], c["experts"]), generator=gen, device=DEV).to(DTYPE[c["x"]])
        s["bias"] = 0.05 * torch.randn(c["experts"], generator=gen, device=DEV) if c["bias"] else None
    elif c["op"] == "gemv":
        s["x"] = _activations(gen, c["m"], c["k"], DTYPE[c["x"]])
        w, ws = _mxfp4_weights(gen, 1, c["n"], c["k"])
        s["w"], s["ws"] = w[0], ws[0]
    else:
        s["x"] = torch.randn((c["tokens"], c["k"]), generator=gen, device=DEV).to(torch.bfloat16)
        p, idx = torch.softmax(torch.randn((c["tokens"], c["experts"]), generator=gen, device=DEV), dim=1).topk(c["top_k"], dim=1)
        s["idx"], s["gate"] = idx.to(torch.int32).contiguous(), (p / p.sum(dim=1, keepdim=True)).contiguous()
        s["w1"], s["w1s"] = _mxfp4_weights(gen, c["experts"], c["n"], c["k"])
        s["w2"], s["w2s"] = _mxfp4_weights(gen, c["experts"], c["k"], c["n"] // 2)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
_BYTE_VALUES = {}


def _dequantized(codes, scales, k):
    """E2M1 codes [..., k / 2] with E8M0 scales [..., >= k / 32] -> fp32 [..., k]."""
    if codes.device not in _BYTE_VALUES:
        four = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
        byte = torch.arange(256, device=codes.device)
        _BYTE_VALUES[codes.device] = torch.stack((four[byte & 15], four[byte >> 4]), dim=1)
    v = _BYTE_VALUES[codes.device][codes.int()].view(*codes.shape[:-1], k // 32, 32)
    return (v * torch.exp2(scales[..., :k // 32].float() - 127.0)[..., None]).view(*codes.shape[:-1], k)


def _norm(s):
    c = s["case"]
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
    out = {}
    if s["residual"] is not None:
        out["total"] = x.to(s["x"].dtype)
    if c["want_y"]:
        out["y"] = y.to(s["x"].dtype)
    if c["fmt"] != "none":
        emax, most, dtype = (8, 448.0, torch.float8_e4m3fn) if c["fmt"] == "E4M3" else (15, 57344.0, torch.float8_e5m2)
        rows, cols = y.shape
        nb = -(-cols // 32)
        v = torch.nn.functional.pad(y, (0, nb * 32 - cols)).view(rows, nb, 32)
        amax = v.abs().amax(dim=2)
        exp = torch.where(amax < 1e-12, 0, torch.frexp(amax).exponent - 1 - emax)
        v = torch.ldexp(v, -exp[:, :, None]).clamp(-most, most).to(dtype)
        out["codes"] = v.view(rows, nb * 32)[:, :cols]
        out["scales"] = torch.nn.functional.pad((exp + 127).to(torch.uint8), (0, nb % 2), value=127).view(torch.float8_e8m0fnu)
    return out


def _gating(s):
    c = s["case"]
    z = s["logits"].double()
    if c["score"] == "softmax":
        score = torch.exp(z - z.amax(dim=1, keepdim=True))
        score = score / score.sum(dim=1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-z))
    choice = score if s["bias"] is None else score + s["bias"].double()
    if c["groups"] > 1:
        grouped = choice.view(c["tokens"], c["groups"], -1)
        best = grouped.sort(dim=2, descending=True).values[:, :, :c["group_best"]].sum(dim=2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        closed = torch.ones_like(best, dtype=torch.bool).scatter(1, kept, False)
        choice = grouped.masked_fill(closed[:, :, None], -math.inf).view_as(choice)
    idx = choice.sort(dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
    weight = score.gather(1, idx)
    if c["renormalize"]:
        weight = weight / weight.sum(dim=1, keepdim=True)
    return {"idx": idx.int(), "weight": weight.float()}


def _ffn(s):
    c = s["case"]
    e, half = s["idx"].view(-1).long(), c["n"] // 2
    x = s["x"].float().repeat_interleave(c["top_k"], dim=0)
    h = torch.matmul(_dequantized(s["w1"][e], s["w1s"][e], c["k"]), x[:, :, None])[:, :, 0]
    gate, up = h[:, :half], h[:, half:]
    act = gate / (1.0 + torch.exp(-gate)) * up
    y = torch.matmul(_dequantized(s["w2"][e], s["w2s"][e], half), act[:, :, None])[:, :, 0]
    return (y.view(c["tokens"], c["top_k"], c["k"]) * s["gate"][:, :, None]).sum(dim=1).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ one pass
def _own_run(s):
    global _ops
    if _ops is None:
        from catccos_amd import ops
        _ops = ops
    c = s["case"]
    if c["op"] == "norm":
        if c["fmt"] == "none":
            y, total = _ops.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"])
            return {"y": y} if total is None else {"y": y, "total": total}
        codes, scales, y, total = _ops.rms_norm_quant(s["x"], s["weight"], EPS, residual=s["residual"], fmt=c["fmt"], want_y=c["want_y"])
        out = {"codes": codes.view(torch.float8_e4m3fn if c["fmt"] == "E4M3" else torch.float8_e5m2), "scales": scales.view(torch.float8_e8m0fnu)}
        if y is not None:
            out["y"] = y
        if total is not None:
            out["total"] = total
        return out
    if c["op"] == "gating":
        idx, weight = _ops.moe_gating(s["logits"], c["top_k"], c["score"], s["bias"], c["groups"], c["top_groups"], c["group_best"], c["renormalize"])
        return {"idx": idx, "weight": weight}
    if c["op"] == "gemv":
        return _ops.mxfp4_gemv(s["x"], s["w"], s["ws"], c["out"])
    return _ops.mxfp4_moe_ffn(s["x"], s["idx"], s["gate"], s["w1"], s["w1s"], s["w2"], s["w2s"])


def run(s):
    if own:
        return _own_run(s)
    c = s["case"]
    if c["op"] == "norm":
        return _norm(s)
    if c["op"] == "gating":
        return _gating(s)
    if c["op"] == "gemv":
        return torch.matmul(s["x"].float(), _dequantized(s["w"], s["ws"], c["k"]).t()).to(DTYPE[c["out"]])
    return _ffn(s)


# ------------------------------------------------------------------------------------------------ what it cannot do without
def work(case):
    c = case
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if c["op"] == "norm":
        b = size[c["x"]]
        an_element = b * (3 if c["residual"] else 1) + (b if c["want_y"] else 0) + (1 + 1 / 32 if c["fmt"] != "none" else 0)
        return {"bytes": c["rows"] * c["cols"] * an_element + c["cols"] * size[c["w"]], "flops": 5 * c["rows"] * c["cols"]}
    if c["op"] == "gating":
        return {"bytes": c["tokens"] * (c["experts"] * size[c["x"]] + 8 * c["top_k"]) + (4 * c["experts"] if c["bias"] else 0),
                "flops": 10 * c["tokens"] * c["experts"]}
    mx = 0.5 + 1 / 32
    if c["op"] == "gemv":
        return {"bytes": c["n"] * c["k"] * mx + c["m"] * (c["k"] * size[c["x"]] + c["n"] * size[c["out"]]), "flops": 2 * c["m"] * c["n"] * c["k"]}
    # experts that get a row, on average, when every token takes top_k of them at random
    used = c["experts"] * (1.0 - (1.0 - c["top_k"] / c["experts"]) ** c["tokens"])
    routes = c["tokens"] * c["top_k"]
    return {"bytes": used * 1.5 * c["n"] * c["k"] * mx + 4 * c["tokens"] * c["k"] + 8 * routes, "flops": 3 * routes * c["n"] * c["k"]}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _rounded(v, mantissa, least, most):
    """v (fp64) to the nearest value with `mantissa` bits behind the point and exponents from `least` on, ties to even, at most `most`."""
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(v.abs().clamp_min(1e-300))), min=least) - mantissa)
    return (torch.round(v / step) * step).clamp(-most, most)


def _weights64(codes, scales, k):
    low, high = (codes & 15).long(), (codes >> 4).long()
    c = torch.stack((low, high), dim=-1).flatten(-2)
    e, m = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e == 0, 0.5 * m, torch.exp2(e.double() - 1.0) * (1.0 + 0.5 * m)) * (1.0 - 2.0 * (c >> 3).double())
    return v * torch.exp2(scales[..., :k // 32].double() - 127.0).repeat_interleave(32, dim=-1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "norm":
        t = s["x"].double() + (0.0 if s["residual"] is None else s["residual"].double())
        y = t / torch.sqrt(t.pow(2).sum(dim=1, keepdim=True) / c["cols"] + EPS) * s["weight"].double()
        out = {}
        if s["residual"] is not None:
            out["total"] = t
        if c["want_y"]:
            out["y"] = y
        if c["fmt"] != "none":
            emax, mantissa, least, most = (8, 3, -6, 448.0) if c["fmt"] == "E4M3" else (15, 2, -14, 57344.0)
            nb = -(-c["cols"] // 32)
            scale = torch.ones((c["rows"], nb + nb % 2), dtype=torch.float64, device=DEV)
            codes = torch.zeros((c["rows"], nb * 32), dtype=torch.float64, device=DEV)
            codes[:, :c["cols"]] = y
            amax = codes.view(c["rows"], nb, 32).abs().max(dim=2).values
            scale[:, :nb] = torch.where(amax < 1e-12, 1.0, torch.exp2(torch.floor(torch.log2(amax.clamp_min(1e-300))) - emax))
            codes = _rounded(codes / scale[:, :nb].repeat_interleave(32, dim=1), mantissa, least, most)
            out["codes"], out["scales"] = codes[:, :c["cols"]], scale
        return out
    if c["op"] == "gating":
        z = s["logits"].double().cpu().numpy()
        if c["score"] == "softmax":
            p = np.exp(z - z.max(axis=1, keepdims=True))
            p /= p.sum(axis=1, keepdims=True)
        else:
            p = 1.0 / (1.0 + np.exp(-z))
        key = p + (0.0 if s["bias"] is None else s["bias"].double().cpu().numpy())
        if c["groups"] > 1:
            members = key.reshape(c["tokens"], c["groups"], -1)
            best = -np.sort(-members, axis=2)[:, :, :c["group_best"]].sum(axis=2)
            order = np.argsort(-best, axis=1, kind="stable")
            closed = np.ones(best.shape, dtype=bool)
            np.put_along_axis(closed, order[:, :c["top_groups"]], False, axis=1)
            key = np.where(closed[:, :, None], -np.inf, members).reshape(key.shape)
        idx = np.argsort(-key, axis=1, kind="stable")[:, :c["top_k"]]
        w = np.take_along_axis(p, idx, axis=1)
        return {"idx": idx.astype(np.int32), "weight": w / w.sum(axis=1, keepdims=True) if c["renormalize"] else w}
    if c["op"] == "gemv":
        return s["x"].double() @ _weights64(s["w"], s["ws"], c["k"]).t()
    half = c["n"] // 2
    x, out = s["x"].double(), torch.zeros((c["tokens"], c["k"]), dtype=torch.float64, device=DEV)
    for e in torch.unique(s["idx"]).tolist():
        t, r = torch.nonzero(s["idx"] == e, as_tuple=True)
        h = x[t] @ _weights64(s["w1"][e], s["w1s"][e], c["k"]).t()
        a = h[:, :half] * torch.sigmoid(h[:, :half]) * h[:, half:]
        out.index_add_(0, t, s["gate"][t, r].double()[:, None] * (a @ _weights64(s["w2"][e], s["w2s"][e], half).t()))
    return out
