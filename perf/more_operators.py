"""The calls that the FP8 operators with a scale for each block of 128, and the ways into and out of the experts' order with their
gradients, are measured on.

  quant    E4M3 / E5M2 codes with fp32 scales for blocks of 1 x 128 or 128 x 128, of a matrix or of its transpose
           (``ops.fp8_block_quant``)
  gemm     such activations times such weights; with scales of 1 x 128 on both sides for the gradient of a weight
           (``ops.fp8_block_gemm``)
  gmm      the same for the rows of every expert (``ops.fp8_block_gmm``)
  permute  token rows to the experts' order, the gradient of that, and the gradient of the weighted way back
           (``ops.moe_token_permute``, ``ops.moe_token_permute_grad``, ``ops.moe_token_unpermute_grad``)

``own`` false: the operators from elementary torch operations, 32 bits throughout (scales and the quotients that are rounded to 8
bits in 64, because these may lie next to a border), one rounding at the end.  ``own`` true: the calls of this package.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda"
BLOCK = 128
LEAST = 2.0 ** -126                                              # the smallest scale
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8 = {"E4M3": torch.float8_e4m3fn, "E5M2": torch.float8_e5m2}
FORMAT = {"E4M3": (3, -6, 448.0), "E5M2": (2, -14, 57344.0)}      # mantissa bits, least exponent, largest value
_ops = None


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one token's activations in front of a projection: latency
        {"name": "quant token", "op": "quant", "rows": 1, "cols": 7168, "x": "bf16", "fmt": "E4M3", "square": False, "transposed": False, "pow2": False},
        # the same for a batch of prompts
        {"name": "quant prefill", "op": "quant", "rows": 8192, "cols": 7168, "x": "bf16", "fmt": "E4M3", "square": False, "transposed": False, "pow2": False},
        # an operand of a weight's gradient: transposed, the blocks along an odd number of tokens
        {"name": "quant turned", "op": "quant", "rows": 2777, "cols": 4096, "x": "bf16", "fmt": "E4M3", "square": False, "transposed": True, "pow2": False},
        # one projection of one token: 29 MB of weights
        {"name": "gemm token", "op": "gemm", "m": 1, "n": 4096, "k": 7168, "fmt": "E4M3", "b_rows": 128, "out": "bf16"},
        # the same for a decode batch
        {"name": "gemm batch", "op": "gemm", "m": 64, "n": 4096, "k": 7168, "fmt": "E4M3", "b_rows": 128, "out": "bf16"},
        # the dense configuration's prefill
        {"name": "gemm prefill", "op": "gemm", "m": 8192, "n": 4096, "k": 7168, "fmt": "E4M3", "b_rows": 128, "out": "bf16"},
        # a weight's gradient over 2777 tokens (the codes end in zeros): scales by the row on both sides, in E5M2
        {"name": "gemm gradient", "op": "gemm", "m": 4096, "n": 2048, "k": 2784, "fmt": "E5M2", "b_rows": 1, "out": "bf16"},
        # the second product of a decode step of 32 tokens, top-8 of 256 experts: one or two rows to an expert
        {"name": "gmm decode", "op": "gmm", "rows": 256, "experts": 256, "n": 7168, "k": 2048, "skew": 0.0, "fmt": "E4M3", "out": "bf16"},
        # the first product of a prefill, 16 experts of uneven load
        {"name": "gmm prefill", "op": "gmm", "rows": 32768, "experts": 16, "n": 4096, "k": 7168, "skew": 1.1, "fmt": "E4M3", "out": "bf16"},
        # a batch of prompts to the experts' order, eight copies of each row
        {"name": "permute prefill", "op": "permute", "way": "permute", "tokens": 8192, "top_k": 8, "hidden": 7168, "experts": 256, "x": "bf16"},
        # the gradients of the weighted way back, for the same batch
        {"name": "unpermute gradient", "op": "permute", "way": "unpermute_grad", "tokens": 8192, "top_k": 8, "hidden": 7168, "experts": 256, "x": "bf16"},
        # the gradient of the way there, small and odd
        {"name": "permute gradient", "op": "permute", "way": "permute_grad", "tokens": 777, "top_k": 3, "hidden": 1000, "experts": 16, "x": "fp32"},
    ]


def _log_int(rng, lo, hi):
    """A whole number from [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _step(rng, lo, hi, by):
    """A multiple of `by` from [lo, hi], its logarithm uniform."""
    return min(hi // by * by, max(-(-lo // by) * by, round(_log_int(rng, lo, hi) / by) * by))


def draw(rng):
    op = rng.choice(("quant", "gemm", "gemm", "gmm", "permute"))
    fmt, out = rng.choice(("E4M3", "E4M3", "E5M2")), rng.choice(("bf16", "bf16", "fp16"))
    if op == "quant":
        cols = _log_int(rng, 64, 16384)
        if rng.random() < 0.6:                                   # hidden sizes are mostly whole blocks
            cols = max(128, cols // 128 * 128)
        return {"op": op, "rows": min(_log_int(rng, 1, 8192), 8192 * 7168 // cols), "cols": cols, "x": rng.choice(("bf16", "bf16", "fp16", "fp32")), "fmt": fmt,
                "square": rng.random() < 0.3, "transposed": rng.random() < 0.4, "pow2": rng.random() < 0.2}
    if op == "gemm":
        k = _step(rng, 128, 16384, 128 if rng.random() < 0.7 else 16)
        n = _log_int(rng, 64, 16384)
        if rng.random() < 0.7:
            n = max(64, n // 64 * 64)
        return {"op": op, "m": min(_log_int(rng, 1, 8192), 8192 * 4096 * 7168 // (n * k)), "n": n, "k": k, "fmt": fmt, "b_rows": rng.choice((128, 128, 128, 1)), "out": out}
    if op == "gmm":
        experts = rng.choice((4, 8, 16, 32, 64, 128, 256))
        k = _step(rng, 256, 7168, 128 if rng.random() < 0.7 else 16)
        n = _step(rng, 128, min(7168, 256 * 7168 * 2048 // (experts * k)), 64)
        return {"op": op, "rows": min(_log_int(rng, 1, 32768), 32768 * 4096 * 7168 // (n * k)), "experts": experts, "n": n, "k": k,
                "skew": rng.choice((0.0, 0.5, 1.1 if experts <= 32 else 0.25)), "fmt": fmt, "out": out}
    hidden = _log_int(rng, 64, 8192)
    if rng.random() < 0.7:
        hidden = max(64, hidden // 64 * 64)
    top_k = rng.randint(1, 8)
    x = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    return {"op": op, "way": rng.choice(("permute", "permute_grad", "unpermute_grad")), "tokens": min(_log_int(rng, 1, 8192), 8192 * 8 * 3584 // (top_k * hidden)),
            "top_k": top_k, "hidden": hidden, "experts": rng.choice((8, 16, 64, 256)), "x": x}


# ------------------------------------------------------------------------------------------------ their inputs
def _activations(gen, rows, cols):
    """fp32 N(0, 1) with 0.1 % outliers thirty times as large, as activations have them."""
    x = torch.randn((rows, cols), generator=gen, device=DEV)
    return x.mul_(1.0 + 29.0 * (torch.rand((rows, cols), generator=gen, device=DEV) < 1e-3))


def _coded(x, block_rows, fmt):
    """fp32 x [rows, k] as codes and fp32 scales of its blocks of block_rows x 128."""
    rows, k = x.shape
    nr, nb = -(-rows // block_rows), -(-k // BLOCK)
    most = FORMAT[fmt][2]
    v = torch.nn.functional.pad(x, (0, nb * BLOCK - k, 0, nr * block_rows - rows)).view(nr, block_rows, nb, BLOCK)
    scale = v.abs().amax(dim=(1, 3)).div_(most).clamp_min_(LEAST)
    codes = (v / scale[:, None, :, None]).clamp_(-most, most).to(FP8[fmt])
    return codes.view(nr * block_rows, nb * BLOCK)[:rows, :k].contiguous().view(torch.uint8), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    c, s = case, {"case": case}
    if c["op"] == "quant":
        s["x"] = _activations(gen, c["rows"], c["cols"]).to(DTYPE[c["x"]])
    elif c["op"] == "gemm":
        s["a"], s["a_scale"] = _coded(_activations(gen, c["m"], c["k"]), 1, c["fmt"])
        s["b"], s["b_scale"] = _coded(torch.randn((c["n"], c["k"]), generator=gen, device=DEV).mul_(0.02), c["b_rows"], c["fmt"])
    elif c["op"] == "gmm":
        e, n, k = c["experts"], c["n"], c["k"]
        load = np.random.default_rng(seed)
        p = load.permutation(1.0 / np.arange(1, e + 1) ** c["skew"])
        sizes = load.multinomial(c["rows"], p / p.sum())
        s["sizes"], s["most"] = torch.tensor(sizes, dtype=torch.int32, device=DEV), int(sizes.max())
        s["a"], s["a_scale"] = _coded(_activations(gen, c["rows"], k), 1, c["fmt"])
        s["b"] = torch.empty((e, n, k), dtype=torch.uint8, device=DEV)
        s["b_scale"] = torch.empty((e, -(-n // BLOCK), -(-k // BLOCK)), dtype=torch.float32, device=DEV)
        for i in range(e):
            s["b"][i], s["b_scale"][i] = _coded(torch.randn((n, k), generator=gen, device=DEV).mul_(0.02), BLOCK, c["fmt"])
    else:
        t, k, h = c["tokens"], c["top_k"], c["hidden"]
        expert = torch.rand((t, c["experts"]), generator=gen, device=DEV).topk(k, dim=1).indices.reshape(-1)
        order = torch.sort(expert, stable=True).indices
        s["src2sorted"] = torch.empty(t * k, dtype=torch.int32, device=DEV)
        s["src2sorted"][order] = torch.arange(t * k, dtype=torch.int32, device=DEV)
        rows = t if c["way"] == "permute" else t * k
        s["x"] = torch.randn((rows, h), generator=gen, device=DEV, dtype=torch.float32).to(DTYPE[c["x"]])
        if c["way"] == "unpermute_grad":
            s["dout"] = torch.randn((t, h), generator=gen, device=DEV, dtype=torch.float32).to(DTYPE[c["x"]])
            s["probs"] = torch.softmax(torch.randn((t, k), generator=gen, device=DEV), dim=1)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _rounded(v, mantissa, least, most):
    """v (fp64) to the nearest value with `mantissa` bits behind the point and exponents from `least` on, ties to even, at most `most`."""
    step = torch.exp2(torch.clamp(torch.frexp(v.abs()).exponent.double() - 1.0, min=least) - mantissa)
    return (torch.round(v / step) * step).clamp(-most, most)


def _quant(s):
    c = s["case"]
    x = s["x"].t() if c["transposed"] else s["x"]
    (rows, cols), height = x.shape, BLOCK if c["square"] else 1
    nr, nb = -(-rows // height), -(-cols // BLOCK)
    mantissa, least, most = FORMAT[c["fmt"]]
    v = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - cols, 0, nr * height - rows)).view(nr, height, nb, BLOCK)
    scale = (v.abs().amax(dim=(1, 3)).double() / most).float().clamp_min(LEAST)
    if c["pow2"]:
        fraction, exponent = torch.frexp(scale)
        scale = torch.ldexp(torch.ones_like(scale), exponent - (fraction == 0.5).int())
    codes = _rounded(v.double() / scale[:, None, :, None].double(), mantissa, least, most).float().to(FP8[c["fmt"]])
    return {"codes": codes.view(nr * height, nb * BLOCK)[:rows, :-(-cols // 16) * 16].contiguous(), "scales": scale}


def _dequantized(codes, scale, fmt, block_rows):
    """Codes [..., rows, k] with scales of block_rows x 128 -> fp32."""
    rows, k = codes.shape[-2:]
    v = codes.view(FP8[fmt]).float()
    wide = scale.repeat_interleave(BLOCK, dim=-1)[..., :k]
    if block_rows > 1:
        wide = wide.repeat_interleave(block_rows, dim=-2)[..., :rows, :]
    return v.mul_(wide)


def _gemm(s):
    c = s["case"]
    a, b = _dequantized(s["a"], s["a_scale"], c["fmt"], 1), _dequantized(s["b"], s["b_scale"], c["fmt"], c["b_rows"])
    return torch.matmul(a, b.t()).to(DTYPE[c["out"]])


def _gmm(s):
    c = s["case"]
    a, b = _dequantized(s["a"], s["a_scale"], c["fmt"], 1), _dequantized(s["b"], s["b_scale"], c["fmt"], BLOCK)
    ends = s["sizes"].long().cumsum(0)
    row = torch.arange(c["rows"], device=DEV)
    group = torch.searchsorted(ends, row, right=True)
    at = group * s["most"] + row - (ends - s["sizes"])[group]                    # its row in groups of equal length
    padded = torch.zeros((c["experts"] * s["most"], c["k"]), device=DEV)
    padded[at] = a
    y = torch.matmul(padded.view(c["experts"], s["most"], c["k"]), b.transpose(1, 2).contiguous())
    return y.view(-1, c["n"])[at].to(DTYPE[c["out"]])


def _permute(s):
    c = s["case"]
    to, t, k = s["src2sorted"].long(), c["tokens"], c["top_k"]
    if c["way"] == "permute":
        out = torch.empty((t * k, c["hidden"]), dtype=s["x"].dtype, device=DEV)
        out[to] = s["x"].repeat_interleave(k, dim=0)
        return out
    rows = s["x"][to].view(t, k, c["hidden"]).float()
    if c["way"] == "permute_grad":
        return rows.sum(dim=1).to(s["x"].dtype)
    dout = s["dout"].float()[:, None, :]
    dy = torch.empty_like(s["x"])
    dy[to] = (dout * s["probs"][:, :, None]).view(t * k, c["hidden"]).to(dy.dtype)
    return {"dy": dy, "dprobs": (dout * rows).sum(dim=2)}


# ------------------------------------------------------------------------------------------------ one pass
def _own_run(s):
    global _ops
    if _ops is None:
        from catccos_amd import ops
        _ops = ops
    c = s["case"]
    if c["op"] == "quant":
        codes, scales = _ops.fp8_block_quant(s["x"], c["fmt"], square=c["square"], transposed=c["transposed"], pow2=c["pow2"])
        return {"codes": codes.view(FP8[c["fmt"]]), "scales": scales}
    if c["op"] == "gemm":
        return _ops.fp8_block_gemm(s["a"], s["a_scale"], s["b"], s["b_scale"], c["fmt"], c["out"])
    if c["op"] == "gmm":
        return _ops.fp8_block_gmm(s["a"], s["a_scale"], s["b"], s["b_scale"], s["sizes"], c["fmt"], c["out"])
    if c["way"] == "permute":
        return _ops.moe_token_permute(s["x"], s["src2sorted"], c["top_k"])
    if c["way"] == "permute_grad":
        return _ops.moe_token_permute_grad(s["x"], s["src2sorted"], c["top_k"])
    dy, dprobs = _ops.moe_token_unpermute_grad(s["dout"], s["x"], s["src2sorted"], s["probs"])
    return {"dy": dy, "dprobs": dprobs}


def run(s):
    if own:
        return _own_run(s)
    return {"quant": _quant, "gemm": _gemm, "gmm": _gmm, "permute": _permute}[s["case"]["op"]](s)


# ------------------------------------------------------------------------------------------------ what it cannot do without
def work(case):
    c = case
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if c["op"] == "quant":
        rows, cols = (c["cols"], c["rows"]) if c["transposed"] else (c["rows"], c["cols"])
        scales = -(-rows // (BLOCK if c["square"] else 1)) * -(-cols // BLOCK)
        return {"bytes": rows * cols * (size[c["x"]] + 1) + 4 * scales, "flops": 2 * rows * cols}
    if c["op"] == "gemm":
        nb = -(-c["k"] // BLOCK)
        return {"bytes": (c["m"] + c["n"]) * c["k"] + 4 * nb * (c["m"] + -(-c["n"] // c["b_rows"])) + c["m"] * c["n"] * size[c["out"]],
                "flops": 2 * c["m"] * c["n"] * c["k"]}
    if c["op"] == "gmm":
        p = 1.0 / np.arange(1, c["experts"] + 1) ** c["skew"]
        used = float((1.0 - (1.0 - p / p.sum()) ** c["rows"]).sum())              # experts that get a row, on average
        nb = -(-c["k"] // BLOCK)
        return {"bytes": used * (c["n"] * c["k"] + 4 * nb * -(-c["n"] // BLOCK)) + c["rows"] * (c["k"] + 4 * nb + c["n"] * size[c["out"]]) + 4 * c["experts"],
                "flops": 2 * c["rows"] * c["n"] * c["k"]}
    token, routes = c["tokens"] * c["hidden"] * size[c["x"]], c["tokens"] * c["top_k"]
    if c["way"] == "unpermute_grad":
        return {"bytes": token * (1 + 2 * c["top_k"]) + 12 * routes, "flops": 3 * routes * c["hidden"]}
    return {"bytes": token * (1 + c["top_k"]) + 4 * routes, "flops": routes * c["hidden"]}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _values(codes, fmt):
    """Codes to the numbers that they stand for, from the bits."""
    mantissa, least, _ = FORMAT[fmt]
    c = codes.long()
    e, m = (c & 127) >> mantissa, (c & ((1 << mantissa) - 1)).double() / 2 ** mantissa
    v = torch.where(e == 0, m * 2.0 ** least, (1.0 + m) * torch.exp2((e - 1 + least).double()))
    return torch.where(c >= 128, -v, v)


def _scaled(codes, scale, fmt, block_rows):
    row = torch.arange(codes.shape[0], device=DEV) // block_rows
    col = torch.arange(codes.shape[1], device=DEV) // BLOCK
    return _values(codes, fmt) * scale.double()[row][:, col]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "quant":
        z = s["x"].double()
        z = z.t().contiguous() if c["transposed"] else z
        (rows, cols), height = z.shape, BLOCK if c["square"] else 1
        mantissa, least, most = FORMAT[c["fmt"]]
        nr, nb, wide = -(-rows // height), -(-cols // BLOCK), -(-cols // 16) * 16
        row, col = torch.arange(rows, device=DEV) // height, torch.arange(cols, device=DEV) // BLOCK
        scale = torch.zeros(nr * nb, dtype=torch.float64, device=DEV)
        scale.scatter_reduce_(0, (row[:, None] * nb + col[None, :]).reshape(-1), z.abs().reshape(-1), "amax")
        scale = scale.view(nr, nb) / most
        if c["pow2"]:
            scale = torch.exp2(torch.ceil(torch.log2(scale.clamp_min(1e-300))))
        scale = scale.clamp_min(LEAST).float().double()                           # a scale is an fp32 number
        q = z / scale[row][:, col]
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** least))) - mantissa)
        codes = torch.zeros((rows, wide), dtype=torch.float64, device=DEV)
        codes[:, :cols] = (torch.round(q / step) * step).clamp(-most, most)
        return {"codes": codes, "scales": scale}
    if c["op"] == "gemm":
        return _scaled(s["a"], s["a_scale"], c["fmt"], 1) @ _scaled(s["b"], s["b_scale"], c["fmt"], c["b_rows"]).t()
    if c["op"] == "gmm":
        out, at = torch.zeros((c["rows"], c["n"]), dtype=torch.float64, device=DEV), 0
        for e, size in enumerate(s["sizes"].tolist()):
            if size:
                mine = slice(at, at + size)
                out[mine] = _scaled(s["a"][mine], s["a_scale"][mine], c["fmt"], 1) @ _scaled(s["b"][e], s["b_scale"][e], c["fmt"], BLOCK).t()
                at += size
        return out
    t, k = c["tokens"], c["top_k"]
    to = s["src2sorted"].long().view(t, k)
    if c["way"] == "permute":
        out = torch.zeros((t * k, c["hidden"]), dtype=torch.float64, device=DEV)
        for r in range(k):
            out[to[:, r]] = s["x"].double()
        return out
    if c["way"] == "permute_grad":
        out = torch.zeros((t, c["hidden"]), dtype=torch.float64, device=DEV)
        for r in range(k):
            out += s["x"][to[:, r]].double()
        return out
    dout, dy = s["dout"].double(), torch.zeros(s["x"].shape, dtype=torch.float64, device=DEV)
    dprobs = torch.zeros((t, k), dtype=torch.float64, device=DEV)
    for r in range(k):
        dy[to[:, r]] = s["probs"][:, r, None].double() * dout
        dprobs[:, r] = (dout * s["x"][to[:, r]].double()).sum(dim=1)
    return {"dy": dy, "dprobs": dprobs}
