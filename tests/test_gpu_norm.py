"""Residual addition + root-mean-square norm + MX codes against the definition in 64 bits, and bit for bit where the norm is exact."""
import numpy as np
import pytest
import torch

from tests.gpu_util import bf16_dev, host

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# What fp32 loses before the one rounding of an output: t 2^-24, the sum of squares (positive terms; at most 40 additions in a thread, 6 in
# a wavefront, 16 across wavefronts, half of it in the root) 31 * 2^-24, division, addition of eps, root and reciprocal 2 * 2^-24 and two
# products 2 * 2^-24: below 2^-18
FP32_LOSS = 2.0 ** -18
FORMATS = {"E4M3": (8, 3, -6, 448.0), "E5M2": (15, 2, -14, 57344.0), "E2M1": (2, 1, 0, 6.0)}


def _inputs(rows, cols, x, w, residual, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda: (torch.randn((rows, cols), generator=g, device="cuda") * torch.exp(torch.randn((rows, 1), generator=g, device="cuda"))).to(DTYPES[x])
    return make(), make() if residual else None, (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).to(DTYPES[w])


def _definition(x, r, w, eps):
    t = x.double() if r is None else x.double() + r.double()
    return t, t / torch.sqrt(t.pow(2).mean(dim=1, keepdim=True) + eps) * w.double()


def _assert_rounded(got, want, what):
    """got: want computed in fp32 and rounded once to got's type."""
    info = torch.finfo(got.dtype)
    step = info.eps / 2 if got.dtype != torch.float32 else 0.0
    bound = want.abs() * (step + FP32_LOSS) + info.smallest_normal * info.eps          # (the spacing of the smallest values)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"{what}: {float((err / bound.clamp_min(1e-300)).max())} times the bound"


def _values(codes, fmt, cols):
    if fmt == "E2M1":
        tab = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device="cuda")
        c = torch.stack((codes & 15, codes >> 4), dim=2).flatten(1)[:, :cols].long()
        return tab[c]
    return codes.view(torch.float8_e4m3fn if fmt == "E4M3" else torch.float8_e5m2).double()


def _assert_codes(codes, scales, y, fmt):
    """Codes and scales of y [rows, cols] (fp64): the shared exponent of each block's maximum - either one where the maximum is within FP32_LOSS of
    a power of two - and under it each element's nearest value, half a step off at most."""
    rows, cols = y.shape
    emax, mantissa, least, most = FORMATS[fmt]
    nb = -(-cols // 32)
    assert scales.shape == (rows, nb + nb % 2)
    if nb % 2:
        assert bool((scales[:, nb] == 127).all())
    padded = torch.nn.functional.pad(y, (0, nb * 32 - cols)).view(rows, nb, 32)
    amax = padded.abs().amax(dim=2)
    exp = lambda a: torch.where(a < 1e-12, 0.0, torch.floor(torch.log2(a.clamp_min(1e-300))) - emax)
    got = scales[:, :nb].double() - 127
    assert bool(((got == exp(amax * (1 - FP32_LOSS))) | (got == exp(amax * (1 + FP32_LOSS)))).all()), "scales"
    scale = torch.exp2(got).repeat_interleave(32, dim=1)[:, :cols]
    v, target = _values(codes, fmt, cols), (y / scale).clamp(-most, most)
    step = torch.exp2(torch.floor(torch.log2(target.abs().clamp_min(2.0 ** least))) - mantissa)
    err = (v - target).abs()
    assert bool((err <= step / 2 + target.abs() * FP32_LOSS).all()), f"codes: {int((err > step / 2 + target.abs() * FP32_LOSS).sum())} of {err.numel()}"


@pytest.mark.parametrize("cols", [1, 7, 8, 31, 32, 33, 96, 511, 512, 513, 1000, 1024, 1025, 2047, 2050, 4096, 4100, 7168, 8191, 8193, 16384, 16391, 40000])
@pytest.mark.parametrize("x,w,residual", [("bf16", "bf16", True), ("fp16", "fp32", False), ("fp32", "fp32", True)])
def test_every_length(cols, x, w, residual):
    from catccos_amd import ops
    for rows in (1, 5):
        a, r, weight = _inputs(rows, cols, x, w, residual, cols + rows)
        t, y = _definition(a, r, weight, 1e-6)
        got_y, got_t = ops.rms_norm(a, weight, 1e-6, residual=r)
        _assert_rounded(got_y, y, "y")
        assert got_y.dtype == a.dtype and (got_t is None) == (r is None)
        if r is not None:
            _assert_rounded(got_t, t, "t")
        for fmt in FORMATS:
            codes, scales, y2, t2 = ops.rms_norm_quant(a, weight, 1e-6, residual=r, fmt=fmt, want_y=fmt != "E5M2")
            _assert_codes(codes, scales, y, fmt)
            assert (y2 is None) == (fmt == "E5M2") and (y2 is None or torch.equal(y2, got_y)) and (r is None or torch.equal(t2, got_t))


@pytest.mark.parametrize("x,w", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("rows", [2, 300, 2000])
def test_types_and_batches(x, w, rows):
    from catccos_amd import ops
    a, r, weight = _inputs(rows, 1536, x, w, True, rows)
    t, y = _definition(a, r, weight, 1e-5)
    codes, scales, got_y, got_t = ops.rms_norm_quant(a, weight, 1e-5, residual=r, want_y=True)
    _assert_rounded(got_y, y, "y")
    _assert_rounded(got_t, t, "t")
    _assert_codes(codes, scales, y, "E4M3")


@pytest.mark.parametrize("fmt", ["E4M3", "E5M2", "E2M1"])
@pytest.mark.parametrize("cols", [512, 2048, 8192, 16384, 65536])
def test_codes_equal_the_quantizers_where_the_norm_is_exact(fmt, cols):
    """Rows of +-2^j have a root mean square of 2^j exactly, so y is +- the weight: with every bf16 pattern as a weight, Inf and NaN among them,
    codes and scales must be those that mx_quant makes of y, bit for bit."""
    from catccos_amd import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    patterns = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(-1, cols)
    for shift in (0, 7):
        weights = patterns[:, torch.randperm(cols, generator=g, device="cuda")] if shift else patterns
        for weight in weights[:: max(1, len(weights) // 16)]:
            x = torch.ones((4, cols), device="cuda") * torch.tensor([1.0, 2.0 ** 9, 2.0 ** -30, -4.0], device="cuda")[:, None]
            codes, scales, y, _ = ops.rms_norm_quant(x.to(torch.bfloat16), weight.contiguous(), 0.0, fmt=fmt, want_y=True)
            want_y = weight.float() * torch.tensor([1.0, 1.0, 1.0, -1.0], device="cuda")[:, None]
            assert torch.equal(y.float().nan_to_num(nan=12345.0), want_y.nan_to_num(nan=12345.0))
            want_codes, want_scales = ops.mx_quant(want_y.to(torch.bfloat16), fmt, "rne")
            assert torch.equal(scales, want_scales)
            same = codes == want_codes
            if fmt != "E2M1":        # the sign of a NaN is not the weight's after a product
                same |= torch.isnan(want_y) & ((codes & 0x7F) == (want_codes & 0x7F))
            assert bool(same.all()), int((~same).sum())


def test_rows_apart_from_each_other_and_what_lies_between_them():
    """Through the C ABI with a pitch of its own for every operand: the bytes behind each row stay as they were, and rows need no more alignment
    than their elements."""
    from catccos_amd import _lib, ops
    for cols, pad in ((1000, 3), (77, 1), (4096, 24), (9000, 5)):
        rows, p = 6, cols + pad
        a, r, weight = _inputs(rows, p, "bf16", "bf16", True, cols)
        t, y = _definition(a[:, :cols], r[:, :cols], weight[:cols], 1e-6)
        nb = ops.scale_cols(cols)
        total, out = (torch.full((rows, p), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        codes, scales = (torch.full((rows, n + pad), 0xEE, dtype=torch.uint8, device="cuda") for n in (cols, nb))
        _lib.check(_lib.load().cmx_rms_norm_quant(a.data_ptr(), p, r.data_ptr(), p, weight.data_ptr(), total.data_ptr(), p, out.data_ptr(), p, codes.data_ptr(),
                                                  cols + pad, scales.data_ptr(), nb + pad, rows, cols, ops._bits(1e-6), 0, 0, 0,
                                                  torch.cuda.current_stream().cuda_stream))
        _assert_rounded(total[:, :cols], t, "t")
        _assert_rounded(out[:, :cols], y, "y")
        _assert_codes(codes[:, :cols].contiguous(), scales[:, :nb].contiguous(), y, "E4M3")
        assert bool((total[:, cols:] == 7).all()) and bool((out[:, cols:] == 7).all()) and bool((codes[:, cols:] == 0xEE).all())
        assert bool((scales[:, nb:] == 0xEE).all())


@pytest.mark.parametrize("cols", [96, 1000, 7168, 16390])
def test_the_total_in_place(cols):
    from catccos_amd import ops
    a, r, weight = _inputs(7, cols, "bf16", "bf16", True, cols)
    want_y, want_t = ops.rms_norm(a, weight, residual=r)
    for into in ("x", "residual"):
        a2, r2 = a.clone(), r.clone()
        buf = a2 if into == "x" else r2
        y, t = ops.rms_norm(a2, weight, residual=r2, total=buf)
        assert t is buf and torch.equal(t, want_t) and torch.equal(y, want_y)


def test_strided_views_and_single_rows():
    from catccos_amd import ops
    a, r, weight = _inputs(9, 640, "bf16", "bf16", True, 1)
    want_y, want_t = ops.rms_norm(a[:, 64:576].contiguous(), weight[:512], residual=r[:, 64:576].contiguous())
    y, t = ops.rms_norm(a[:, 64:576], weight[:512], residual=r[:, 64:576])
    assert torch.equal(y, want_y) and torch.equal(t, want_t)
    y, t = ops.rms_norm(a[::3, 65:577], weight[:512], residual=r[::3, 65:577])
    want_y, want_t = ops.rms_norm(a[::3, 65:577].contiguous(), weight[:512], residual=r[::3, 65:577].contiguous())
    assert torch.equal(y, want_y) and torch.equal(t, want_t)
    column = a[0].clone().view(-1, 1).t()                        # one row whose row stride says 1
    assert torch.equal(ops.rms_norm(column, weight)[0], ops.rms_norm(a[:1], weight)[0])
    y, t = ops.rms_norm(a[:0], weight, residual=r[:0])
    assert y.shape == t.shape == (0, 640)


def test_rows_past_32_bits_of_elements():
    from catccos_amd import ops
    apart, cols = (1 << 32) - 8, 1000                                     # 17 GB from the first row to the last
    buf = torch.empty(2 * apart + cols, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, cols), (apart, 1))
    a, _, weight = _inputs(3, cols, "bf16", "bf16", False, 5)
    x.copy_(a)
    assert torch.equal(ops.rms_norm(x, weight)[0], ops.rms_norm(a, weight)[0])


def test_non_finite_and_empty_rows():
    from catccos_amd import ops
    a, _, weight = _inputs(6, 96, "bf16", "bf16", False, 2)
    a[0] = 0
    a[1, 5] = float("nan")
    a[2, 40] = float("inf")
    a[3, 41] = float("-inf")
    a[4] = 1e30                                                    # squares past fp32
    codes, scales, y, _ = ops.rms_norm_quant(a, weight, 1e-6, want_y=True)
    assert bool((y[0] == 0).all()) and bool((codes[0] == 0).all()) and bool((scales[0] == 127).all())
    assert bool(y[1].isnan().all()) and bool(((codes[1] & 0x7F) == 0x7F).all())
    for row, at in ((2, 40), (3, 41)):
        assert bool(y[row, at].isnan()) and bool((y[row, torch.arange(96, device="cuda") != at] == 0).all())
    assert bool((y[4] == 0).all())
    assert torch.equal(y[5], ops.rms_norm(a[5:], weight)[0][0])
    assert bool(ops.rms_norm(a[:1], weight, 0.0)[0].isnan().all())          # 0 / 0, as the formula says


def test_on_a_side_stream_and_captured():
    from catccos_amd import ops
    ops.init()
    a, r, weight = _inputs(33, 7168, "bf16", "bf16", True, 9)
    want = ops.rms_norm_quant(a, weight, residual=r, want_y=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rms_norm_quant(a, weight, residual=r, want_y=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rms_norm_quant(a, weight, residual=r, want_y=True)
    for rep in range(3):
        a.copy_(torch.randn(a.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, ops.rms_norm_quant(a, weight, residual=r, want_y=True))), rep


@pytest.mark.parametrize("x,w,residual", [("bf16", "bf16", True), ("fp16", "fp32", False), ("fp32", "fp32", True)])
@pytest.mark.parametrize("cols", [1025, 1348, 1600, 2041, 2048])
def test_many_rows_of_middling_length(cols, x, w, residual):
    """Rows of 16 bits of which there are many: a wavefront to each."""
    from catccos_amd import ops
    a, r, weight = _inputs(5003, cols, x, w, residual, cols)
    t, y = _definition(a, r, weight, 1e-6)
    codes, scales, got, total = ops.rms_norm_quant(a, weight, residual=r, want_y=True)
    _assert_rounded(got, y, "y")
    _assert_codes(codes, scales, y, "E4M3")
    if residual:
        assert torch.equal(total, (a.float() + r.float()).to(a.dtype))


@pytest.mark.parametrize("x,w,residual", [("bf16", "bf16", True), ("bf16", "fp32", False), ("fp16", "fp16", True), ("fp32", "fp32", True)])
@pytest.mark.parametrize("rows,cols", [(20000, 96), (6000, 1000), (5000, 1531), (1500, 4096), (700, 12288), (300, 20007)])
def test_codes_are_those_of_the_exact_norm(rows, cols, x, w, residual):
    """Every code and every scale of millions, in all formats, against 64 bits with no tolerance: fp32 arithmetic would put about one in a million elsewhere."""
    from catccos_amd import ops
    a, r, weight = _inputs(rows, cols, x, w, residual, rows)
    t = a.float() if r is None else a.float() + r.float()
    y = t.double() / torch.sqrt(t.double().pow(2).mean(dim=1, keepdim=True) + float(np.float32(1e-6))) * weight.double()
    nb = -(-cols // 32)
    amax = torch.nn.functional.pad(y, (0, nb * 32 - cols)).view(rows, nb, 32).abs().amax(dim=2)
    for fmt, (emax, mantissa, least, most) in FORMATS.items():
        codes, scales, _, _ = ops.rms_norm_quant(a, weight, residual=r, fmt=fmt)
        exp = torch.frexp(amax).exponent - 1 - emax
        exp = torch.where(amax < 1e-12, 0, exp)
        assert torch.equal(scales[:, :nb].int(), (exp + 127).int())
        target = torch.ldexp(y, -exp.repeat_interleave(32, dim=1)[:, :cols])
        step = torch.exp2((torch.frexp(target.abs().clamp_min(2.0 ** least)).exponent - 1 - mantissa).double())
        want = (torch.round(target / step) * step).clamp(-most, most)
        off = (_values(codes, fmt, cols) != want).sum()
        assert int(off) == 0, (fmt, int(off))


@pytest.mark.parametrize("x,w", [("bf16", "bf16"), ("fp32", "fp32"), ("bf16", "fp32")])
@pytest.mark.parametrize("cols", [96, 1000, 2048, 4100, 12288, 20007])
@pytest.mark.parametrize("eps", [0.0, 1e-44, 1e-38])
def test_rows_whose_squares_fp32_cannot_hold(cols, x, w, eps):
    """Rows of 2^-20 down to the smallest numbers of the type, with an eps of their size or none: y, codes and scales are as exact as elsewhere."""
    from catccos_amd import ops
    g = torch.Generator(device="cuda").manual_seed(cols)
    scale = 2.0 ** -torch.tensor([20.0, 44, 46, 60, 63, 64, 70, 74, 75, 90, 110, 126, 128, 131], dtype=torch.float64, device="cuda")
    a, r = ((torch.randn((len(scale), cols), generator=g, device="cuda").double() * scale[:, None]).to(DTYPES[x]) for _ in range(2))
    weight = (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).to(DTYPES[w])
    for residual in (None, r):
        t, y = _definition(a, residual, weight, float(np.float32(eps)))
        got_y, got_t = ops.rms_norm(a, weight, eps, residual=residual)
        _assert_rounded(got_y, y, "y")
        if residual is not None:
            _assert_rounded(got_t, t, "t")
        for fmt in FORMATS:
            codes, scales, y2, t2 = ops.rms_norm_quant(a, weight, eps, residual=residual, fmt=fmt, want_y=True)
            _assert_codes(codes, scales, y, fmt)
            assert torch.equal(y2, got_y) and (residual is None or torch.equal(t2, got_t))
