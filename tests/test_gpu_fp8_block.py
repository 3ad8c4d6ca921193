"""FP8 with an fp32 scale for each block of 128: the quantiser bit for bit, the products exactly where their sums are exact and within derived bounds else."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8 = {"E4M3": torch.float8_e4m3fn, "E5M2": torch.float8_e5m2}
FORMATS = {"E4M3": (3, -6, 448.0), "E5M2": (2, -14, 57344.0)}
LEAST = 2.0 ** -126


def _blocks(z, square):
    """Largest magnitude of each block of z (fp64, 2-D)."""
    rows, cols = z.shape
    h, nb = 128 if square else 1, -(-cols // 128)
    nr = -(-rows // h)
    v = torch.nn.functional.pad(z.abs(), (0, nb * 128 - cols, 0, nr * h - rows)).view(nr, h, nb, 128)
    return v.amax(dim=(1, 3))


def _definition(x, fmt, square, transposed, pow2):
    """(values of the codes fp64 [R, C16], scales fp64) of finite x."""
    mantissa, least, most = FORMATS[fmt]
    z = x.double()
    z = z.t().contiguous() if transposed else z
    rows, cols = z.shape
    scale = (_blocks(z, square) / most).float().double()
    if pow2:
        exact = _blocks(z, square) / most
        e = torch.floor(torch.log2(exact.clamp_min(1e-300)))
        e = torch.where(torch.exp2(e) < exact, e + 1, e)
        scale = torch.exp2(e)
    scale = scale.clamp_min(LEAST)
    wide = scale.repeat_interleave(128, dim=1)[:, :cols]
    if square:
        wide = wide.repeat_interleave(128, dim=0)[:rows]
    q = z / wide                                              # (64 bits: 2^-29 above what a border of 5 bits and a scale of 24 can be missed by)
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(q.abs().clamp_min(1e-300))), min=least) - mantissa)
    values = torch.zeros((rows, -(-cols // 16) * 16), dtype=torch.float64, device=x.device)
    values[:, :cols] = (torch.round(q / step) * step).clamp(-most, most)
    return values, scale


def _check_quant(x, fmt, square, transposed, pow2):
    from catccos_amd import ops
    codes, scales = ops.fp8_block_quant(x, fmt, square, transposed, pow2)
    for i in range(x.shape[0] if x.dim() == 3 else 1):
        want, want_scale = _definition(x[i] if x.dim() == 3 else x, fmt, square, transposed, pow2)
        c, s = (codes[i], scales[i]) if x.dim() == 3 else (codes, scales)
        assert torch.equal(s.double(), want_scale)
        assert torch.equal(c.view(FP8[fmt]).double(), want)


@pytest.mark.parametrize("square,transposed", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("rows,cols,x,fmt", [(1, 1, "bf16", "E4M3"), (1, 7168, "bf16", "E4M3"), (3, 127, "fp16", "E5M2"), (5, 1000, "bf16", "E4M3"), (129, 136, "fp32", "E4M3"),
                                             (128, 128, "bf16", "E5M2"), (777, 1000, "fp16", "E4M3"), (300, 2049, "fp32", "E5M2"), (17, 4112, "bf16", "E4M3")])
def test_quant_is_the_definition(rows, cols, x, fmt, square, transposed):
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + cols)
    v = torch.randn((rows, cols), generator=g, device="cuda") * torch.exp(2 * torch.randn((rows, 1), generator=g, device="cuda"))
    for pow2 in (False, True):
        _check_quant(v.to(DTYPES[x]), fmt, square, transposed, pow2)


@pytest.mark.parametrize("fmt", ["E4M3", "E5M2"])
@pytest.mark.parametrize("pow2", [False, True])
def test_quant_next_to_borders(fmt, pow2):
    """fp32 values one unit of the last place to either side of every border times the scale, and on it where it is a number."""
    mantissa, least, most = FORMATS[fmt]
    values = torch.arange(127 if fmt == "E4M3" else 124, dtype=torch.uint8).view(FP8[fmt]).double()
    borders = (values[1:] + values[:-1]) / 2
    for amax in (448.0, 1.0, 3.1415926, 0.3333333, 7.0, 1e-3, 1.7e20, 2.9e-34):
        s = torch.tensor(amax, dtype=torch.float32).double() / most
        s = torch.exp2(torch.ceil(torch.log2(s))) if pow2 else s.float().double()
        near = (borders * s).float()
        v = torch.cat([near, torch.nextafter(near, torch.full_like(near, torch.inf)), torch.nextafter(near, torch.zeros_like(near))])
        v = torch.cat([v, -v])
        rows = -(-v.numel() // 127)
        x = torch.zeros((rows, 128))
        x[:, 1:].reshape(-1)[:] = 0
        flat = torch.zeros(rows * 127)
        flat[:v.numel()] = v
        x[:, 1:] = flat.view(rows, 127).clamp(-amax, amax)
        x[:, 0] = amax
        _check_quant(x.cuda(), fmt, False, False, pow2)
        _check_quant(x.cuda(), fmt, False, True, pow2)


@pytest.mark.parametrize("x,values", [("fp32", (0.0, 1e-45, 1e-38, 3e38)), ("bf16", (0.0, 9e-41, 3e38)), ("fp16", (0.0, 6e-8, 65504.0))])
def test_quant_of_the_smallest_and_largest_blocks(x, values):
    for v in values:
        t = torch.full((4, 300), v, dtype=DTYPES[x], device="cuda")
        t[1, 5:200:7] = 0
        t[2] = -t[2]
        for square in (False, True):
            for pow2 in (False, True):
                _check_quant(t, "E4M3", square, square, pow2)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("square,transposed", [(False, False), (False, True), (True, False), (True, True)])
def test_quant_of_a_block_that_is_not_finite(bad, square, transposed):
    from catccos_amd import ops
    x = torch.randn((200, 300), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    clean, clean_scales = ops.fp8_block_quant(x, "E4M3", square, transposed)
    x[150, 290] = bad
    codes, scales = ops.fp8_block_quant(x, "E4M3", square, transposed)
    r, c = (290, 150) if transposed else (150, 290)
    br = slice(r // 128 * 128, r // 128 * 128 + 128) if square else slice(r, r + 1)
    live = torch.zeros_like(codes, dtype=torch.bool)
    live[br, c // 128 * 128:c // 128 * 128 + 128] = True
    live[:, 200 if transposed else 300:] = False                               # the zeros behind a row
    assert bool((codes[live] == 0x7F).all()) and torch.equal(codes[~live], clean[~live])
    hit = scales[r // 128 if square else r, c // 128]
    assert bool(torch.isnan(hit)) if bad != bad else float(hit) == float("inf")
    other = torch.ones_like(scales, dtype=torch.bool)
    other[r // 128 if square else r, c // 128] = False
    assert torch.equal(scales[other], clean_scales[other])


def test_quant_of_strided_and_batched_matrices():
    from catccos_amd import ops
    big = torch.randn((3, 140, 1040), device="cuda").to(torch.bfloat16)
    for view in (big[1, :, :1000], big[1, :, 3:900], big[0, ::2, :130], big[:, :, 5:700], big[:, :130], big.view(3, 140 * 1040)[:, :999]):
        for square, transposed in ((False, False), (False, True), (True, False), (True, True)):
            _check_quant(view, "E4M3", square, transposed, False)
    codes, scales = ops.fp8_block_quant(big[:0], square=True)
    assert codes.shape == (0, 140, 1040) and scales.shape == (0, 2, 9)


def test_square_blocks_are_the_same_both_ways():
    from catccos_amd import ops
    w = torch.randn((384, 512), device="cuda").to(torch.bfloat16)
    codes, scales = ops.fp8_block_quant(w, square=True)
    codes_t, scales_t = ops.fp8_block_quant(w, square=True, transposed=True)
    assert torch.equal(codes.t(), codes_t) and torch.equal(scales.t(), scales_t)


# ------------------------------------------------------------------------------------------------ products
def _exact_operand(g, rows, k, scale_rows, fmt):
    """Codes of -2 .. 2 and scales of powers of two: products and sums are whole multiples of one power of two, within 24 bits up to k = 2^16."""
    v = torch.randint(-2, 3, (rows, k), generator=g, device="cuda").float()
    s = torch.exp2(torch.randint(-2, 3, (-(-rows // scale_rows), -(-k // 128)), generator=g, device="cuda").float())
    return v.to(FP8[fmt]).view(torch.uint8), s


def _operand(g, rows, k, scale_rows, fmt):
    """Codes of normal values, scales that are no powers of two."""
    v = torch.randn((rows, k), generator=g, device="cuda") * (120 if fmt == "E4M3" else 15000)
    s = torch.rand((-(-rows // scale_rows), -(-k // 128)), generator=g, device="cuda") * 0.01 + 0.001
    return v.clamp(-FORMATS[fmt][2], FORMATS[fmt][2]).to(FP8[fmt]).view(torch.uint8), s


def _dequantized(codes, s, scale_rows, fmt):
    wide = s.double().repeat_interleave(128, dim=1)[:, :codes.shape[1]].repeat_interleave(scale_rows, dim=0)[:codes.shape[0]]
    return codes.view(FP8[fmt]).double() * wide


# (few rows, one round of small tiles, large tiles; the last column and row of tiles ragged, K that ends in a block and in a piece of it)
SHAPES = [(1, 1, 16), (1, 130, 128), (1, 4096, 1040), (2, 7, 112), (7, 64, 144), (15, 1000, 1024), (16, 257, 2064), (17, 128, 128), (33, 300, 400), (63, 72, 16), (64, 512, 1152), (65, 129, 272),
          (100, 1000, 1040), (128, 128, 128), (129, 256, 2048), (300, 999, 144), (1000, 1030, 528), (2049, 520, 1168), (4101, 4105, 272), (4352, 4096, 1296)]


# sizes that take each of the kernels (few rows in tiles of 16 x 16 to 64 x 32, tiles of 128 x 128 to 256 x 256, K in parts), ragged in each axis
WAYS = [(300, 999, 144), (30, 4100, 1040), (64, 4100, 1168), (100, 4104, 912), (90, 16388, 2064), (250, 4100, 7184), (66, 16380, 7184), (1400, 4100, 1040), (5000, 4100, 1168), (4000, 4090, 2064)]


@pytest.mark.parametrize("m,n,k", SHAPES + WAYS)
@pytest.mark.parametrize("b_rows", [128, 1])
@pytest.mark.parametrize("fmt", ["E4M3", "E5M2"])
def test_gemm_of_exact_sums(m, n, k, b_rows, fmt):
    from catccos_amd import ops
    g = torch.Generator(device="cuda").manual_seed(m + 3 * n + 5 * k)
    (a, sa), (b, sb) = _exact_operand(g, m, k, 1, fmt), _exact_operand(g, n, k, b_rows, fmt)
    want = _dequantized(a, sa, 1, fmt) @ _dequantized(b, sb, b_rows, fmt).t()
    got = ops.fp8_block_gemm(a, sa, b, sb, fmt, "fp32")
    assert torch.equal(got.double(), want)
    for out in ("bf16", "fp16"):
        assert torch.equal(ops.fp8_block_gemm(a, sa, b, sb, fmt, out), want.float().to(DTYPES[out]))


@pytest.mark.parametrize("m,n,k", [(1, 4096, 7168), (5, 256, 4096), (40, 512, 1040), (64, 1000, 2048), (129, 300, 1168), (1000, 777, 784), (4101, 4105, 272), (4352, 4096, 1296)])
@pytest.mark.parametrize("b_rows", [128, 1])
@pytest.mark.parametrize("fmt,out", [("E4M3", "bf16"), ("E4M3", "fp32"), ("E5M2", "fp16")])
def test_gemm_within_the_derived_bound(m, n, k, b_rows, fmt, out):
    from catccos_amd import ops
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    (a, sa), (b, sb) = _operand(g, m, k, 1, fmt), _operand(g, n, k, b_rows, fmt)
    if out == "fp16":
        sa, sb = sa * 2.0 ** -12, sb * 2.0 ** -8                               # (within fp16's range)
    da, db = _dequantized(a, sa, 1, fmt), _dequantized(b, sb, b_rows, fmt)
    want, absolute = da @ db.t(), da.abs() @ db.abs().t()
    got = ops.fp8_block_gemm(a, sa, b, sb, fmt, out).double()
    # eight products aligned to the largest of them lose up to 2^-13 of it each: 2^-10 of their sum of magnitudes; 16 such sums a block, then a
    # multiply-add a block and the product of the scales, 2^-23 each at most
    loss = 2.0 ** -10 + (-(-k // 128) + 20) * 2.0 ** -23
    eps = torch.finfo(DTYPES[out]).eps / 2 if out != "fp32" else 0.0
    assert bool(((got - want).abs() <= absolute * loss + want.abs() * eps * 1.01 + 1e-7).all())
    # as a whole: what a product loses lies between 0 and 2^-13 of the largest of eight, which of normal values is some 2.5 times their root mean square, and
    # carries the product's sign, so losses add up like the products do: 2.5 / sqrt(3) * 2^-13 of the result
    assert float((got - want).norm() / want.norm()) <= 2.0 ** -12 + eps


def test_gemm_takes_rows_anywhere():
    """Operands, scales and result as parts of larger tensors, what lies around them NaN or kept."""
    from catccos_amd import ops
    g = torch.Generator(device="cuda").manual_seed(8)
    for m, n, k in ((3, 40, 144), (70, 200, 272), (300, 300, 400), (4100, 4100, 144)):
        (a, sa), (b, sb) = _exact_operand(g, m, k, 1, "E4M3"), _exact_operand(g, n, k, 128, "E4M3")
        big = [torch.full((r + 2, c + 32), 0x7F, dtype=torch.uint8, device="cuda") for r, c in (a.shape, b.shape)]
        scale = [torch.full((r + 2, c + 3), float("nan"), device="cuda") for r, c in (sa.shape, sb.shape)]
        va, vb = big[0][1:m + 1, 16:16 + k], big[1][1:n + 1, 16:16 + k]
        vsa, vsb = scale[0][1:-1, 1:sa.shape[1] + 2], scale[1][1:-1, 1:sb.shape[1] + 2]
        va.copy_(a)
        vb.copy_(b)
        vsa[:, :-1], vsb[:, :-1] = sa, sb
        c = torch.full((m + 2, n + 5), 7.0, dtype=torch.bfloat16, device="cuda")
        want = ops.fp8_block_gemm(a, sa, b, sb)
        assert ops.fp8_block_gemm(va, vsa, vb, vsb, c=c[1:m + 1, 3:n + 3]).data_ptr() == c[1:, 3:].data_ptr()
        assert torch.equal(c[1:m + 1, 3:n + 3], want)
        c[1:m + 1, 3:n + 3] = 7.0
        assert bool((c == 7.0).all())


@pytest.mark.parametrize("m,n", [(1, 256), (40, 256), (200, 256), (4352, 4096)])
def test_gemm_keeps_what_is_not_finite_in_its_place(m, n):
    from catccos_amd import ops
    g = torch.Generator(device="cuda").manual_seed(4)
    (a, sa), (b, sb) = _exact_operand(g, m, 256, 1, "E4M3"), _exact_operand(g, n, 256, 128, "E4M3")
    want = ops.fp8_block_gemm(a, sa, b, sb, out="fp32")
    a[m - 1, 200] = 0x7F
    sb[1, 0] = float("nan")
    got = ops.fp8_block_gemm(a, sa, b, sb, out="fp32")
    nan = torch.zeros_like(want, dtype=torch.bool)
    nan[m - 1] = True
    nan[:, 128:256] = True
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want[~nan])
    sa[0, 1] = 3e38                                                            # a sum past fp32 is Inf
    sb[1, 0] = 1.0
    sb[:, 1] = 3e38
    got = ops.fp8_block_gemm(a, sa, b, sb, out="bf16")
    assert not bool(torch.isfinite(got[0]).any()) if m == 1 else bool(torch.isinf(got[0]).any())


def _groups(sizes, n, k, seed, fmt="E4M3", extra=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m = max(0, sum(max(0, s) for s in sizes)) + extra
    a, sa = _exact_operand(g, m, k, 1, fmt)
    b = torch.empty((len(sizes), n, k), dtype=torch.uint8, device="cuda")
    sb = torch.empty((len(sizes), -(-n // 128), -(-k // 128)), device="cuda")
    want = torch.zeros((m, n), dtype=torch.float64, device="cuda")
    at = 0
    for i, s in enumerate(sizes):
        b[i], sb[i] = _exact_operand(g, n, k, 128, fmt)
        s = max(0, s)
        want[at:at + s] = _dequantized(a[at:at + s], sa[at:at + s], 1, fmt) @ _dequantized(b[i], sb[i], 128, fmt).t()
        at += s
    return a, sa, b, sb, torch.tensor(sizes, dtype=torch.int32, device="cuda"), want


MANY = [0] * 300 + [3, 0, 17, 1] * 20 + [0, 40] + [0] * 200 + [5]
GROUPS = [([1], 64, 128), ([0, 0, 1, 0], 130, 144), ([3, 0, 16, 17, 1], 200, 272), ([33, 64, 0, 5], 129, 1040), ([100, 0, 200, 70], 256, 400), ([300, 1, 0, 513, 128], 384, 528), (MANY, 40, 144),
          ([2100, 0, 2500, 1], 4100, 144), ([1] * 256, 136, 256), ([0, 0, 0], 64, 128), ([5, -3, 9], 64, 128), ([4, 6, 0, 9] * 16, 8200, 272), ([100, 130, 0, 128] * 2, 2060, 400),
          ([2500, 10, 300, 0, 200], 4090, 2064)]


@pytest.mark.parametrize("sizes,n,k", GROUPS)
@pytest.mark.parametrize("fmt", ["E4M3", "E5M2"])
def test_gmm_of_exact_sums(sizes, n, k, fmt):
    from catccos_amd import ops
    for extra in (0, 37):
        a, sa, b, sb, counts, want = _groups(sizes, n, k, len(sizes) + n, fmt, extra)
        got = ops.fp8_block_gmm(a, sa, b, sb, counts, fmt, "fp32")
        assert torch.equal(got.double(), want)                                 # (zeros behind the groups)
        assert torch.equal(ops.fp8_block_gmm(a, sa, b, sb, counts, fmt), want.float().to(torch.bfloat16))
        c = torch.full((a.shape[0], n + 3), 7.0, dtype=torch.float16, device="cuda")
        ops.fp8_block_gmm(a, sa, b, sb, counts, fmt, "fp16", c=c[:, :n])
        m = a.shape[0] - extra
        assert torch.equal(c[:m, :n], want[:m].float().to(torch.float16)) and bool((c[m:] == 7.0).all()) and bool((c[:, n:] == 7.0).all())


def test_gmm_of_sizes_that_add_up_to_more_than_there_are():
    from catccos_amd import ops
    a, sa, b, sb, counts, want = _groups([20, 30, 10], 72, 256, 5)
    a, sa = a[:35].contiguous(), sa[:35].contiguous()
    assert torch.equal(ops.fp8_block_gmm(a, sa, b, sb, counts, out="fp32").double(), want[:35])
    counts[1] = 2 ** 31 - 1
    counts[2] = 2 ** 31 - 1
    assert torch.equal(ops.fp8_block_gmm(a, sa, b, sb, counts, out="fp32").double(), want[:35])


def test_products_of_nothing():
    from catccos_amd import ops
    u, f = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda"), lambda *s: torch.ones(s, device="cuda")
    assert ops.fp8_block_gemm(u(0, 128), f(0, 1), u(8, 128), f(1, 1)).shape == (0, 8) and ops.fp8_block_gemm(u(5, 128), f(5, 1), u(0, 128), f(0, 1)).shape == (5, 0)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert not bool(ops.fp8_block_gmm(u(5, 128), f(5, 1), u(0, 8, 128), f(0, 1, 1), none).any())
    c = torch.full((5, 8), 7.0, dtype=torch.bfloat16, device="cuda")
    assert bool((ops.fp8_block_gmm(u(5, 128), f(5, 1), u(0, 8, 128), f(0, 1, 1), none, c=c) == 7).all())
    assert ops.fp8_block_gmm(u(0, 128), f(0, 1), u(2, 8, 128), f(2, 1, 1), torch.zeros(2, dtype=torch.int32, device="cuda")).shape == (0, 8)


def test_equal_calls_give_equal_bits():
    from catccos_amd import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    for m, n, k in ((1, 512, 7168), (64, 512, 7168), (300, 512, 2048), (4352, 4096, 512)):
        (a, sa), (b, sb) = _operand(g, m, k, 1, "E4M3"), _operand(g, n, k, 128, "E4M3")
        first = ops.fp8_block_gemm(a, sa, b, sb, out="fp32")
        for _ in range(3):
            assert torch.equal(ops.fp8_block_gemm(a, sa, b, sb, out="fp32"), first)
