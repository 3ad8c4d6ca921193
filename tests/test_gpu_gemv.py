"""MXFP4 weights times a few rows of 16- and 32-bit activations, against 64 bits; exactly where every sum fits fp32."""
import math

import numpy as np
import pytest
import torch

from catccos_amd import ops
from oracle import mx_oracle as O
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def weights(n, k, seed, lo=100, hi=130):
    """Random codes and scale bytes from [lo, hi)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    nb = k // 32
    scales = torch.full((n, nb + nb % 2), 127, dtype=torch.uint8, device="cuda")
    scales[:, :nb] = torch.randint(lo, hi, (n, nb), generator=g, device="cuda").to(torch.uint8)
    return torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, generator=g, device="cuda"), scales


def dequantized(codes, scales):
    n, half = codes.shape
    v = torch.tensor(E2M1, dtype=torch.float64, device="cuda")[torch.stack((codes & 15, codes >> 4), dim=2).flatten(1).long()]
    return v * torch.exp2(scales[:, : half // 16].double() - 127).repeat_interleave(32, dim=1)


def check(got, x, w):
    """Products are exact.  A matrix instruction adds 32 of them to its sum, losing at most 2^-22 of the magnitudes it adds; a result passes k / 32
    instructions for each piece (1, 2 or 3) of an activation and the sums of 16 wavefronts; then one rounding to got's type, to half its spacing where it
    is subnormal."""
    pieces = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[x.dtype]
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    info = torch.finfo(got.dtype)
    bound = size * (pieces * x.shape[1] / 32 + 16) * 2.0 ** -22 + want.abs() * (info.eps / 2) + info.smallest_normal * info.eps
    fits = want.abs() < info.max * (1 - info.eps)
    err = (got.double() - want).abs()
    assert bool((err <= bound)[fits].all()), float((err / bound)[fits].max())


@pytest.mark.parametrize("k", [32, 64, 96, 128, 160, 256, 288, 512, 960, 1024, 2080, 4096, 7168, 16384])
@pytest.mark.parametrize("x,out", [("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32"), ("bf16", "fp32"), ("fp32", "bf16")])
def test_every_length_of_k(k, x, out):
    for n in (1, 15, 100):
        w, s = weights(n, k, k + n)
        wide = dequantized(w, s)
        for m in (1, 2, 5):
            a = torch.randn((m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(m)).to(DTYPES[x])
            got = ops.mxfp4_gemv(a, w, s, out)
            assert got.shape == (m, n) and got.dtype == DTYPES[out]
            check(got, a, wide)


@pytest.mark.parametrize("k", [32, 96, 544, 2080, 5120])
@pytest.mark.parametrize("x,out", [("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32")])
def test_every_length_of_k_under_many_rows(k, x, out):
    """Enough weight rows for two tiles of them to a workgroup, the last one in part."""
    w, s = weights(8209, k, k)
    wide = dequantized(w, s)
    for m in (5, 9, 20):
        a = torch.randn((m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(m)).to(DTYPES[x])
        check(ops.mxfp4_gemv(a, w, s, out), a, wide)


@pytest.mark.parametrize("n,k", [(5, 4128), (130, 15616), (700, 4640), (2000, 5152)])
@pytest.mark.parametrize("x,out", [("bf16", "fp32"), ("fp16", "fp32"), ("fp32", "fp32")])
def test_long_rows_of_few_weights(n, k, x, out):
    """K long and weight rows few: the rows of x are spread over more workgroups, one or a few to each."""
    w, s = weights(n, k, k)
    wide = dequantized(w, s)
    for m in (1, 3, 7, 8, 12, 33):
        a = torch.randn((m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(m)).to(DTYPES[x])
        check(ops.mxfp4_gemv(a, w, s, out), a, wide)


@pytest.mark.parametrize("n", [1, 2, 3, 16, 17, 31, 33, 1000, 4096, 4099, 20000])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 7, 8, 15, 16, 17, 31, 33, 48, 64, 65, 130])
def test_whole_numbers_are_exact(m, n):
    """Small whole activations and scales from 2^0 to 2^3: every sum is a multiple of 1/2 below 2^22, so fp32 results are exact and 16-bit ones correctly
    rounded, whatever the order of the sums."""
    g = torch.Generator(device="cuda").manual_seed(m * n)
    for k, x in ((416, "bf16"), (1056, "fp16"), (640, "fp32")):
        w, s = weights(n, k, n, 127, 131)
        a = torch.randint(-16, 17, (m, k), generator=g, device="cuda").to(DTYPES[x])
        want = a.double() @ dequantized(w, s).t()
        for out in DTYPES:
            assert torch.equal(ops.mxfp4_gemv(a, w, s, out), want.to(DTYPES[out])), (k, x, out)


def test_every_code_under_every_scale():
    """One activation of one: each code times each scale byte, NaN for 255 and Inf past fp32."""
    codes = torch.arange(16, device="cuda", dtype=torch.uint8)
    row = (codes | (codes << 4)).view(1, 16)                             # columns 2 c and 2 c + 1 hold code c
    w, s = row.expand(256, 16).contiguous(), torch.arange(256, device="cuda", dtype=torch.int32).to(torch.uint8).view(256, 1)
    x = torch.eye(32, device="cuda")
    want = dequantized(w, s).float().t()                                  # [32, 256]
    want[:, 255] = math.nan
    for dtype in DTYPES.values():
        got = ops.mxfp4_gemv(x.to(dtype), w, s, "fp32")
        nan = torch.isnan(got)
        # 6 * 2^126 and larger overflow, and the zeros of the other columns then give 0 * Inf
        finite = want.abs().amax(dim=0) < math.inf
        assert torch.equal(got[:, finite], want[:, finite]), (got[:, finite] != want[:, finite]).nonzero()[:8].tolist()
        assert bool(nan[:, 255].all())


def test_activations_are_taken_exactly():
    """Every bf16 and fp16 value, and fp32 values of every exponent, times one: the value itself comes back in fp32."""
    w = torch.zeros((32, 16), dtype=torch.uint8, device="cuda")
    w[torch.arange(32), torch.arange(32) // 2] = torch.tensor([2, 32], dtype=torch.uint8, device="cuda").repeat(16)      # code 1.0 on the diagonal
    s = torch.full((32, 2), 127, dtype=torch.uint8, device="cuda")
    every = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16)
    for dtype in (torch.bfloat16, torch.float16):
        x = every.view(dtype)
        x = x[torch.isfinite(x)].view(-1, 32)
        assert torch.equal(ops.mxfp4_gemv(x, w, s, "fp32"), x.float())
    g = torch.Generator(device="cuda").manual_seed(0)
    bits = torch.randint(-2 ** 31, 2 ** 31, (64000, 32), generator=g, device="cuda").to(torch.int32).view(torch.float32)
    x = torch.where(torch.isfinite(bits), bits, 1.0)
    got = ops.mxfp4_gemv(x, w, s, "fp32")
    # three pieces of eight bits: what lies below the smallest bf16 number (2^-133) is lost
    assert bool(((got - x).abs().double() <= 2.0 ** -133).all()), ((got - x).abs() / x.abs()).max()


def test_non_finite_activations():
    w, s = weights(64, 256, 1)
    wide = dequantized(w, s)
    for dtype in DTYPES.values():
        x = torch.randn((3, 256), device="cuda").to(dtype)
        x[1, 77] = math.inf
        x[2, 78] = math.nan
        got = ops.mxfp4_gemv(x, w, s, "fp32")
        check(got[:1], x[:1], wide)
        at = wide[:, 77]
        assert bool(torch.isnan(got[1, at == 0]).all()) and bool((got[1, at > 0] == math.inf).all()) and bool((got[1, at < 0] == -math.inf).all())
        assert bool(torch.isnan(got[2]).all())


def test_the_quantizers_weights():
    """Codes and scales as mx_quant writes them for a weight."""
    rng = np.random.default_rng(3)
    wq, ws = O.mx_quant(O.bf16_round(rng.standard_normal((200, 96)).astype(np.float32) * 0.05), "E2M1", "lut")
    x = torch.randn((5, 96), device="cuda").to(torch.bfloat16)
    w, s = ops.mx_quant(dev(O.f32_to_bf16_bits(O.mx_dequant(wq, ws, "E2M1"))).view(torch.bfloat16), "E2M1")
    assert s.shape == (200, 4)                                            # three blocks, padded to four
    check(ops.mxfp4_gemv(x, w, s, "fp32"), x, torch.from_numpy(O.mx_dequant(wq, ws, "E2M1").astype(np.float64)).cuda())


def test_strides_and_the_bytes_between_rows():
    from catccos_amd import _lib
    m, n, k = 9, 77, 288
    w, s = weights(n, k + 32, 5)
    a = torch.randn((m, k + 3), device="cuda").to(torch.bfloat16)
    want = ops.mxfp4_gemv(a[:, 1:k + 1].contiguous(), w[:, :k // 2].contiguous(), s[:, :k // 32].contiguous(), "bf16")
    assert torch.equal(ops.mxfp4_gemv(a[:, 1:k + 1], w[:, :k // 2], s, "bf16"), want)
    assert torch.equal(ops.mxfp4_gemv(a[::2, 1:k + 1], w[::3, :k // 2], s[::3], "bf16"), want[::2, ::3])
    for pad in (1, 3, 8):
        out = torch.full((m, n + pad), 7.0, dtype=torch.bfloat16, device="cuda")
        _lib.check(_lib.load().cmx_mxfp4_gemv(a.data_ptr() + 2, k + 3, 0, w.data_ptr(), w.stride(0), s.data_ptr(), s.stride(0), out.data_ptr(), n + pad, 0, m, n, k,
                                              torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out[:, :n], want) and bool((out[:, n:] == 7).all())
    assert ops.mxfp4_gemv(a[:0, :k], w[:, :k // 2], s).shape == (0, n)


def test_weights_past_32_bits():
    n, k, apart = 20, 512, (1 << 32) - 16
    w, s = weights(n, k, 6)
    buf = torch.empty(2 * apart + k // 2, dtype=torch.uint8, device="cuda")
    far = buf.as_strided((3, k // 2), (apart, 1))
    far.copy_(w[:3])
    x = torch.randn((4, k), device="cuda").to(torch.bfloat16)
    assert torch.equal(ops.mxfp4_gemv(x, far, s[:3]), ops.mxfp4_gemv(x, w, s)[:, :3])


def test_on_a_side_stream_and_captured():
    ops.init()
    w, s = weights(1000, 2048, 8)
    x = torch.randn((20, 2048), device="cuda").to(torch.bfloat16)
    want = ops.mxfp4_gemv(x, w, s), ops.mxfp4_gemv(x[:3], w, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.mxfp4_gemv(x, w, s), ops.mxfp4_gemv(x[:3], w, s)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.mxfp4_gemv(x, w, s), ops.mxfp4_gemv(x[:3], w, s)
    for rep in range(3):
        x.copy_(torch.randn(x.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], ops.mxfp4_gemv(x, w, s)) and torch.equal(out[1], ops.mxfp4_gemv(x[:3], w, s)), rep
