"""FP8 products in the kernels and lengths of K that test_gpu_fp8_block's sizes leave out: groups in tiles of 32 x 64, and in each kind of tile K over two changes of the span
whose scales lie in LDS (8 blocks of 128, 4 with a scale for every row of b).  test_fp8_ways holds which kernel each size takes."""
import pytest
import torch

from tests.test_gpu_fp8_block import DTYPES, _dequantized, _exact_operand, _groups

pytestmark = pytest.mark.gpu

DENSE = [(1300, 4100, 2192), (4096, 4096, 2064), (97, 4103, 2064), (250, 4100, 2320)]
GROUPED = [([33, 0, 700, 1, 190, 64], 520, 528), ([300, 1, 0, 513, 128], 1030, 2192), ([100, 7, 130, 0, 260, 61, 64, 65], 2060, 2192), ([300, 1, 0, 513, 128], 4090, 2192),
           ([1000, 0, 30, 400], 8200, 2192), ([4, 6, 0, 9] * 16, 1000, 2192), ([20, 30, 0, 90, 70] * 4, 1000, 2192)]


@pytest.mark.parametrize("m,n,k", DENSE)
@pytest.mark.parametrize("b_rows", [128, 1])
@pytest.mark.parametrize("fmt", ["E4M3", "E5M2"])
def test_gemm_of_exact_sums(m, n, k, b_rows, fmt):
    from catccos_amd import ops
    g = torch.Generator(device="cuda").manual_seed(m + 3 * n + 5 * k)
    (a, sa), (b, sb) = _exact_operand(g, m, k, 1, fmt), _exact_operand(g, n, k, b_rows, fmt)
    want = _dequantized(a, sa, 1, fmt) @ _dequantized(b, sb, b_rows, fmt).t()
    assert torch.equal(ops.fp8_block_gemm(a, sa, b, sb, fmt, "fp32").double(), want)
    for out in ("bf16", "fp16"):
        assert torch.equal(ops.fp8_block_gemm(a, sa, b, sb, fmt, out), want.float().to(DTYPES[out]))


@pytest.mark.parametrize("sizes,n,k", GROUPED)
@pytest.mark.parametrize("fmt", ["E4M3", "E5M2"])
def test_gmm_of_exact_sums(sizes, n, k, fmt):
    from catccos_amd import ops
    for extra in (0, 37):
        a, sa, b, sb, counts, want = _groups(sizes, n, k, len(sizes) + n, fmt, extra)
        assert torch.equal(ops.fp8_block_gmm(a, sa, b, sb, counts, fmt, "fp32").double(), want)
        c = torch.full((a.shape[0], n + 3), 7.0, dtype=torch.float16, device="cuda")
        ops.fp8_block_gmm(a, sa, b, sb, counts, fmt, "fp16", c=c[:, :n])
        m = a.shape[0] - extra
        assert torch.equal(c[:m, :n], want[:m].float().to(torch.float16)) and bool((c[m:] == 7.0).all()) and bool((c[:, n:] == 7.0).all())
