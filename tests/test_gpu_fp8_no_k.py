"""FP8 products over no K at all, as the weight's gradient of an expert without rows is one: sums of nothing, zeros."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _nothing(rows, cols, square=False):
    from catccos_amd import ops
    return ops.fp8_block_quant(torch.empty((0, rows), dtype=torch.bfloat16, device="cuda"), square=square, transposed=True)


@pytest.mark.parametrize("m,n", [(1, 1), (5, 130), (300, 7), (0, 8), (8, 0)])
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("out", ["bf16", "fp16", "fp32"])
def test_gemm(m, n, square, out):
    from catccos_amd import ops
    a, b = _nothing(m, 0), _nothing(n, 0, square)
    assert a[0].shape == (m, 0) and b[0].shape == (n, 0)
    got = ops.fp8_block_gemm(*a, *b, out=out)
    assert got.shape == (m, n) and got.dtype == DTYPES[out] and not bool(got.any())
    around = torch.full((m + 2, n + 5), 7.0, dtype=DTYPES[out], device="cuda")
    c = around[1:m + 1, 3:n + 3]
    assert ops.fp8_block_gemm(*a, *b, out=out, c=c) is c and not bool(c.any())
    c.fill_(7.0)
    assert bool((around == 7.0).all())


@pytest.mark.parametrize("sizes,extra", [([3, 0, 4], 0), ([3, -2, 4], 9), ([0, 0], 5), ([100, 2 ** 31 - 1], 0), ([], 4)])
@pytest.mark.parametrize("out", ["bf16", "fp32"])
def test_gmm(sizes, extra, out):
    from catccos_amd import ops
    rows = min(sum(max(0, s) for s in sizes), 107)
    m, n, g = rows + extra, 130, len(sizes)
    u, f = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda"), lambda *s: torch.zeros(s, device="cuda")
    call = (u(m, 0), f(m, 0), u(g, n, 0), f(g, 2, 0), torch.tensor(sizes, dtype=torch.int32, device="cuda"))
    got = ops.fp8_block_gmm(*call, out=out)
    assert got.shape == (m, n) and got.dtype == DTYPES[out] and not bool(got.any())
    around = torch.full((m + 1, n + 3), 7.0, dtype=DTYPES[out], device="cuda")
    c = around[:m, 1:n + 1]
    assert ops.fp8_block_gmm(*call, out=out, c=c) is c
    assert not bool(c[:rows].any()) and bool((c[rows:] == 7.0).all())         # rows behind the groups stay
    c.fill_(7.0)
    assert bool((around == 7.0).all())


def test_what_is_refused_stays_refused():
    from catccos_amd import ops
    a, b = _nothing(4, 0), _nothing(8, 0)
    with pytest.raises(ValueError, match="E4M3 or E5M2"):
        ops.fp8_block_gemm(*a, *b, fmt="E2M1")
    with pytest.raises(KeyError):
        ops.fp8_block_gemm(*a, *b, out="int8")
    with pytest.raises(AssertionError):
        ops.fp8_block_gemm(*a, *b, c=torch.zeros((4, 9), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(AssertionError):
        ops.fp8_block_gemm(a[0], a[1][:3], *b)


def test_the_weight_gradients_of_all_experts():
    """One of them has no rows; captured and replayed too."""
    from catccos_amd import ops
    ops.init()
    g = torch.Generator(device="cuda").manual_seed(5)
    n, h, counts = 136, 272, [40, 0, 3, 0, 130]
    dy, x = (torch.randn((sum(counts), c), generator=g, device="cuda").to(torch.bfloat16) for c in (n, h))
    dw = torch.full((len(counts), n, h), float("nan"), device="cuda")

    def gradients():
        at = 0
        for e, rows in enumerate(counts):
            mine = slice(at, at + rows)
            ops.fp8_block_gemm(*ops.fp8_block_quant(dy[mine], transposed=True), *ops.fp8_block_quant(x[mine], transposed=True), out="fp32", c=dw[e])
            at += rows

    gradients()
    at = 0
    for e, rows in enumerate(counts):
        want = dy[at:at + rows].double().t() @ x[at:at + rows].double()
        # codes are half a step off at most, 2^-4 of themselves, spread evenly: 2^-4 / sqrt(3), and sqrt(2) as much for a product of two
        assert torch.equal(dw[e], torch.zeros_like(dw[e])) if rows == 0 else float((dw[e].double() - want).norm() / want.norm()) < 2.0 ** -4
        at += rows
    first = dw.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        gradients()
    for _ in range(3):
        dw.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dw, first)
