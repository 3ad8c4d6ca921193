"""FP8 products whose parts meet in a workspace: eager calls on two streams beside replays of two graphs, each result compared."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_eager_products_beside_replays():
    from catccos_amd import ops
    ops.init()
    g = torch.Generator(device="cuda").manual_seed(19)
    assert ops.fp8_block_gemm_workspace_bytes(256, 4096, 7168) > 0
    sides = []
    for _ in range(2):
        a, b = (ops.fp8_block_quant(torch.randn((r, 7168), generator=g, device="cuda").to(torch.bfloat16), square=sq) for r, sq in ((256, False), (4096, True)))
        want = ops.fp8_block_gemm(*a, *b, out="fp32")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.fp8_block_gemm(*a, *b, out="fp32")
        sides.append((graph, got, want, torch.cuda.Stream(), a, b))
    for _ in range(3):
        eager = []
        for graph, got, want, stream, a, b in sides:
            got.zero_()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
                eager += [(ops.fp8_block_gemm(*a, *b, out="fp32"), want) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(got, want) for _, got, want, *_ in sides)
        assert all(torch.equal(again, want) for again, want in eager)
