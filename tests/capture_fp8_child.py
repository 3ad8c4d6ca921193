"""Child process of test_gpu_fp8_chain.test_captured_right_after_init: in a process that has launched none of the library's kernels, cmx_init() alone must be enough to
capture the FP8 quantiser and products with blocks of 128 and the token permutes, each at sizes that take different kernels.  The graph is replayed three times on other
inputs, with eager work in between, and every replay compared bit for bit with eager runs made afterwards.  Prints CAPTURE-OK."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

from catccos_amd import ops                     # noqa: E402

# (few rows to large tiles; the third in parts along K)
PRODUCTS = [(1, 4096, 1024), (60, 4096, 400), (256, 4096, 7168), (1400, 4096, 1040), (4000, 4090, 2064)]


def main() -> int:
    torch.manual_seed(3)
    bf16 = lambda *shape: torch.randn(shape, device="cuda").to(torch.bfloat16)
    a, b = {s: bf16(s[0], s[2]) for s in PRODUCTS}, {s: bf16(s[1], s[2]) for s in PRODUCTS}
    tokens, experts, top_k, h, n = 300, 8, 3, 400, 264
    x, w, dout = bf16(tokens, h), bf16(experts, n, h), bf16(tokens, n)
    idx = torch.randint(0, experts, (tokens, top_k), dtype=torch.int32, device="cuda")
    probs = torch.rand((tokens, top_k), device="cuda")
    inputs = [*a.values(), *b.values(), x, w, dout, probs]

    def run():
        out = []
        for s in PRODUCTS:
            pa, pb, rows = ops.fp8_block_quant(a[s]), ops.fp8_block_quant(b[s], square=True), ops.fp8_block_quant(b[s])
            out += [*pa, *pb, ops.fp8_block_gemm(*pa, *pb), ops.fp8_block_gemm(*pa, *rows, out="fp32"), *ops.fp8_block_quant(a[s], "E5M2", transposed=True, pow2=True)]
        _, to, counts = ops.moe_init_routing(idx, experts)
        rows = ops.moe_token_permute(x, to, top_k)
        y = ops.fp8_block_gmm(*ops.fp8_block_quant(rows), *ops.fp8_block_quant(w, square=True), counts)
        dy, dprobs = ops.moe_token_unpermute_grad(dout, y, to, probs)
        dx = ops.moe_token_permute_grad(ops.fp8_block_gmm(*ops.fp8_block_quant(dy), *ops.fp8_block_quant(w, square=True, transposed=True), counts), to, top_k)
        return out + [rows, y, dy, dprobs, dx]

    ops.init()                                   # the only library call before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for rep in range(3):
        for t in inputs:
            t.copy_(torch.randn(t.shape, device="cuda"))
        idx.copy_(torch.randint(0, experts, idx.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        eager = run()
        torch.cuda.synchronize()
        if not all(torch.equal(p, q) for p, q in zip(captured, eager)):
            print(f"replay {rep} differs from the eager run", flush=True)
            return 1
    print("CAPTURE-OK", flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
