"""Child process of test_gpu_moe_ffn_mxfp4.test_captured_right_after_init: in a process that has launched none of the library's kernels, cmx_init() alone must
be enough to capture norm, gate, matrix-vector product and the FFN of a few tokens, each at sizes that take different kernels.  The graph is replayed twice,
with eager work in between, and every replay compared bit for bit with eager runs made afterwards.  Prints CAPTURE-OK."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

from catccos_amd import ops                     # noqa: E402


def main() -> int:
    torch.manual_seed(3)
    k, n, experts, top_k = 512, 256, 16, 4

    def weights(*shape):
        return (torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), dtype=torch.uint8, device="cuda"),
                torch.full((*shape[:-1], shape[-1] // 32), 120, dtype=torch.uint8, device="cuda"))
    w1, w2, b, wide = weights(experts, n, k), weights(experts, k, n // 2), weights(experts, k), weights(8192, k)
    rows = {t: torch.randn((t, k), device="cuda").to(torch.bfloat16) for t in (1, 5, 40)}
    tall, long = torch.randn((4000, 200), device="cuda"), torch.randn((2, 20000), device="cuda")
    norm, long_norm = torch.ones(k, device="cuda"), torch.ones(20000, device="cuda")
    works = {t: torch.empty(ops.mxfp4_moe_ffn_workspace_bytes(t, n, top_k), dtype=torch.uint8, device="cuda") for t in rows}

    def run():
        out = [*ops.moe_gating(tall, 8), *ops.rms_norm_quant(long, long_norm, want_y=True)[:3]]
        for t, x in rows.items():
            h, scales, y, total = ops.rms_norm_quant(x, norm, residual=x, want_y=True)
            logits = ops.mxfp4_gemv(y, *b, "fp32")
            idx, gate = ops.moe_gating(logits, top_k)
            out += [h, scales, y, total, logits, idx, gate, ops.mxfp4_gemv(y, *wide), ops.mxfp4_gemv(x.float(), *wide, "fp32"),
                    ops.mxfp4_moe_ffn(y, idx, gate, *w1, *w2, workspace=works[t])]
        return out

    ops.init()                                   # the only library call before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for rep in range(2):
        for x in rows.values():
            x.copy_(torch.randn(x.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        if not all(torch.equal(p, q) for p, q in zip(captured, run())):
            print(f"replay {rep} differs from the eager run", flush=True)
            return 1
    print("CAPTURE-OK", flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
