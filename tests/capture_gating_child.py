"""Child process of test_gpu_gating.test_the_largest_workgroups_captured_right_after_init: in a process that has launched none of the library's kernels,
cmx_init() alone must be enough to capture the gate at the size whose workgroups hold the most LDS.  The graph is replayed twice, with eager work in between,
and every replay compared bit for bit with an eager run made afterwards.  Prints CAPTURE-OK."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

from catccos_amd import ops                     # noqa: E402


def main() -> int:
    torch.manual_seed(5)
    tokens = 14 * torch.cuda.get_device_properties(0).multi_processor_count
    z, bias = torch.randn((tokens, 512), device="cuda"), 0.05 * torch.randn(512, device="cuda")

    def run():
        return ops.moe_gating(z, 64, "sigmoid", bias, 64, 32, 2)

    ops.init()                                   # the only library call before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for rep in range(2):
        z.copy_(torch.randn(z.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        if not all(torch.equal(p, q) for p, q in zip(captured, run())):
            print(f"replay {rep} differs from the eager run", flush=True)
            return 1
    print("CAPTURE-OK", flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
