"""The FP8 operators and the permutes as they are used together: a token's way through the experts and its gradients; captured, on streams, past 4 GiB."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


def _bf16(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


# Codes are at most half a step, 2^-4 of themselves, off; between two codes the error is spread evenly, so 2^-4 / sqrt(3) of an operand is lost at most and sqrt(2) as much of
# a product of two: 0.051.  Rows of bf16 on the way lose 2^-9 each.
LOST = 2.0 ** -4


@pytest.mark.parametrize("tokens,experts,top_k,h,n", [(300, 8, 3, 512, 384), (1, 16, 4, 1024, 640), (45, 4, 2, 272, 136), (2000, 8, 2, 400, 1040)])
def test_a_layer_and_its_gradients(tokens, experts, top_k, h, n):
    from catccos_amd import ops
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x, w, dout = _bf16(g, tokens, h), _bf16(g, experts, n, h) * 0.05, _bf16(g, tokens, n)
    idx, probs = ops.moe_gating(_bf16(g, tokens, experts), top_k)
    _, to, counts = ops.moe_init_routing(idx, experts)
    xd, wd, dd, pd = x.double(), w.double(), dout.double(), probs.double()
    each = torch.stack([torch.stack([wd[e] @ xd[t] for e in idx[t].tolist()]) for t in range(min(tokens, 100))])                 # [t, top_k, n]

    # there, through the experts, and back
    rows = ops.moe_token_permute(x, to, top_k)
    codes, scales = ops.fp8_block_quant(rows)
    few = ops.fp8_block_quant(x)                                              # quantised first and then moved: the same bits
    assert torch.equal(ops.moe_token_permute(few[0], to, top_k), codes) and torch.equal(ops.moe_token_permute(few[1], to, top_k), scales)
    w8 = ops.fp8_block_quant(w, square=True)
    y = ops.fp8_block_gmm(codes, scales, *w8, counts)
    out = ops.moe_token_unpermute(y, to, probs)
    some = each.shape[0]
    assert _off(out[:some], (pd[:some, :, None] * each).sum(dim=1)) < LOST

    # the gradients of the probabilities, of the rows and of the tokens
    dy, dprobs = ops.moe_token_unpermute_grad(dout, y, to, probs)
    # dprobs[t, r] = <dout[t], y[t, r]>: by Cauchy and Schwarz off by no more than |dout[t]| times what y[t, r] as a vector is off.  (Not as a share of dprobs, which
    # are sums of either sign: four of them can be small by chance.)
    most = LOST * dd[:some].norm(dim=1)[:, None] * each.norm(dim=2)
    assert bool(((dprobs[:some].double() - (dd[:some, None, :] * each).sum(dim=2)).abs() <= most).all())
    w8t = ops.fp8_block_quant(w, square=True, transposed=True)
    assert torch.equal(w8t[0][:, :, :n], w8[0][:, :, :h].transpose(1, 2)) and torch.equal(w8t[1], w8[1].transpose(1, 2))
    drows = ops.fp8_block_gmm(*ops.fp8_block_quant(dy), *w8t, counts)
    dx = ops.moe_token_permute_grad(drows[:, :h], to, top_k)
    want = torch.stack([sum(pd[t, r] * (dd[t] @ wd[e]) for r, e in enumerate(idx[t].tolist())) for t in range(some)])
    assert _off(dx[:some], want) < LOST

    # an expert's weight gradient: blocks along its tokens, scales by the row on both sides
    e = int(counts.argmax())
    mine = slice(int(counts[:e].sum()), int(counts[:e + 1].sum()))
    dw = ops.fp8_block_gemm(*ops.fp8_block_quant(dy[mine], transposed=True), *ops.fp8_block_quant(rows[mine], transposed=True), out="fp32")
    assert dw.shape == (n, h) and _off(dw, dy[mine].double().t() @ rows[mine].double()) < LOST


def test_captured_right_after_init():
    """First launches inside a stream capture, after cmx_init() alone (tests/capture_fp8_child.py)."""
    child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "capture_fp8_child.py")
    r = subprocess.run([sys.executable, child], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "CAPTURE-OK" in r.stdout, (r.returncode, r.stdout[-2000:], r.stderr[-2000:])


def test_two_graphs_and_two_streams_at_once():
    """Products whose parts meet in a workspace of their own, captured twice and replayed on two streams at the same time."""
    from catccos_amd import ops
    ops.init()
    g = torch.Generator(device="cuda").manual_seed(9)
    sides = []
    for _ in range(2):
        a, b = ops.fp8_block_quant(_bf16(g, 256, 7168)), ops.fp8_block_quant(_bf16(g, 4096, 7168), square=True)
        want = ops.fp8_block_gemm(*a, *b, out="fp32")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.fp8_block_gemm(*a, *b, out="fp32")
        sides.append((graph, got, want, torch.cuda.Stream(), a, b))
    assert ops.fp8_block_gemm_workspace_bytes(256, 4096, 7168) > 0
    for _ in range(3):
        for graph, got, _, stream, a, b in sides:
            got.zero_()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
                again = ops.fp8_block_gemm(*a, *b, out="fp32")
                again.record_stream(stream)
        torch.cuda.synchronize()
        for _, got, want, *_ in sides:
            assert torch.equal(got, want)


def test_a_workspace_of_the_caller():
    from catccos_amd import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    a, b = ops.fp8_block_quant(_bf16(g, 250, 7168)), ops.fp8_block_quant(_bf16(g, 4100, 7168), square=True)
    need = ops.fp8_block_gemm_workspace_bytes(250, 4100, 7168)
    whole = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    got = ops.fp8_block_gemm(*a, *b, workspace=whole[:need])
    assert torch.equal(got, ops.fp8_block_gemm(*a, *b)) and bool((whole[need:] == 0xA5).all())
    with pytest.raises(AssertionError):
        ops.fp8_block_gemm(*a, *b, workspace=whole[:need - 16])


def test_on_another_stream_than_the_inputs():
    from catccos_amd import ops
    side = torch.cuda.Stream()
    x = torch.randn((500, 1000), device="cuda").to(torch.bfloat16)
    want = ops.fp8_block_quant(x)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = (x.float() * 1.0).to(torch.bfloat16)                           # made on the side stream, used there
        got = ops.fp8_block_quant(late)
        c = ops.fp8_block_gemm(*got, *ops.fp8_block_quant(late, square=True))
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and torch.equal(c, ops.fp8_block_gemm(*want, *ops.fp8_block_quant(x, square=True)))


def test_operands_past_4_gib():
    from catccos_amd import ops
    k, rows = 16384, 270000                                                   # 4.4 GB of codes
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
    ends = torch.randint(-2, 3, (4, k), device="cuda").to(torch.bfloat16)
    ends[:, ::128] = 7                                                        # the same scale, 1/64, everywhere
    x[:2], x[-2:] = ends[:2], ends[2:]
    codes, scales = ops.fp8_block_quant(x)
    few = ops.fp8_block_quant(ends)
    del x
    assert torch.equal(torch.cat([codes[:2], codes[-2:]]), few[0]) and torch.equal(torch.cat([scales[:2], scales[-2:]]), few[1]) and not bool(codes[2:-2:1000].any())
    b = ops.fp8_block_quant(ends[:, :].repeat(4, 1), square=True)             # 16 rows
    want = (ends.double() @ ends.double().t()).repeat(1, 4)
    c = ops.fp8_block_gemm(codes, scales, *b, out="fp32")
    assert torch.equal(torch.cat([c[:2], c[-2:]]).double(), want) and not bool(c[2:-2].any())
    sizes = torch.tensor([rows - 1, 0, 1], dtype=torch.int32, device="cuda")
    w = torch.stack([b[0], b[0], b[0].flip(0)]).contiguous()
    c = ops.fp8_block_gmm(codes, scales, w, b[1][None].repeat(3, 1, 1).contiguous(), sizes, out="fp32")
    assert torch.equal(torch.cat([c[:2], c[-2:-1]]).double(), want[:3]) and torch.equal(c[-1].double(), want[3].flip(0))


def test_expert_weights_past_4_gib():
    from catccos_amd import ops
    experts, n, k = 40, 8192, 16384                                           # 5.4 GB
    g = torch.Generator(device="cuda").manual_seed(4)
    w = torch.zeros((experts, n, k), dtype=torch.uint8, device="cuda")
    last = torch.randint(-2, 3, (n, k), generator=g, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8)
    w[-1] = last
    ws = torch.ones((experts, n // 128, k // 128), device="cuda")
    a = torch.randint(-2, 3, (5, k), generator=g, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8)
    sizes = torch.zeros(experts, dtype=torch.int32, device="cuda")
    sizes[0], sizes[-1] = 2, 3
    got = ops.fp8_block_gmm(a, torch.ones((5, k // 128), device="cuda"), w, ws, sizes, out="fp32")
    assert not bool(got[:2].any()) and torch.equal(got[2:].double(), a[2:].view(torch.float8_e4m3fn).double() @ last.view(torch.float8_e4m3fn).double().t())
