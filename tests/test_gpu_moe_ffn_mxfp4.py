"""The routed FFN of a few tokens on MXFP4 weights against the formula in 64 bits, and the whole decode step that it ends."""
import pytest
import torch

from catccos_amd import ops
from tests.test_gpu_gemv import dequantized, weights

pytestmark = pytest.mark.gpu


def experts_of(e, n, k, seed):
    """(w1, w1_scale, w2, w2_scale): random codes under scales that keep activations near one."""
    both = [[weights(rows, cols, seed + 10 * i + j, lo, lo + 3) for i in range(e)] for j, (rows, cols, lo) in
            enumerate(((n, k, 121), (k, n // 2, 121)))]
    return tuple(torch.stack([p[i] for p in part]) for part in both for i in (0, 1))


def definition(x, idx, gate, w1, w1s, w2, w2s):
    """(out, size): size bounds how far fp32 arithmetic may take out from its value."""
    half, x = w1.shape[1] // 2, x.double()
    out, size = torch.zeros_like(x), torch.zeros_like(x)
    for e in range(w1.shape[0]):
        t, r = (idx == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        a, b, p = dequantized(w1[e], w1s[e]), dequantized(w2[e], w2s[e]), gate[t, r].double()[:, None]
        h, room = x[t] @ a.t(), x[t].abs() @ a.abs().t()
        g, u = h[:, :half], h[:, half:]
        silu = g * torch.sigmoid(g)
        # a matrix product in fp32 loses (k / 32 + 16) * 2^-22 of the magnitudes that it adds; |silu'| < 1.1; exp, division, products and the two halves of
        # the value together less than 2^-15
        loss = (x.shape[1] / 32 + 16) * 2.0 ** -22
        off = 1.1 * loss * room[:, :half] * (u.abs() + loss * room[:, half:]) + silu.abs() * loss * room[:, half:] + (silu * u).abs() * 2.0 ** -15
        out.index_add_(0, t, p * (silu * u @ b.t()))
        size.index_add_(0, t, p.abs() * ((off + (silu * u).abs() * (2 * half / 32 + 80) * 2.0 ** -22) @ b.abs().t()))
    return out, size


def check(got, x, idx, gate, *w):
    want, size = definition(x, idx, gate, *w)
    err = (got.double() - want).abs()
    bound = want.abs() * 2.0 ** -8 + size + 2.0 ** -133
    assert bool((err <= bound).all()), float((err / bound).max())
    # rounding to bf16 alone: errors spread evenly over a step, whose root mean square is 2^-7 / sqrt(12) = 2.3e-3 of a value at the foot of its binade and less
    # above; over many values what is added before it has to stay well below that
    if want.numel() >= 4096:
        assert float(err.norm()) <= 2.5e-3 * float(want.norm())


def routing(tokens, e, top_k, seed):
    z = torch.randn((tokens, e), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    return ops.moe_gating(z, top_k)


@pytest.mark.parametrize("k,n", [(32, 64), (96, 192), (128, 128), (512, 256), (992, 1088), (2080, 640)])
@pytest.mark.parametrize("tokens,e,top_k", [(1, 8, 2), (1, 3, 1), (2, 8, 8), (5, 16, 3), (17, 4, 2), (33, 2, 2), (64, 40, 6), (65, 7, 3), (150, 12, 5)])
def test_against_the_formula(tokens, e, top_k, k, n):
    w = experts_of(e, n, k, k + e)
    x = torch.randn((tokens, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(tokens)).to(torch.bfloat16)
    idx, gate = routing(tokens, e, top_k, tokens + e)
    check(ops.mxfp4_moe_ffn(x, idx, gate, *w), x, idx, gate, *w)


@pytest.mark.parametrize("tokens", [1, 2, 9, 70])
def test_wide_rows(tokens):
    """Rows of W2 for two tiles to a workgroup of the second matmul, the last one in part; k is no multiple of a whole step."""
    w = experts_of(5, 64, 6176, 11)
    x = torch.randn((tokens, 6176), device="cuda", generator=torch.Generator(device="cuda").manual_seed(tokens)).to(torch.bfloat16)
    idx, gate = routing(tokens, 5, 2, tokens)
    check(ops.mxfp4_moe_ffn(x, idx, gate, *w), x, idx, gate, *w)


def test_experts_past_four_gib():
    """W1 of 5 GB: experts on both sides of an offset of 2^32 bytes, weights and sums of the named ones against the formula."""
    e, n, k, named = 600, 1024, 16384, [0, 255, 511, 512, 513, 599]
    few = experts_of(len(named), n, k, 21)
    w = [torch.zeros((e, *t.shape[1:]), dtype=torch.uint8, device="cuda") for t in few]
    assert w[0].numel() > 1 << 32
    for whole, part in zip(w, few):
        whole[torch.tensor(named, device="cuda")] = part
    x = torch.randn((3, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).to(torch.bfloat16)
    local = torch.tensor([[0, 5], [2, 3], [4, 1]], dtype=torch.int32, device="cuda")
    gate = torch.tensor([[0.75, 0.25], [0.5, 0.5], [1.0, 0.125]], device="cuda")
    idx = torch.tensor(named, dtype=torch.int32, device="cuda")[local.long()].contiguous()
    got = ops.mxfp4_moe_ffn(x, idx, gate, *w)
    check(got, x, local, gate, *few)
    assert torch.equal(got, ops.mxfp4_moe_ffn(x, local, gate, *few))


def test_captured_right_after_init():
    """First launches inside a stream capture, after cmx_init() alone (tests/capture_decode_child.py)."""
    import os
    import subprocess
    import sys
    child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "capture_decode_child.py")
    r = subprocess.run([sys.executable, child], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "CAPTURE-OK" in r.stdout, (r.returncode, r.stdout[-2000:], r.stderr[-2000:])


def test_many_routes_and_the_widest_top_k():
    w = experts_of(64, 128, 256, 1)
    for tokens in (3, 64, 70):
        x = torch.randn((tokens, 256), device="cuda").to(torch.bfloat16)
        idx, gate = routing(tokens, 64, 64, tokens)
        check(ops.mxfp4_moe_ffn(x, idx, gate, *w), x, idx, gate, *w)


def test_one_expert_for_all_and_one_named_twice():
    w = experts_of(6, 256, 288, 2)
    x = torch.randn((70, 288), device="cuda").to(torch.bfloat16)
    gate = torch.rand((70, 4), device="cuda")
    for idx in (torch.full((70, 4), 3, dtype=torch.int32, device="cuda"), torch.randint(0, 2, (70, 4), dtype=torch.int32, device="cuda")):
        check(ops.mxfp4_moe_ffn(x, idx, gate, *w), x, idx, gate, *w)


def test_routes_outside_the_experts_add_nothing():
    w = experts_of(8, 192, 160, 3)
    x = torch.randn((9, 160), device="cuda").to(torch.bfloat16)
    idx = torch.randint(-4, 12, (9, 5), dtype=torch.int32, device="cuda")
    idx[0] = -1
    idx[1] = 8
    idx[2] = torch.tensor([2 ** 31 - 1, -2 ** 31, 7, 0, -1], dtype=torch.int32)
    gate = torch.rand((9, 5), device="cuda")
    out = ops.mxfp4_moe_ffn(x, idx, gate, *w)
    check(out, x, idx, gate, *w)
    assert bool((out[:2] == 0).all())
    gone = torch.full((9, 5), -1, dtype=torch.int32, device="cuda")
    assert bool((ops.mxfp4_moe_ffn(x, gone, gate, *w, out=torch.full_like(x, 7.0)) == 0).all())


def test_equal_calls_give_equal_bits_and_garbage_does_no_harm():
    w = experts_of(16, 512, 512, 4)
    x = torch.randn((40, 512), device="cuda").to(torch.bfloat16)
    idx, gate = routing(40, 16, 4, 9)
    want = ops.mxfp4_moe_ffn(x, idx, gate, *w)
    for fill in (0, 0xFF, 0x7F):
        ws = torch.full((ops.mxfp4_moe_ffn_workspace_bytes(40, 512, 4) + 512,), fill, dtype=torch.uint8, device="cuda")
        out = torch.full_like(x, 7.0)
        assert ops.mxfp4_moe_ffn(x, idx, gate, *w, workspace=ws[:-512], out=out) is out and torch.equal(out, want)
        assert bool((ws[-512:] == fill).all())
    for _ in range(5):
        assert torch.equal(ops.mxfp4_moe_ffn(x, idx, gate, *w), want)
    assert ops.mxfp4_moe_ffn(x[:0], idx[:0], gate[:0], *w).shape == (0, 512)


def test_non_finite_tokens_stay_alone():
    w = experts_of(4, 128, 128, 5)
    x = torch.randn((6, 128), device="cuda").to(torch.bfloat16)
    idx, gate = routing(6, 4, 2, 1)
    want = ops.mxfp4_moe_ffn(x, idx, gate, *w)
    x[2, 5] = float("nan")
    x[4, 7] = float("inf")
    got = ops.mxfp4_moe_ffn(x, idx, gate, *w)
    others = torch.tensor([0, 1, 3, 5], device="cuda")
    assert torch.equal(got[others], want[others]) and bool(got[2].isnan().all())


def test_captured_with_graphs_of_its_own_and_on_side_streams():
    ops.init()
    w = experts_of(16, 256, 512, 6)
    xs = [torch.randn((t, 512), device="cuda").to(torch.bfloat16) for t in (1, 20)]
    routes = [routing(t, 16, 4, t) for t in (1, 20)]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in xs], []
    for g, x, (idx, gate) in zip(graphs, xs, routes):
        with torch.cuda.graph(g):
            outs.append(ops.mxfp4_moe_ffn(x, idx, gate, *w))
    for rep in range(3):
        for x, (idx, gate) in zip(xs, routes):
            x.copy_(torch.randn(x.shape, device="cuda"))
            idx.copy_(routing(len(x), 16, 4, 100 + rep)[0])
        streams = [torch.cuda.Stream() for _ in xs]
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for x, (idx, gate), out in zip(xs, routes, outs):
            assert torch.equal(out, ops.mxfp4_moe_ffn(x, idx, gate, *w)), rep


@pytest.mark.parametrize("tokens", [1, 6, 40])
def test_a_decode_step_of_the_layer(tokens):
    """Residual + norm, router logits, gate and experts, as a layer calls them: each stage against its formula on the stage before."""
    k, n, e, top_k = 512, 512, 32, 4
    w = experts_of(e, n, k, 7)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x, residual = (torch.randn((tokens, k), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    norm = (1 + 0.1 * torch.randn(k, generator=g, device="cuda")).to(torch.bfloat16)
    router, router_scale = weights(e, k, 8, 119, 123)
    bias = 0.05 * torch.randn(e, generator=g, device="cuda")

    def step():
        h, total = ops.rms_norm(x, norm, residual=residual)
        logits = ops.mxfp4_gemv(h, router, router_scale, "fp32")
        idx, gate = ops.moe_gating(logits, top_k, "sigmoid", bias, 8, 4, 2, scale=2.5)
        return h, total, logits, idx, gate, ops.mxfp4_moe_ffn(h, idx, gate, *w)
    h, total, logits, idx, gate, out = step()
    t = x.double() + residual.double()
    want = t / torch.sqrt(t.pow(2).mean(dim=1, keepdim=True) + 1e-6) * norm.double()
    assert bool(((h.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -18) + 2.0 ** -133).all()) and torch.equal(total, t.to(torch.bfloat16))
    wide = dequantized(router, router_scale)
    assert bool(((logits.double() - h.double() @ wide.t()).abs() <= (h.double().abs() @ wide.abs().t()) * (k / 32 + 16) * 2.0 ** -22).all())
    from tests.test_gpu_gating import _check
    _check(logits, top_k, "sigmoid", bias, 8, 4, 2, scale=2.5)
    check(out, h, idx, gate, *w)
    # the prefill's way through the same layer: the same gate's answer into the sort
    order, place, counts = ops.moe_init_routing(idx, e)
    assert int(counts.sum()) == tokens * top_k
    ops.init()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for rep in range(3):
        x.copy_(torch.randn(x.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(captured, step())), rep
